"""The block-scaled ("microscaled") operators as they are measured: quantisation to 4 and 8 bits, the product with 4-bit
weights and its input gradient, the gated activation whose backward pass reads an 8-bit checkpoint, and the weight gradient
from an 8-bit checkpoint.  ``run`` computes them in plain torch, or, where ``own`` is true, by the framework's kernels.

Formats (blocks of 32 consecutive columns of a row, one power-of-two scale a block, held as its exponent + 127 in a byte):
  mx4   elements 0, .5, 1, 1.5, 2, 3, 4, 6 and their negatives (sign, two exponent bits, one mantissa bit), two to a byte, the
        lower column in the lower half; the exponent of a block is floor(log2(largest magnitude)) - 2
  mx8   whole numbers -127 .. 127 in 64ths; the exponent of a block is floor(log2(largest magnitude))
Elements are rounded to the nearest value, ties to the even code, and held to the largest one.  Exponents are held to -127 and
above.  A block with an infinity or a NaN in it stands for NaN (scale byte 255).  Rows are filled up with zeros to whole blocks,
rows of scale bytes to whole groups of four.
"""
import math
import os
import sys

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


def _ops():
    package = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "latent-diffusion_amd")
    if package not in sys.path:
        sys.path.insert(0, package)
    from ldm import ops
    return ops


# ------------------------------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # a gated projection's float32 weights (1280 -> 2 x 5120 channels) become 4-bit weights, once a model
        {"name": "quantise weights", "op": "quantise", "fmt": "mx4", "dtype": "f32", "rows": 10240, "cols": 1280},
        # the tokens of two prompts' text context, a ragged width, kept in 8 bits
        {"name": "quantise context, ragged", "op": "quantise", "fmt": "mx8", "dtype": "bf16", "rows": 154, "cols": 765},
        # the gated projection of the 64 x 64 level for eight images: short rows, many tokens
        {"name": "product, 64x64 level", "op": "linear", "act": "mx4", "out": "bf16", "rows": 32768, "k": 320, "n": 2560},
        # a large square product: what the matrix cores reach with 4-bit operands
        {"name": "product, large", "op": "linear", "act": "mx4", "out": "bf16", "rows": 8192, "k": 8192, "n": 8192},
        # one image's time embedding, a single token: latency
        {"name": "product, one token", "op": "linear", "act": "bf16", "out": "bf16", "rows": 1, "k": 1280, "n": 1280},
        # a few tokens against large 4-bit weights: the rate at which weights are read
        {"name": "product, 16 tokens", "op": "linear", "act": "bf16", "out": "f32", "rows": 16, "k": 8192, "n": 10240},
        # input gradient of the 32 x 32 level's gated projection for eight images
        {"name": "input gradient, 32x32", "op": "dgrad", "rows": 8192, "k": 640, "n": 5120},
        # input gradient of the context projection for two prompts, odd sizes
        {"name": "input gradient, ragged", "op": "dgrad", "rows": 154, "k": 765, "n": 1290},
        # gated activation of the 32 x 32 level for eight images, forward and backward
        {"name": "gated activation, 32x32", "op": "glu", "act": "geglu", "dtype": "bf16", "rows": 8192, "ff": 2560},
        # the same of a small float32 model
        {"name": "gated activation, small", "op": "glu", "act": "swiglu", "dtype": "f32", "rows": 77, "ff": 256},
        # weight gradient of the 64 x 64 level's gated projection for eight images
        {"name": "weight gradient, 64x64", "op": "wgrad", "rows": 32768, "k": 320, "n": 2560},
        # weight gradient of the context projection for two prompts, odd sizes
        {"name": "weight gradient, ragged", "op": "wgrad", "rows": 154, "k": 765, "n": 1290},
    ]


def _log(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["quantise", "linear", "linear", "dgrad", "glu", "wgrad"])
    if op == "quantise":
        return {"op": op, "fmt": rng.choice(["mx4", "mx8"]), "dtype": rng.choice(["f32", "bf16"]),
                "rows": _log(rng, 1, 10240), "cols": _log(rng, 1, 1280)}
    if op == "glu":
        return {"op": op, "act": rng.choice(["geglu", "swiglu"]), "dtype": rng.choice(["f32", "bf16"]),
                "rows": _log(rng, 1, 8192), "ff": 16 * _log(rng, 1, 160)}
    rows, k, n = _log(rng, 1, 8192), _log(rng, 32, 2560), _log(rng, 16, 2560)
    if rng.random() < 0.5:      # half of the cases with channel counts as models have them, half with any
        k, n = -(-k // 32) * 32, -(-n // 32) * 32
    if op == "linear":
        return {"op": op, "act": rng.choice(["mx4", "bf16"]), "out": rng.choice(["bf16", "f32"]), "rows": rows, "k": k, "n": n}
    return {"op": op, "rows": rows, "k": k, "n": n}


# ----------------------------------------------------------------------------------------------------------------- inputs
def _activations(gen, rows, cols, dtype):
    """Roughly normal values with a few channels of several times the others' size, as a network's activations have."""
    x = torch.randn(rows, cols, device="cuda", generator=gen)
    gain = torch.exp(0.7 * torch.randn(cols, device="cuda", generator=gen))
    return (x * gain).to(dtype)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    op = case["op"]
    state = dict(case)
    if op == "quantise":
        dtype = _DTYPES[case["dtype"]]
        if case["fmt"] == "mx4":
            state["x"] = (torch.randn(case["rows"], case["cols"], device="cuda", generator=gen) / math.sqrt(case["cols"])).to(dtype)
        else:
            state["x"] = _activations(gen, case["rows"], case["cols"], dtype)
        return state
    if op == "glu":
        dtype = _DTYPES[case["dtype"]]
        state["h"] = _activations(gen, case["rows"], 2 * case["ff"], dtype)
        state["dout"] = torch.randn(case["rows"], case["ff"], device="cuda", generator=gen).to(dtype)
        return state
    rows, k, n = case["rows"], case["k"], case["n"]
    if op in ("linear", "wgrad"):
        state["x"] = _activations(gen, rows, k, torch.bfloat16)
    if op in ("dgrad", "wgrad"):
        state["dy"] = torch.randn(rows, n, device="cuda", generator=gen).to(torch.bfloat16)
    if op in ("linear", "dgrad"):
        w = torch.randn(n, k, device="cuda", generator=gen) / math.sqrt(k)
        state["data"], state["scale"] = _pack4(w)
    if op == "linear":
        state["bias"] = torch.randn(n, device="cuda", generator=gen)
    return state


def _blocks(x):
    """float32 (rows, blocks, 32), filled up with zeros."""
    rows, cols = x.shape
    return torch.nn.functional.pad(x.float(), (0, -cols % 32)).view(rows, -1, 32)


def _block_exponents(b, below):
    """floor(log2(largest magnitude)) - below, at least -127; and which blocks are finite."""
    largest = b.abs().amax(dim=2, keepdim=True)
    finite = torch.isfinite(b).all(dim=2, keepdim=True)
    _, e = torch.frexp(torch.where(finite, largest, torch.ones_like(largest)))
    e = torch.where(largest > 0, e - 1 - below, torch.full_like(e, -127))
    return e.clamp(min=-127), finite


def _scaled(b, e):
    """b * 2^-e in two exact steps: 2^127 and 2^126 are the largest powers that both exist in float32 both ways."""
    half = torch.div(-e, 2, rounding_mode="floor")
    return torch.ldexp(torch.ldexp(b, half), -e - half)


def _codes4(b):
    """Codes 0 .. 7 of the magnitudes and the scale exponents."""
    e, finite = _block_exponents(b, 2)
    y = _scaled(b, e).abs()
    code = ((y > 0.25).int() + (y >= 0.75).int() + (y > 1.25).int() + (y >= 1.75).int() + (y > 2.5).int() + (y >= 3.5).int()
            + (y > 5.0).int())
    return torch.where(finite, code, torch.zeros_like(code)), e, finite


_GRID4 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _pack4(w):
    """The bytes that 4-bit weights are kept in: (rows, 16 * blocks) elements and (rows, blocks up to a multiple of 4) scales."""
    b = _blocks(w)
    code, e, finite = _codes4(b)
    nibble = (code | ((b < 0).int() << 3)).view(w.shape[0], -1, 2)
    data = (nibble[..., 0] | (nibble[..., 1] << 4)).to(torch.uint8)
    scale = torch.where(finite, e + 127, torch.full_like(e, 255)).to(torch.uint8).squeeze(2)
    return data.contiguous(), torch.nn.functional.pad(scale, (0, -scale.shape[1] % 4)).contiguous()


# ------------------------------------------------------------------------------------------------------------ plain forms
def _values4(x):
    """What x stands for in mx4, in float32."""
    b = _blocks(x)
    code, e, finite = _codes4(b)
    grid = torch.tensor(_GRID4, device=x.device)
    v = _scaled(torch.where(b < 0, -grid[code], grid[code]), -e)
    return torch.where(finite, v, torch.full_like(v, math.nan)).flatten(1)[:, :x.shape[1]]


def _values8(x):
    """What x stands for in mx8, in float32."""
    b = _blocks(x)
    e, finite = _block_exponents(b, 0)
    q = torch.round(_scaled(b, e - 6)).clamp(-127, 127)
    v = _scaled(q, 6 - e)
    return torch.where(finite, v, torch.full_like(v, math.nan)).flatten(1)[:, :x.shape[1]]


def _unpack4(data, scale, cols):
    nibble = torch.stack((data & 15, data >> 4), dim=2).view(data.shape[0], -1, 32).int()
    grid = torch.tensor(_GRID4 + tuple(-v for v in _GRID4), device=data.device)
    e = scale[:, :nibble.shape[1], None].int() - 127
    return _scaled(grid[nibble], -e).flatten(1)[:, :cols]


def _gate(g, act):
    """The gate's activation and its derivative."""
    if act == "geglu":
        cdf = 0.5 * (1 + torch.erf(g / math.sqrt(2)))
        return g * cdf, cdf + g * torch.exp(-0.5 * g * g) / math.sqrt(2 * math.pi)
    s = torch.sigmoid(g)
    return g * s, s * (1 + g * (1 - s))


def _pairs(h):
    """Values and gates of pre-activations whose columns go 16 values, their 16 gates, the next 16 values, ..."""
    v = h.view(h.shape[0], -1, 2, 16)
    return v[:, :, 0].reshape(h.shape[0], -1), v[:, :, 1].reshape(h.shape[0], -1)


def _paired(v, g):
    return torch.stack((v.view(v.shape[0], -1, 16), g.view(v.shape[0], -1, 16)), dim=2).flatten(1)


def run(state):
    op = state["op"]
    if own:
        return _run_own(state, op)
    if op == "quantise":
        return (_values4 if state["fmt"] == "mx4" else _values8)(state["x"]).to(state["x"].dtype)
    if op == "linear":
        x = _values4(state["x"]) if state["act"] == "mx4" else state["x"].float()
        w = _unpack4(state["data"], state["scale"], state["k"])
        return (x @ w.t() + state["bias"]).to(_DTYPES[state["out"]])
    if op == "dgrad":
        return (state["dy"].float() @ _unpack4(state["data"], state["scale"], state["k"])).to(torch.bfloat16)
    if op == "wgrad":
        return state["dy"].float().t() @ _values8(state["x"])
    h, dout = state["h"], state["dout"]
    v, g = _pairs(h.float())
    out = (v * _gate(g, state["act"])[0]).to(h.dtype)
    v, g = _pairs(_values8(h))                  # the backward pass has the checkpoint alone
    a, da = _gate(g, state["act"])
    d = dout.float()
    return {"out": out, "dh": _paired(d * a, d * v * da).to(h.dtype)}


def _run_own(state, op):
    ops = _ops()
    if op == "quantise":
        q = ops.mx4_quantize(state["x"]) if state["fmt"] == "mx4" else ops.mx8_quantize(state["x"])
        return ops.mx_dequantize(q, state["x"].dtype)
    if op == "glu":
        out, h8 = ops.glu_forward_mx8(state["h"], state["act"])
        return {"out": out, "dh": ops.glu_backward_mx8(h8, state["dout"], state["act"])}
    if op == "wgrad":
        return ops.linear_wgrad_mx8(ops.mx8_quantize(state["x"]), state["dy"])
    w = ops.MxTensor(state["data"], state["scale"], state["k"])
    if op == "dgrad":
        return ops.mx4_linear_dgrad(state["dy"], w)
    x = ops.mx4_quantize(state["x"]) if state["act"] == "mx4" else state["x"]
    return ops.mx4_linear(x, w, bias=state["bias"], out_dtype=_DTYPES[state["out"]])


# ------------------------------------------------------------------------------------------------------------------- work
def _mx_bytes(rows, cols, bits):
    """Elements and one scale byte a block."""
    return rows * -(-cols // 32) * (4 * bits + 1)


def work(case):
    op = case["op"]
    if op == "quantise":        # x in, the quantised form out and in again (it is what one call leaves for the other), values out
        size = 2 if case["dtype"] == "bf16" else 4
        n = case["rows"] * case["cols"]
        return {"bytes": 2 * size * n + 2 * _mx_bytes(case["rows"], case["cols"], 4 if case["fmt"] == "mx4" else 8), "flops": 0}
    if op == "glu":             # h and dout in, out and dh out, the checkpoint out in the forward pass and in in the backward pass
        size = 2 if case["dtype"] == "bf16" else 4
        return {"bytes": 6 * size * case["rows"] * case["ff"] + 2 * _mx_bytes(case["rows"], 2 * case["ff"], 8), "flops": 0}
    rows, k, n = case["rows"], case["k"], case["n"]
    flops = 2.0 * rows * k * n
    if op == "linear":
        return {"bytes": 2 * rows * k + _mx_bytes(n, k, 4) + 4 * n + (2 if case["out"] == "bf16" else 4) * rows * n, "flops": flops}
    if op == "dgrad":
        return {"bytes": 2 * rows * n + _mx_bytes(n, k, 4) + 2 * rows * k, "flops": flops}
    return {"bytes": 2 * rows * k + 2 * rows * n + 4 * n * k, "flops": flops}


# ------------------------------------------------------------------------------------------------ the definition in 64 bits
def _exact_values(x, fmt):
    """Each block's values from the format's definition: the nearest multiple of the step that holds at the value's size."""
    rows, cols = x.shape
    v = torch.zeros(rows, -(-cols // 32) * 32, dtype=torch.float64, device=x.device)
    v[:, :cols] = x.double()
    v = v.view(rows, -1, 32)
    top = v.abs().max(dim=2, keepdim=True).values
    power = torch.floor(torch.log2(torch.where(top > 0, top, torch.ones_like(top))))
    power = torch.where(torch.exp2(power) > top, power - 1, power)              # a logarithm that came out a hair too large
    power = torch.where(torch.exp2(power + 1) <= top, power + 1, power)         # or too small
    unit = torch.exp2(torch.where(top > 0, power - (2 if fmt == "mx4" else 0), torch.zeros_like(power)).clamp(min=-127))
    y = v / unit
    if fmt == "mx4":
        size = y.abs()
        step = torch.where(size < 2, 0.5, torch.where(size < 4, 1.0, 2.0)).double()
        y = (torch.round(y / step) * step).clamp(-6, 6)
    else:
        y = (torch.round(y * 64)).clamp(-127, 127) / 64
    return (y * unit).view(rows, -1)[:, :cols]


def _exact_weights(state):
    low, high = state["data"].long() % 16, state["data"].long() // 16
    code = torch.cat((low[:, :, None], high[:, :, None]), dim=2).view(state["n"], -1)
    exponent, mantissa = (code % 8) // 2, code % 2
    size = torch.where(exponent == 0, 0.5 * mantissa, (1 + 0.5 * mantissa) * torch.exp2(exponent.double() - 1))
    unit = torch.exp2(state["scale"].double() - 127).repeat_interleave(32, dim=1)[:, :code.shape[1]]
    return (torch.where(code >= 8, -size, size) * unit)[:, :state["k"]]


def exact(case, seed):
    state = prepare(case, seed)
    op = case["op"]
    if op == "quantise":
        return _exact_values(state["x"], case["fmt"])
    if op == "linear":
        x = _exact_values(state["x"], "mx4") if case["act"] == "mx4" else state["x"].double()
        return torch.matmul(x, _exact_weights(state).t().contiguous()) + state["bias"].double()
    if op == "dgrad":
        return torch.matmul(state["dy"].double(), _exact_weights(state))
    if op == "wgrad":
        return torch.matmul(state["dy"].double().t().contiguous(), _exact_values(state["x"], "mx8"))

    def gate(t):
        if case["act"] == "geglu":
            tail = torch.special.erfc(-t * math.sqrt(0.5)) / 2
            return t * tail, tail + t * torch.exp(-t * t / 2) * math.sqrt(0.5 / math.pi)
        s = 1 / (1 + torch.exp(-t))
        return t * s, s + t * s * (1 - s)

    def halves(h):
        columns = torch.arange(2 * case["ff"], device=h.device)
        return h[:, columns % 32 < 16], h[:, columns % 32 >= 16]

    v, g = halves(state["h"].double())
    out = v * gate(g)[0]
    v, g = halves(_exact_values(state["h"], "mx8"))
    a, da = gate(g)
    d = state["dout"].double()
    dh = torch.empty(case["rows"], 2 * case["ff"], dtype=torch.float64, device=d.device)
    columns = torch.arange(2 * case["ff"], device=d.device)
    dh[:, columns % 32 < 16] = d * a
    dh[:, columns % 32 >= 16] = d * v * da
    return {"out": out, "dh": dh}
