"""Block-scaled rows (mx4 / mx8) and the operators on them from their definitions, in float64 torch on the CPU.

A row is blocks of 32 columns (the last one filled up with zeros), each under one power of two 2^e with
    mx4   e = max(floor(log2 a) - 2, -127), elements +-{0, .5, 1, 1.5, 2, 3, 4, 6}      (a: the block's largest magnitude)
    mx8   e = max(floor(log2 a), -127),     elements q / 64, q = -127 .. 127
rounded to nearest, ties to the even code, held to the largest element.  A block with an infinity or a NaN is NaN throughout.
"""
import math

import torch

GRID4 = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)


def _blocks(x):
    rows, cols = x.shape
    b = torch.zeros(rows, -(-cols // 32) * 32, dtype=torch.float64)
    b[:, :cols] = x.detach().cpu().double()
    return b.view(rows, -1, 32)


def quantize(x, bits):
    """(codes, scale, values): 0 .. 15 sign-and-magnitude codes or -127 .. 127 (rows, blocks, 32), scale bytes (rows, blocks), float64
    values (rows, cols)."""
    b = _blocks(x)
    finite = torch.isfinite(b).all(dim=2)
    top = torch.where(finite, b.abs().amax(dim=2), torch.zeros(()).double())
    mantissa, e = torch.frexp(top)
    del mantissa
    e = torch.where(top > 0, e - 1 - (2 if bits == 4 else 0), torch.full_like(e, -127)).clamp(min=-127)
    y = torch.where(finite[..., None], b, torch.zeros(()).double()) / torch.exp2(e.double())[..., None]
    if bits == 4:
        size = y.abs()[..., None]
        lower = (GRID4 <= size).sum(dim=-1) - 1                     # the grid point at or below
        upper = (lower + 1).clamp(max=7)
        below, above = size[..., 0] - GRID4[lower], GRID4[upper] - size[..., 0]
        code = torch.where((above < below) | ((above == below) & (lower % 2 == 1)), upper, lower)
        value = torch.where(torch.signbit(y), -GRID4[code], GRID4[code])
        code = code + 8 * torch.signbit(y).long()
    else:
        code = torch.round(64 * y).clamp(-127, 127)
        value = code / 64
        code = code.long()
    value = torch.where(finite[..., None], value * torch.exp2(e.double())[..., None], torch.full((), math.nan).double())
    scale = torch.where(finite, e + 127, torch.full_like(e, 255))
    return code, scale, value.flatten(1)[:, :x.shape[1]]


def pack(codes, scale):
    """The bytes of (codes, scale): what ldm_mx_quantize stores.  4-bit when a code is at most 15 and none is negative is NOT inferred:
    pass 4-bit codes as int64 0 .. 15 and 8-bit codes as int8."""
    rows, blocks = scale.shape
    pad = torch.zeros(rows, -blocks % 4, dtype=torch.uint8)
    s = torch.cat((scale.to(torch.uint8), pad), dim=1)
    if codes.dtype == torch.int8:
        return codes.reshape(rows, -1), s
    pair = codes.reshape(rows, -1, 2)
    return (pair[..., 0] | pair[..., 1] << 4).to(torch.uint8), s


def values(data, scale, cols):
    """float64 values of stored bytes."""
    rows = data.shape[0]
    if data.dtype == torch.uint8:
        code = torch.stack((data.long() & 15, data.long() >> 4), dim=2).reshape(rows, -1, 32)
        v = torch.where(code >= 8, -GRID4[code & 7], GRID4[code & 7])
    else:
        v = data.double().reshape(rows, -1, 32) / 64
    e = scale[:, :v.shape[1]].double() - 127
    unit = torch.where(scale[:, :v.shape[1]] == 255, torch.full((), math.nan).double(), torch.exp2(e))
    return (v * unit[..., None]).flatten(1)[:, :cols]


def gate(g, act):
    """(a(g), a'(g)) of the gate, float64."""
    if act == "geglu":
        cdf = torch.special.erfc(-g / math.sqrt(2)) / 2
        return g * cdf, cdf + g * torch.exp(-g * g / 2) / math.sqrt(2 * math.pi)
    s = torch.sigmoid(g)
    return g * s, s * (1 + g * (1 - s))


def split_pairs(h):
    """Paired columns (16 values, their 16 gates, ...) -> (values, gates)."""
    v = h.reshape(h.shape[0], -1, 2, 16)
    return v[:, :, 0].flatten(1), v[:, :, 1].flatten(1)


def join_pairs(v, g):
    return torch.stack((v.reshape(v.shape[0], -1, 16), g.reshape(g.shape[0], -1, 16)), dim=2).flatten(1)


def glu(h, act):
    v, g = split_pairs(h)
    return v * gate(g, act)[0]


def glu_backward(h, dout, act):
    v, g = split_pairs(h)
    a, da = gate(g, act)
    return join_pairs(dout * a, dout * v * da)
