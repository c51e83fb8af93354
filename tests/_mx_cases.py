"""Bodies of the block-scaled operators' tests, shared by tests/test_mx_cpu.py (the kernel sources on the host emulator, guard pages
behind every buffer) and tests/test_mx_gpu.py (the GPU).  Values against oracle/mx_ref.py in float64.

Tolerances, from the formats and the types alone:
  * quantisation and reading back: equal, scaling by a power of two is exact and the one rounding is the format's.
  * products: every product of two elements is exact in float32 (at most 2 + 2, 8 + 2 or 8 + 7 significant bits), so a sum of K of them
    is off by at most K roundings of partial sums, each at most 2^-23 (nearest or truncated) of the sum of magnitudes; then half a step
    of the output type.
  * gated activation: see glu_tolerance."""
import math

import torch

from conftest import seeded
from oracle import mx_ref

bf = torch.bfloat16
HALF_STEP = {torch.float32: 2.0 ** -24, bf: 2.0 ** -8}


def activations(rows, cols, seed, dtype=bf):
    """Normal values under channel gains of very different sizes, some rows zero and some blocks tiny."""
    x = seeded((rows, cols), seed) * torch.exp(2.0 * seeded((cols,), seed + 1))
    if rows > 2:
        x[rows // 2] = 0
        x[1, : min(cols, 40)] *= 2.0 ** -120
    return x.to(dtype)


def check_quantize(ops, x, bits, dev):
    """Stored bytes and values of a (rows, cols) tensor against the definition, bit for bit."""
    codes, scale, want = mx_ref.quantize(x, bits)
    q = (ops.mx4_quantize if bits == 4 else ops.mx8_quantize)(dev(x))
    assert q.shape == x.shape and q.rows == x.shape[0]
    data, s = mx_ref.pack(codes if bits == 4 else codes.to(torch.int8), scale)
    assert torch.equal(q.scale.cpu(), s)
    if bits == 4:
        # a negative zero in a block filled up with zeros or written for a NaN block carries no sign
        live = (scale != 255)[..., None]
        data, _ = mx_ref.pack(torch.where(live, codes, torch.zeros_like(codes)), scale)
    else:
        data = torch.where((scale != 255)[..., None], codes, torch.zeros_like(codes)).to(torch.int8).reshape(x.shape[0], -1)
    assert torch.equal(q.data.cpu(), data)
    for dtype in (torch.float32, bf):
        got = ops.mx_dequantize(q, dtype)
        assert got.dtype == dtype and got.shape == x.shape
        assert torch.equal(torch.nan_to_num(got.cpu().double(), nan=1e300), torch.nan_to_num(want, nan=1e300))
    return q


def product_error(got, x, w, bias=None, terms=None):
    """Largest excess of |got - x w^T - bias| over its tolerance (<= 0 is a pass); x, w float64."""
    want = x @ w.t() + (0 if bias is None else bias.double())
    size = x.abs() @ w.abs().t() + (0 if bias is None else bias.double().abs())
    tol = (x.shape[1] + 16) * 2.0 ** -23 * size + HALF_STEP[got.dtype] * want.abs()
    return float(((got.cpu().double() - want).abs() - tol).max()) if got.numel() else 0.0


def check_linear(ops, rows, n, k, seed, act, out_dtype, with_bias, dev):
    w = seeded((n, k), seed) / math.sqrt(k)
    x = activations(rows, k, seed + 1)
    b = seeded((n,), seed + 2) if with_bias else None
    wq = ops.mx4_quantize(dev(w))
    wv = mx_ref.quantize(w, 4)[2]
    if act == "mx4":
        xa, xv = ops.mx4_quantize(dev(x)), mx_ref.quantize(x, 4)[2]
    else:
        xa, xv = dev(x), x.double()
    y = ops.mx4_linear(xa, wq, bias=None if b is None else dev(b), out_dtype=out_dtype)
    assert y.shape == (rows, n) and y.dtype == (out_dtype or bf)
    assert product_error(y, xv, wv, b) <= 0


def check_dgrad(ops, rows, n, k, seed, dev):
    w = seeded((n, k), seed) / math.sqrt(k)
    dy = seeded((rows, n), seed + 1).to(bf)
    dx = ops.mx4_linear_dgrad(dev(dy), ops.mx4_quantize(dev(w)))
    assert dx.shape == (rows, k) and dx.dtype == bf
    assert product_error(dx, dy.double(), mx_ref.quantize(w, 4)[2].t().contiguous()) <= 0


def check_wgrad(ops, rows, n, k, seed, dev, accumulate=False):
    x = activations(rows, k, seed)
    dy = seeded((rows, n), seed + 1).to(bf)
    x8 = ops.mx8_quantize(dev(x))
    xv = mx_ref.quantize(x, 8)[2]
    if accumulate:
        first = seeded((n, k), seed + 2)
        out = dev(first.clone())
        got = ops.linear_wgrad_mx8(x8, dev(dy), out=out)
        assert got.data_ptr() == out.data_ptr()
        want, size = first.double(), first.double().abs()
    else:
        got = ops.linear_wgrad_mx8(x8, dev(dy))
        want, size = torch.zeros(n, k, dtype=torch.float64), torch.zeros(n, k, dtype=torch.float64)
    assert got.shape == (n, k) and got.dtype == torch.float32
    want = want + dy.double().t() @ xv
    size = size + dy.double().abs().t() @ xv.abs()
    tol = (rows + 64) * 2.0 ** -23 * size + 2.0 ** -24 * want.abs()
    assert float(((got.cpu().double() - want).abs() - tol).max()) <= 0


def glu_tolerance(g, act, dtype):
    """Bounds on the errors of a(g) and a'(g), absolute, before the result's own rounding.
    float32: a few roundings of each factor; the exponential's and erfc's argument is off by a rounding, which they carry on times
    its own size (g^2 / 2, or g for the sigmoid).  bfloat16: the erfc polynomial's 1.5e-7 / 2 and two one-step instructions on top."""
    u = 2.0 ** -24
    size = g.abs()
    if act == "geglu":
        cdf = torch.special.erfc(-g / math.sqrt(2)) / 2
        pdf = torch.exp(-g * g / 2) / math.sqrt(2 * math.pi)
        extra = 4e-7 if dtype == bf else 0.0
        cdf_tol = u * (16 * cdf + (16 + 4 * g * g) * size * pdf) + extra
        return size * (cdf_tol + 4 * u * cdf), cdf_tol + u * (16 + 4 * g * g) * size * pdf + 4 * u * cdf
    s = torch.sigmoid(g)
    rel = u * (16 + 4 * size)
    return size * s * rel, s * (1 + size) * 2 * rel


def check_glu(ops, rows, ff, seed, act, dtype, recompute, dev):
    h = (1.5 * seeded((rows, 2 * ff), seed)).to(dtype)
    if rows > 1:
        h[0, :64] *= 6.0                         # gates far in both tails
        h[rows - 1, -32:] = 0
    dout = seeded((rows, ff), seed + 1).to(dtype)
    out, h8 = ops.glu_forward_mx8(dev(h), act)
    codes, scale, hv = mx_ref.quantize(h, 8)
    data, s = mx_ref.pack(codes.to(torch.int8), scale)
    assert torch.equal(h8.scale.cpu(), s) and torch.equal(h8.data.cpu(), data) and h8.cols == 2 * ff
    half = HALF_STEP[dtype]
    v, g = mx_ref.split_pairs(h.double())
    ta, _ = glu_tolerance(g, act, dtype)
    want = mx_ref.glu(h.double(), act)
    assert out.dtype == dtype and out.shape == (rows, ff)
    assert float(((out.cpu().double() - want).abs() - (v.abs() * ta + 2 * half * want.abs() + 1e-37)).max()) <= 0
    res = ops.glu_backward_mx8(h8, dev(dout), act, recompute=recompute)
    dh = res[0] if recompute else res
    v, g = mx_ref.split_pairs(hv)
    d = dout.double()
    ta, tda = glu_tolerance(g, act, dtype)
    want = mx_ref.glu_backward(hv, d, act)
    tol = mx_ref.join_pairs(d.abs() * ta, (d * v).abs() * tda) + 2 * half * want.abs() + 1e-37
    assert dh.dtype == dtype and dh.shape == (rows, 2 * ff)
    assert float(((dh.cpu().double() - want).abs() - tol).max()) <= 0
    if recompute:
        want = mx_ref.glu(hv, act)
        assert float(((res[1].cpu().double() - want).abs() - (v.abs() * ta + 2 * half * want.abs() + 1e-37)).max()) <= 0
