"""Bodies of tests/test_mx_storage_cpu.py and tests/test_mx_storage_gpu.py: what a row's storage holds behind its last column."""
import torch

from _mx_paths import exact4
from conftest import seeded

bf = torch.bfloat16


def stored(ops, x, cols, dev):
    """(clean, dirty): the first `cols` columns of x in 4 bits as mx4_quantize leaves them -- zeros behind -- and the same rows with live elements
    behind the last column and NaN scales behind the last block."""
    whole = ops.mx4_quantize(dev(x))
    blocks = (cols + 31) // 32
    data, scale = whole.data[:, :16 * blocks].cpu().clone(), whole.scale[:, :(blocks + 3) // 4 * 4].cpu().clone()
    dirty = ops.MxTensor(dev(data.clone()), dev(torch.where(torch.arange(scale.shape[1]) < blocks, scale, torch.full_like(scale, 255))), cols)
    element = torch.arange(32 * blocks).view(-1, 2) < cols
    data &= (element[:, 0] * 0x0F + element[:, 1] * 0xF0).to(torch.uint8)
    clean = ops.MxTensor(dev(data), dev(torch.where(torch.arange(scale.shape[1]) < blocks, scale, torch.zeros_like(scale))), cols)
    assert not torch.equal(clean.data, dirty.data) or not torch.equal(clean.scale, dirty.scale)
    return clean, dirty


def check_product(ops, rows, n, k, act, dev):
    """A product of rows with anything behind their last column has the bits of the one with zeros there."""
    wide = -(-k // 128) * 128
    w, w_dirty = stored(ops, seeded((n, wide), 5), k, dev)
    if act == "mx4":
        x, x_dirty = stored(ops, seeded((rows, wide), 6), k, dev)
    else:
        x = x_dirty = dev(seeded((rows, k), 6).to(bf))
    want = ops.mx4_linear(x, w, out_dtype=torch.float32)
    assert torch.isfinite(want).all()
    for a, b in ((x_dirty, w_dirty), (x_dirty, w), (x, w_dirty)):
        assert torch.equal(ops.mx4_linear(a, b, out_dtype=torch.float32), want)


def check_exact_product(ops, rows, n, k, dev):
    """One product of 4-bit rows with anything behind their last column, against sums that are exact (_mx_paths.exact4)."""
    wide = -(-k // 128) * 128
    x, w = exact4(rows, wide, 1), exact4(n, wide, 2)
    got = ops.mx4_linear(stored(ops, x, k, dev)[1], stored(ops, w, k, dev)[1], out_dtype=torch.float32)
    assert torch.equal(got.cpu(), x[:, :k] @ w[:, :k].t())


def check_other_readers(ops, dev):
    """Reading back, the input gradient, and 8-bit rows in the weight gradient."""
    w, w_dirty = stored(ops, seeded((48, 128), 5), 45, dev)
    assert torch.equal(ops.mx_dequantize(w, bf), ops.mx_dequantize(w_dirty, bf))
    dy = dev(seeded((20, 48), 7).to(bf))
    assert torch.equal(ops.mx4_linear_dgrad(dy, w), ops.mx4_linear_dgrad(dy, w_dirty))
    q = ops.mx8_quantize(dev(seeded((20, 45), 8)))
    data, scale = q.data.cpu().clone(), q.scale.cpu().clone()
    data[:, 45:], scale[:, 2:] = 99, 255
    dirty = ops.MxTensor(dev(data), dev(scale), 45)
    assert torch.equal(ops.linear_wgrad_mx8(q, dy), ops.linear_wgrad_mx8(dirty, dy))
    assert torch.equal(ops.mx_dequantize(q, bf), ops.mx_dequantize(dirty, bf))
