"""The block-scaled operators on the host emulator (guard pages behind every buffer, both LDS-DMA completion models), their definition in
oracle/mx_ref.py by itself, and what the front ends and the C entries refuse."""
import math
import os
import sys

import pytest
import torch

HERE = os.path.dirname(os.path.abspath(__file__))
sys.path.insert(0, os.path.join(HERE, "emu"))

import _mx_cases as mx  # noqa: E402
from conftest import seeded  # noqa: E402
from harness import Guarded, emu_lib, emulated  # noqa: E402
from ldm import _lib  # noqa: E402
from oracle import mx_ref  # noqa: E402

bf = torch.bfloat16


# ------------------------------------------------------------------------------------------------------------ the definition
def test_oracle_ties_saturation_and_scales():
    row = torch.zeros(1, 32)
    row[0, :8] = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 4.0])       # ties, scale 1 (largest 5 -> e = 0)
    codes, scale, v = mx_ref.quantize(row, 4)
    assert scale.tolist() == [[127]]
    assert v[0, :8].tolist() == [0.0, 1.0, 1.0, 2.0, 2.0, 4.0, 4.0, 4.0]
    row[0, 8] = -7.9                                                                # held to 6
    assert mx_ref.quantize(row, 4)[2][0, 8] == -6.0
    row = torch.zeros(1, 33)
    row[0, 0], row[0, 32] = 1.999, 2.0 ** -140
    codes, scale, v = mx_ref.quantize(row, 8)
    assert scale.tolist() == [[127, 0]] and v[0, 0] == 127 / 64 and codes[0, 1, 0] == 0
    row[0, 5], row[0, 32] = math.inf, 2.0 ** -133                                  # one step of the smallest scale
    codes, scale, v = mx_ref.quantize(row, 8)
    assert scale.tolist() == [[255, 0]] and torch.isnan(v[0, :32]).all() and v[0, 32] == 2.0 ** -133


# ----------------------------------------------------------------------------------------------------------------- kernels
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dtype", [torch.float32, bf])
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 31), (2, 32), (5, 33), (4, 64), (3, 129), (2, 320), (7, 77), (130, 40)])
def test_quantize(rows, cols, dtype, bits):
    with Guarded() as g, emulated(guard=True) as ops:
        mx.check_quantize(ops, mx.activations(rows, cols, 3, dtype), bits, g.like)


@pytest.mark.parametrize("bits", [4, 8])
def test_quantize_every_exponent_and_special(bits):
    rows = []
    for e in list(range(-149, 128, 7)) + [-128, -127, -126, -125, 126, 127]:
        r = seeded((32,), e + 500).double()
        r = r / r.abs().max() * 1.93
        rows.append((r * 2.0 ** e).clamp(-3.4e38, 3.4e38).float())
    x = torch.stack(rows)
    sp = seeded((6, 64), 9)
    sp[0, 3], sp[1, 40], sp[2, 0] = math.inf, -math.inf, math.nan
    sp[3, :32], sp[4] = 0.0, -0.0
    sp[5, 32:] = torch.finfo(torch.float32).max
    with Guarded() as g, emulated(guard=True) as ops:
        mx.check_quantize(ops, x, bits, g.like)
        mx.check_quantize(ops, sp, bits, g.like)
        mx.check_quantize(ops, sp.to(bf), bits, g.like)


def test_quantize_column_slices_and_leading_dimensions():
    wide = mx.activations(6, 200, 4)
    with Guarded() as g, emulated(guard=True) as ops:
        w = g.like(wide)
        for lo, hi in ((0, 64), (8, 72), (3, 67), (100, 200)):
            q = ops.mx4_quantize(w[:, lo:hi])
            assert torch.equal(ops.mx_dequantize(q, torch.float32).double(), mx_ref.quantize(wide[:, lo:hi], 4)[2])
        q = ops.mx8_quantize(w.view(2, 3, 200))
        assert q.shape == (2, 3, 200) and q.data.shape == (2, 3, 224) and q.scale.shape == (2, 3, 8)
        v = ops.mx_dequantize(q, torch.float32)
        assert torch.equal(v.view(6, 200).double(), mx_ref.quantize(wide, 8)[2])
        assert ops.mx_dequantize(ops.mx4_quantize(w[0, :40]), bf).shape == (40,)
        empty = ops.mx4_quantize(w[:0])
        assert empty.rows == 0 and ops.mx_dequantize(empty, bf).shape == (0, 200)


@pytest.mark.parametrize("dma", ["lazy", "eager"])
@pytest.mark.parametrize("rows,n,k", [(65, 40, 1), (70, 130, 32), (130, 40, 130), (100, 136, 320), (129, 257, 520), (70, 64, 1100)])
def test_product_both_4bit(rows, n, k, dma):
    with Guarded() as g, emulated(dma, guard=True) as ops:
        mx.check_linear(ops, rows, n, k, 11, "mx4", torch.float32 if n % 2 else bf, k != 130, g.like)


@pytest.mark.parametrize("dma", ["lazy", "eager"])
def test_product_both_4bit_large_tile(dma):
    """Enough tiles that the 256 x 256 one is taken: 8 x 16 of them, the last row and column of tiles cut short."""
    with Guarded() as g, emulated(dma, guard=True) as ops:
        mx.check_linear(ops, 1800, 3900, 328, 12, "mx4", bf, True, g.like)


@pytest.mark.parametrize("act", ["mx4", "bf16"])
@pytest.mark.parametrize("rows,n,k", [(1, 1, 1), (1, 48, 320), (2, 17, 33), (16, 40, 130), (17, 33, 96), (33, 20, 1100), (64, 16, 64), (5, 12, 77)])
def test_product_few_rows(rows, n, k, act):
    with Guarded() as g, emulated(guard=True) as ops:
        mx.check_linear(ops, rows, n, k, 13, act, torch.float32 if n % 2 else None, rows != 2, g.like)


def test_product_few_rows_wide_and_unaligned():
    with Guarded() as g, emulated(guard=True) as ops:
        mx.check_linear(ops, 3, 8200, 64, 14, "bf16", bf, True, g.like)
        mx.check_linear(ops, 3, 8200, 64, 14, "mx4", torch.float32, False, g.like)
        w = seeded((40, 64), 5) / 8
        x = seeded((1 + 6 * 64,), 6).to(bf)
        off = g.like(x)[1:].view(6, 64)                    # 2-byte aligned only
        y = ops.mx4_linear(off, ops.mx4_quantize(g.like(w)))
        assert mx.product_error(y, x[1:].view(6, 64).double(), mx_ref.quantize(w, 4)[2]) <= 0


@pytest.mark.parametrize("dma", ["lazy", "eager"])
@pytest.mark.parametrize("rows,n,k", [(66, 200, 2100), (130, 70, 777), (1100, 1300, 300), (1030, 1410, 1100), (2050, 4104, 200)])
def test_product_both_4bit_tiles(rows, n, k, dma):
    """Outputs of every tile's choice -- 64 x 64 with its columns split, 128 x 128, 256 x 128 -- with more steps than LDS has slots."""
    with Guarded() as g, emulated(dma, guard=True) as ops:
        mx.check_linear(ops, rows, n, k, 21, "mx4", bf if n % 4 else torch.float32, True, g.like)


def test_product_both_4bit_largest_tile():
    """256 x 256: many outputs and long sums."""
    with Guarded() as g, emulated("lazy", guard=True) as ops:
        mx.check_linear(ops, 2050, 4104, 2050, 21, "mx4", bf, True, g.like)


@pytest.mark.parametrize("dma", ["lazy", "eager"])
@pytest.mark.parametrize("rows,n,k", [(300, 3200, 200), (1300, 1000, 77), (300, 130, 1300), (66, 130, 1300), (70, 33, 8), (1030, 1000, 200), (500, 10230, 200), (1000, 10230, 200)])
def test_product_bf16_tiles(rows, n, k, dma):
    """Likewise for bfloat16 activations: 64 x 64, 128 x 128, 128 x 160, 256 x 160."""
    with Guarded() as g, emulated(dma, guard=True) as ops:
        mx.check_linear(ops, rows, n, k, 22, "bf16", bf if n % 3 else torch.float32, True, g.like)


@pytest.mark.parametrize("act", ["mx4", "bf16"])
@pytest.mark.parametrize("dma", ["lazy", "eager"])
@pytest.mark.parametrize("rows,n,k", [(5, 24, 9000), (3, 20, 2049), (20, 18, 3100), (40, 18, 3100), (3, 4100, 300), (2, 12300, 70), (2, 16500, 64),
                                      (20, 4100, 136), (40, 4100, 136)])
def test_product_few_rows_variants(rows, n, k, dma, act):
    """Fragments of the weights a workgroup from one to four, rings that wrap, an odd number of columns."""
    with Guarded() as g, emulated(dma, guard=True) as ops:
        mx.check_linear(ops, rows, n, k, 23, act, bf if n % 3 else torch.float32, True, g.like)


@pytest.mark.parametrize("rows,n,k", [(3, 40, 160), (70, 72, 96), (70, 72, 160), (70, 72, 520), (70, 72, 1100), (1030, 1100, 520)])
def test_product_nan_block_reaches_its_rows_only(rows, n, k):
    """The last block of a row and the first of the next lie side by side, and so do their scales: a NaN in one of them stays there."""
    x, w = seeded((rows, k), 1), seeded((n, k), 2)
    x[1, k - 1], w[9, 0], w[20, k - 1] = math.nan, math.inf, math.nan
    want = torch.zeros(rows, n, dtype=torch.bool)
    want[1], want[:, 9], want[:, 20] = True, True, True
    with Guarded() as g, emulated(guard=True) as ops:
        wq = ops.mx4_quantize(g.like(w))
        assert torch.equal(torch.isnan(ops.mx4_linear(ops.mx4_quantize(g.like(x)), wq)), want)
        assert torch.equal(torch.isnan(ops.mx4_linear(g.like(x.to(bf)), wq)), want)


@pytest.mark.parametrize("rows,n,k", [(70, 64, 96), (90, 50, 77)])
def test_product_many_bf16_rows(rows, n, k):
    with Guarded() as g, emulated(guard=True) as ops:
        mx.check_linear(ops, rows, n, k, 15, "bf16", bf, True, g.like)


@pytest.mark.parametrize("rows,n,k", [(1, 32, 8), (70, 96, 64), (33, 50, 77), (5, 200, 300)])
def test_input_gradient(rows, n, k):
    with Guarded() as g, emulated(guard=True) as ops:
        mx.check_dgrad(ops, rows, n, k, 17, g.like)


@pytest.mark.parametrize("act", ["geglu", "swiglu"])
@pytest.mark.parametrize("dtype", [torch.float32, bf])
@pytest.mark.parametrize("rows,ff,recompute", [(1, 16, False), (5, 48, True), (33, 80, True), (130, 16, False)])
def test_gated_activation(rows, ff, recompute, dtype, act):
    with Guarded() as g, emulated(guard=True) as ops:
        mx.check_glu(ops, rows, ff, 19, act, dtype, recompute, g.like)


@pytest.mark.parametrize("dma", ["lazy", "eager"])
@pytest.mark.parametrize("rows,n,k,acc", [(1, 8, 1, False), (33, 16, 40, True), (70, 264, 300, False), (100, 320, 64, False), (97, 56, 320, True),
                                          (1100, 24, 40, False), (40, 13, 77, True)])
def test_weight_gradient(rows, n, k, acc, dma):
    with Guarded() as g, emulated(dma, guard=True) as ops:
        mx.check_wgrad(ops, rows, n, k, 23, g.like, accumulate=acc)


@pytest.mark.parametrize("rows", [700, 2900])
def test_weight_gradient_of_many_splits(rows):
    with Guarded() as g, emulated(guard=True) as ops:
        mx.check_wgrad(ops, rows, 24, 40, 24, g.like, accumulate=rows == 2900)


def test_gradients_of_rows_at_any_alignment():
    x, flat = mx.activations(30, 72, 3), seeded((1 + 30 * 40,), 4).to(bf)
    with Guarded() as g, emulated(guard=True) as ops:
        off, dy = g.like(flat)[1:].view(30, 40), g.like(flat[1:].view(30, 40))
        x8, w = ops.mx8_quantize(g.like(x)), ops.mx4_quantize(g.like(seeded((40, 72), 5)))
        assert torch.equal(ops.linear_wgrad_mx8(x8, off), ops.linear_wgrad_mx8(x8, dy))
        assert torch.equal(ops.mx4_linear_dgrad(off, w), ops.mx4_linear_dgrad(dy, w))


def test_weight_gradient_of_nan_blocks_stays_in_their_columns():
    x = seeded((40, 96), 1)
    x[7, 40] = math.nan
    dy = seeded((40, 16), 2).to(bf)
    with Guarded() as g, emulated(guard=True) as ops:
        dw = ops.linear_wgrad_mx8(ops.mx8_quantize(g.like(x)), g.like(dy))
        assert torch.isnan(dw[:, 32:64]).all() and torch.isfinite(dw[:, :32]).all() and torch.isfinite(dw[:, 64:]).all()


# ---------------------------------------------------------------------------------------------------------------- refusals
def _refused(fn, exc=(TypeError, ValueError)):
    lib = emu_lib()
    before = lib.emu_launch_count()
    with pytest.raises(exc):
        fn()
    assert lib.emu_launch_count() == before, "a refused call must not launch a kernel"


def test_front_ends_refuse():
    with emulated() as ops:
        x = torch.randn(4, 64)
        q4, q8 = ops.mx4_quantize(x), ops.mx8_quantize(x)
        w = ops.mx4_quantize(torch.randn(48, 64))
        xb, bias = x.to(bf), torch.zeros(48)
        w3, w8, odd8 = ops.mx4_quantize(torch.randn(2, 48, 64)), ops.mx8_quantize(torch.randn(48, 64)), ops.mx8_quantize(torch.randn(4, 48))
        _refused(lambda: ops.mx4_quantize(x.double()))
        _refused(lambda: ops.mx4_quantize(x.t()))
        _refused(lambda: ops.mx8_quantize(x[:, ::2]))
        _refused(lambda: ops.mx8_quantize(torch.randn(1, 64).expand(4, 64)))                  # overlapping rows
        _refused(lambda: ops.mx4_quantize(torch.randn(4, 0)))
        _refused(lambda: ops.mx4_quantize(torch.tensor(1.0)))
        _refused(lambda: ops.mx_dequantize(x, bf))
        _refused(lambda: ops.mx_dequantize(q4, torch.float16))
        _refused(lambda: ops.MxTensor(q4.data, q4.scale, 65))
        _refused(lambda: ops.MxTensor(q4.data, q4.scale[:, :2], 64))
        _refused(lambda: ops.MxTensor(q4.data.float(), q4.scale, 64))
        _refused(lambda: ops.MxTensor(q4.data, q4.scale.float(), 64))
        _refused(lambda: ops.MxTensor(q4.data, q4.scale[:2], 64))
        _refused(lambda: ops.MxTensor(torch.empty(4, 64, dtype=torch.uint8)[:, ::2], q4.scale, 64))
        ops.mx4_linear(q4, w, bias=bias)
        ops.mx4_linear(xb, w, bias=bias)
        _refused(lambda: ops.mx4_linear(x, w))                                                # float32 activations
        _refused(lambda: ops.mx4_linear(q8, w))
        _refused(lambda: ops.mx4_linear(xb, q8))
        _refused(lambda: ops.mx4_linear(xb, x))
        _refused(lambda: ops.mx4_linear(xb[:, :32], w))
        _refused(lambda: ops.mx4_linear(xb[:, :32].contiguous(), w))
        _refused(lambda: ops.mx4_linear(xb, w, bias=bias.to(bf)))
        _refused(lambda: ops.mx4_linear(xb, w, bias=bias[:40]))
        _refused(lambda: ops.mx4_linear(xb, w, out_dtype=torch.float16))
        _refused(lambda: ops.mx4_linear(xb, w3))
        dy = torch.randn(4, 48).to(bf)
        ops.mx4_linear_dgrad(dy, w)
        _refused(lambda: ops.mx4_linear_dgrad(dy.float(), w))
        _refused(lambda: ops.mx4_linear_dgrad(dy[:, :32], w))
        _refused(lambda: ops.mx4_linear_dgrad(torch.randn(48, 4).to(bf).t(), w))
        _refused(lambda: ops.mx4_linear_dgrad(dy, w8))
        h = torch.randn(4, 64).to(bf)
        _, h8 = ops.glu_forward_mx8(h, "geglu")
        _refused(lambda: ops.glu_forward_mx8(h, "relu"))
        _refused(lambda: ops.glu_forward_mx8(torch.randn(4, 48).to(bf), "geglu"))
        _refused(lambda: ops.glu_forward_mx8(torch.randn(64, 4).to(bf).t(), "geglu"))
        _refused(lambda: ops.glu_forward_mx8(h.half(), "geglu"))
        d = torch.randn(4, 32).to(bf)
        ops.glu_backward_mx8(h8, d, "geglu")
        _refused(lambda: ops.glu_backward_mx8(q4, d, "geglu"))
        _refused(lambda: ops.glu_backward_mx8(h8, d, "glu"))
        _refused(lambda: ops.glu_backward_mx8(h8, d[:3], "geglu"))
        _refused(lambda: ops.glu_backward_mx8(h8, torch.randn(32, 4).to(bf).t(), "geglu"))
        _refused(lambda: ops.glu_backward_mx8(odd8, torch.randn(4, 24).to(bf), "geglu"))
        ops.linear_wgrad_mx8(q8, dy)
        _refused(lambda: ops.linear_wgrad_mx8(q4, dy))
        _refused(lambda: ops.linear_wgrad_mx8(q8, dy.float()))
        _refused(lambda: ops.linear_wgrad_mx8(q8, dy[:3]))
        _refused(lambda: ops.linear_wgrad_mx8(q8, dy, out=torch.zeros(48, 65)))
        _refused(lambda: ops.linear_wgrad_mx8(q8, dy, out=torch.zeros(64, 48).t()))
        _refused(lambda: ops.linear_wgrad_mx8(q8, dy, out=torch.zeros(48, 64).to(bf)))


def test_front_ends_refuse_cpu_tensors():
    from ldm import ops
    x = torch.randn(4, 64)
    for fn in (lambda: ops.mx4_quantize(x), lambda: ops.mx8_quantize(x), lambda: ops.glu_forward_mx8(x, "geglu")):
        with pytest.raises(RuntimeError):
            fn()


def test_c_entries_refuse_without_a_launch():
    """Host checks of the library itself (no GPU needed: every call returns before a launch)."""
    lib = _lib.load()
    a = torch.zeros(4096, dtype=torch.uint8)
    p = (a.data_ptr() + 15) // 16 * 16

    def bad(rc):
        return rc == -1 and lib.ldm_last_error() != b""

    assert bad(lib.ldm_mx_quantize(p, 7, 1, 32, 32, 4, p, p, 0))
    assert bad(lib.ldm_mx_quantize(p, 0, 1, 32, 32, 5, p, p, 0))
    assert bad(lib.ldm_mx_quantize(p, 0, 1, 0, 32, 4, p, p, 0))
    assert bad(lib.ldm_mx_quantize(p, 0, 1, 32, 31, 4, p, p, 0))
    assert bad(lib.ldm_mx_quantize(0, 0, 1, 32, 32, 4, p, p, 0))
    assert bad(lib.ldm_mx_quantize(p + 2, 0, 1, 32, 32, 4, p, p, 0))
    assert bad(lib.ldm_mx_quantize(p, 0, 1, 32, 32, 4, p + 4, p, 0))
    assert bad(lib.ldm_mx_quantize(p, 0, 1, 32, 32, 4, p, p + 1, 0))
    assert lib.ldm_mx_quantize(0, 0, 0, 32, 32, 4, 0, 0, 0) == 0
    assert bad(lib.ldm_mx_dequantize(p, p, 4, -1, 32, p, 0, 32, 0))
    assert bad(lib.ldm_mx_dequantize(p, 0, 4, 1, 32, p, 0, 32, 0))
    assert bad(lib.ldm_mx4_dequantize_t(p, p, 32, 32, p, 28, 0))
    assert bad(lib.ldm_mx4_dequantize_t(p, p, 32, 32, p, 33, 0))
    assert bad(lib.ldm_glu_forward_mx8(p, p, p, p, 1, 1, 24, 1, 0))
    assert bad(lib.ldm_glu_backward_mx8(p, p, p, 0, 0, 1, 1, 16, 1, 0))
    assert bad(lib.ldm_glu_backward_mx8(p, p, p, p, p + 2, 1, 1, 16, 1, 0))
    assert bad(lib.ldm_mx4_linear(p, p, p, p, 0, p, 9, 1, 1, 1, 0))
    assert bad(lib.ldm_mx4_linear(p, p, p, p, 0, p, 0, 1, 0, 1, 0))
    assert bad(lib.ldm_mx4_linear(p, p, p, p, 0, 0, 0, 1, 1, 1, 0))
    assert bad(lib.ldm_mx4_linear(p + 2, p, p, p, 0, p, 0, 1, 1, 1, 0))
    assert bad(lib.ldm_mx4_linear(p, p, p, p, 0, p, 0, 1, 1, (1 << 22) + 1, 0))
    assert lib.ldm_mx4_linear(0, 0, 0, 0, 0, 0, 0, 0, 1, 1, 0) == 0
    assert bad(lib.ldm_mx4_linear(p, p, p, p, 0, p, 0, 1 << 39, 1 << 30, 1, 0))
    assert bad(lib.ldm_linear_bf16(p, p, 0, p, 1, 1, 1, 12, 0))                               # k not a multiple of 8
    assert bad(lib.ldm_linear_bf16(p + 2, p, 0, p, 1, 1, 1, 8, 0))
    assert bad(lib.ldm_linear_bf16(p, p + 8, 0, p, 1, 1, 1, 8, 0))
    assert bad(lib.ldm_linear_bf16(p, p, 0, p + 1, 1, 1, 1, 8, 0))
    assert bad(lib.ldm_linear_bf16(p, p, 0, p, 5, 1, 1, 8, 0))
    assert bad(lib.ldm_linear_bf16(p, p, 0, p, 1, 1 << 39, 1 << 30, 8, 0))
    assert lib.ldm_linear_bf16(0, 0, 0, 0, 1, 0, 1, 8, 0) == 0
    assert bad(lib.ldm_mx4_linear_wide(p, p, p, 0, p, 1, 1, 8, 8, p, 127, 0))                 # 2 * 8 * 8 bytes of workspace
    assert bad(lib.ldm_mx4_linear_wide(p, p, p, 0, p, 1, 1, 8, 8, 0, 128, 0))
    assert bad(lib.ldm_mx4_linear_wide(p, p, p, 0, p, 1, 1, 8, 7, p, 128, 0))                 # and 2 * 8 for the row laid out anew
    assert bad(lib.ldm_mx4_linear_wide(p, 0, p, 0, p, 1, 1, 8, 7, p, 4096, 0))                # nothing launched for the rows either
    assert bad(lib.ldm_mx4_linear_wide(p, p, p, 0, p + 1, 1, 1, 8, 7, p, 4096, 0))
    assert bad(lib.ldm_mx4_linear_wide(p, p, p, 0, p, 7, 1, 8, 7, p, 4096, 0))
    assert bad(lib.ldm_mx4_linear_dgrad(p, p, 0, p, 1, 7, 8, p, 4096, 0))
    assert bad(lib.ldm_mx4_linear_wide(p, p, p + 2, 0, p, 1, 1, 8, 7, p, 4096, 0))
    assert bad(lib.ldm_mx4_linear_wide(p + 1, p, p, 0, p, 1, 1, 8, 8, p, 4096, 0))
    assert bad(lib.ldm_mx4_linear_wide(p, p, p, 0, p, 1, 1, 8, (1 << 21) + 1, p, 4096, 0))
    assert lib.ldm_mx4_linear_wide(0, 0, 0, 0, 0, 1, 0, 8, 8, 0, 0, 0) == 0
    assert bad(lib.ldm_mx4_linear_dgrad(p, p, p, p, 1, 8, 8, p, 127, 0))
    assert bad(lib.ldm_mx4_linear_dgrad(p + 2, p, p, p, 1, 8, 8, p, 128, 0))
    assert bad(lib.ldm_mx4_linear_dgrad(p, p, p, p, 1, 0, 8, p, 4096, 0))
    assert lib.ldm_mx4_linear_dgrad(0, 0, 0, 0, 0, 8, 8, 0, 0, 0) == 0
    assert bad(lib.ldm_pad_columns_bf16(p, p, 1, 8, 12, 0))
    assert bad(lib.ldm_pad_columns_bf16(p, p, 1, 9, 8, 0))
    assert bad(lib.ldm_pad_columns_bf16(p + 1, p, 1, 7, 8, 0))
    assert bad(lib.ldm_pad_columns_bf16(p, p + 2, 1, 7, 8, 0))
    assert lib.ldm_pad_columns_bf16(0, 0, 0, 7, 8, 0) == 0
    assert bad(lib.ldm_linear_wgrad_mx8(p, p, p, p, 1, 12, 32, 0, 0, 0, 0))                   # n not a multiple of 8
    assert bad(lib.ldm_linear_wgrad_mx8(p, p, p, p, 0, 8, 32, 0, 0, 0, 0))
    need = lib.ldm_linear_wgrad_mx8_workspace_bytes(1 << 20, 8, 32)
    assert need > 0 and bad(lib.ldm_linear_wgrad_mx8(p, p, p, p, 1 << 20, 8, 32, 0, p, need - 1, 0))
    assert bad(lib.ldm_linear_wgrad_mx8(p, p, p, p, 1 << 20, 8, 32, 0, 0, 0, 0))
    assert lib.ldm_linear_wgrad_mx8_workspace_bytes(0, 8, 32) == 0
