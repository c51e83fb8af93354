"""Which kernel a product with block-scaled operands runs, case by case, and operands whose sums are exact.

The cases name the kernel that they are there for; tests/test_mx_paths_cpu.py holds them against the dispatch, at every size, and against the
kernels that the library has.  A change of the dispatch thus fails there instead of leaving a kernel without a test.

Exact operands: 4-bit elements under scale 1 (every block starts with a 4 or a 6), bfloat16 whole numbers, 8-bit whole numbers (every block
starts with one of 64 .. 127).  Products are multiples of 1/4 and sums of k of them stay below 2^24 / 4 (k <= 9000: 36 k = 324,000), those of
the weight gradient whole numbers below 2^24 (508 rows <= 2^24 up to 33,000 rows): every partial sum is a float32, in any order, so the
results are equal to the definition's.  One column too many or too few shows, however long the sum."""
import math

import torch

from oracle import mx_ref

bf = torch.bfloat16

# (rows, n, k, kernel without the output type): both operands 4-bit
MX4 = [
    (3, 40, 300, "mx4_rows_kernel<true, 1, 1, 8, 2, true"),
    (5, 24, 9000, "mx4_rows_kernel<true, 1, 1, 8, 2, true"),
    (2, 4100, 300, "mx4_rows_kernel<true, 1, 2, 8, 3, true"),
    (2, 8200, 70, "mx4_rows_kernel<true, 1, 3, 8, 2, true"),
    (2, 12300, 70, "mx4_rows_kernel<true, 1, 4, 8, 2, true"),
    (2, 16500, 64, "mx4_rows_kernel<true, 1, 2, 4, 3, true"),
    (20, 18, 3100, "mx4_rows_kernel<true, 2, 1, 8, 2, true"),
    (20, 4100, 136, "mx4_rows_kernel<true, 2, 2, 4, 3, true"),
    (40, 18, 3100, "mx4_rows_kernel<true, 4, 1, 8, 3, true"),
    (130, 70, 777, "mx4_rows_kernel<true, 4, 1, 8, 3, true"),
    (40, 4100, 136, "mx4_rows_kernel<true, 4, 2, 4, 4, true"),
    # 64 x 64, columns split between the waves of a workgroup: one step a wave, rings that wrap, sums that end inside a block
    (290, 900, 77, "mx_gemm_kernel<64, 64, 1, 1, 4, 2, true"),
    (290, 901, 1050, "mx_gemm_kernel<64, 64, 1, 1, 4, 2, true"),
    (290, 900, 2100, "mx_gemm_kernel<64, 64, 1, 1, 4, 2, true"),
    (290, 901, 3333, "mx_gemm_kernel<64, 64, 1, 1, 4, 2, true"),
    (290, 900, 4097, "mx_gemm_kernel<64, 64, 1, 1, 4, 2, true"),
    (1030, 1410, 300, "mx_gemm_kernel<128, 128, 2, 2, 1, 3, true"),
    (1030, 1411, 1100, "mx_gemm_kernel<128, 128, 2, 2, 1, 3, true"),
    (2050, 4104, 200, "mx4_gemm_kernel<256, 128, 2, 2, 2"),
]
MX4_LARGE = [
    (154, 2560, 2560, "mx_gemm_kernel<64, 64, 1, 1, 4, 2, true"),
    (290, 901, 8999, "mx_gemm_kernel<64, 64, 1, 1, 4, 2, true"),
    (1030, 1410, 8999, "mx_gemm_kernel<128, 128, 2, 2, 1, 3, true"),
    (2050, 4104, 1999, "mx4_gemm_kernel<256, 128, 2, 2, 2"),
    (2050, 4104, 2050, "mx4_gemm_kernel<256, 256, 2, 4, 4"),
    (2050, 4105, 8999, "mx4_gemm_kernel<256, 256, 2, 4, 4"),
]
# bfloat16 rows on 4-bit weights
BF16 = [
    (3, 40, 304, "mx4_rows_kernel<false, 1, 1, 8, 2, true"),
    (3, 40, 301, "mx4_rows_kernel<false, 1, 1, 8, 2, false"),
    (5, 24, 9000, "mx4_rows_kernel<false, 1, 1, 8, 2, true"),
    (2, 4100, 304, "mx4_rows_kernel<false, 1, 2, 8, 3, true"),
    (2, 4100, 301, "mx4_rows_kernel<false, 1, 2, 8, 3, false"),
    (2, 8200, 72, "mx4_rows_kernel<false, 1, 3, 8, 2, true"),
    (2, 8200, 70, "mx4_rows_kernel<false, 1, 3, 8, 2, false"),
    (2, 12300, 72, "mx4_rows_kernel<false, 1, 4, 8, 2, true"),
    (2, 12300, 70, "mx4_rows_kernel<false, 1, 4, 8, 2, false"),
    (2, 16500, 64, "mx4_rows_kernel<false, 1, 2, 4, 3, true"),
    (2, 16500, 65, "mx4_rows_kernel<false, 1, 2, 4, 3, false"),
    (20, 18, 3096, "mx4_rows_kernel<false, 2, 1, 8, 2, true"),
    (20, 18, 3100, "mx4_rows_kernel<false, 2, 1, 8, 2, false"),
    (20, 4100, 136, "mx4_rows_kernel<false, 2, 2, 4, 3, true"),
    (20, 4100, 137, "mx4_rows_kernel<false, 2, 2, 4, 3, false"),
    (40, 18, 3096, "mx4_rows_kernel<false, 4, 1, 4, 2, true"),
    (300, 130, 1300, "mx4_rows_kernel<false, 4, 1, 4, 2, false"),
    (40, 4100, 136, "mx4_rows_kernel<false, 4, 2, 4, 2, true"),
    (40, 4100, 137, "mx4_rows_kernel<false, 4, 2, 4, 2, false"),
    (4000, 16, 64, "mx4_rows_kernel<false, 4, 1, 4, 2, true"),
    # widened once
    (4000, 160, 1288, "mx_gemm_kernel<64, 64, 1, 1, 4, 2, false"),       # few workgroups, but a large x
    (300, 3200, 1100, "mx_gemm_kernel<64, 64, 1, 1, 4, 2, false"),
    (300, 3201, 2101, "mx_gemm_kernel<64, 64, 1, 1, 4, 2, false"),
    (66000, 16, 9, "mx_gemm_kernel<64, 64, 1, 1, 4, 2, false"),          # more rows to pad than a grid's second dimension has
    (1300, 1000, 77, "mx_gemm_kernel<128, 128, 2, 2, 1, 3, false"),
    (1030, 1001, 901, "mx_gemm_kernel<128, 128, 2, 2, 1, 3, false"),
    (500, 10230, 200, "mx_gemm_kernel<128, 160, 4, 1, 1, 3, false"),
    (1000, 10230, 200, "mx_gemm_kernel<256, 160, 4, 1, 1, 3, false"),
]
BF16_LARGE = [
    (300, 3200, 8999, "mx_gemm_kernel<64, 64, 1, 1, 4, 2, false"),
    (1030, 1000, 5001, "mx_gemm_kernel<128, 128, 2, 2, 1, 3, false"),
    (500, 10230, 2001, "mx_gemm_kernel<128, 160, 4, 1, 1, 3, false"),
    (1000, 10231, 2000, "mx_gemm_kernel<256, 160, 4, 1, 1, 3, false"),
]
# input gradient: (rows, n, k), sums over n
DGRAD = [
    (33, 50, 77, "mx_gemm_kernel<64, 64, 1, 1, 4, 2, false"),
    (70, 2101, 300, "mx_gemm_kernel<64, 64, 1, 1, 4, 2, false"),
    (1100, 301, 3000, "mx_gemm_kernel<128, 128, 2, 2, 1, 3, false"),
]
DGRAD_LARGE = [(154, 8999, 765, "mx_gemm_kernel<64, 64, 1, 1, 4, 2, false"), (8192, 5120, 640, "mx_gemm_kernel<128, 160, 4, 1, 1, 3, false")]
# weight gradient: (rows, n, k), whole and split over rows
WGRAD = [
    (150, 320, 160, "linear_wgrad_mx8_kernel<320, 160, 4, 2>"),
    (600, 320, 150, "linear_wgrad_mx8_kernel<320, 160, 4, 2>"),
    (150, 250, 190, "linear_wgrad_mx8_kernel<256, 192, 4, 2>"),
    (600, 256, 192, "linear_wgrad_mx8_kernel<256, 192, 4, 2>"),
    (150, 256, 160, "linear_wgrad_mx8_kernel<256, 160, 4, 2>"),
    (600, 249, 150, "linear_wgrad_mx8_kernel<256, 160, 4, 2>"),
    (150, 13, 77, "linear_wgrad_mx8_kernel<256, 128, 4, 2>"),
    (1100, 256, 128, "linear_wgrad_mx8_kernel<256, 128, 4, 2>"),
]
WGRAD_LARGE = [
    (154, 1290, 765, "linear_wgrad_mx8_kernel<256, 192, 4, 2>"),
    (20000, 250, 190, "linear_wgrad_mx8_kernel<256, 192, 4, 2>"),
    (32768, 2560, 320, "linear_wgrad_mx8_kernel<320, 160, 4, 2>"),
]
SPLIT_ROWS = 512        # rows from which a weight gradient of few tiles is split: partial tiles and their fold


def exact4(rows, cols, seed):
    g = torch.Generator().manual_seed(seed)
    grid = mx_ref.GRID4.float()
    x = grid[torch.randint(0, 8, (rows, cols), generator=g)]
    x[:, ::32] = grid[torch.randint(6, 8, (rows, -(-cols // 32)), generator=g)]
    return torch.where(torch.rand(rows, cols, generator=g) < 0.5, -x, x)


def exact8(rows, cols, seed):
    g = torch.Generator().manual_seed(seed)
    x = torch.randint(0, 128, (rows, cols), generator=g)
    x[:, ::32] = torch.randint(64, 128, (rows, -(-cols // 32)), generator=g)
    return torch.where(torch.rand(rows, cols, generator=g) < 0.5, -x, x).float()


def whole(rows, cols, seed, most):
    return torch.randint(-most, most + 1, (rows, cols), generator=torch.Generator().manual_seed(seed)).float()


def check_linear(ops, rows, n, k, act, dev, out_dtypes=(torch.float32, bf)):
    w = exact4(n, k, 1)
    x = exact4(rows, k, 2) if act == "mx4" else whole(rows, k, 2, 6)
    bias = whole(1, n, 3, 32)[0] / 4
    wq = ops.mx4_quantize(dev(w))
    xa = ops.mx4_quantize(dev(x)) if act == "mx4" else dev(x.to(bf))
    want = x @ w.t() + bias
    for dtype in out_dtypes:
        assert torch.equal(ops.mx4_linear(xa, wq, bias=dev(bias), out_dtype=dtype).cpu(), want.to(dtype))


def check_dgrad(ops, rows, n, k, dev):
    w, dy = exact4(n, k, 1), whole(rows, n, 2, 6)
    assert torch.equal(ops.mx4_linear_dgrad(dev(dy.to(bf)), ops.mx4_quantize(dev(w))).cpu(), (dy @ w).to(bf))


def check_wgrad(ops, rows, n, k, dev):
    x, dy, first = exact8(rows, k, 1), whole(rows, n, 2, 4), whole(n, k, 3, 100)
    x8, dyd = ops.mx8_quantize(dev(x)), dev(dy.to(bf))
    want = (dy.double().t() @ x.double()).float()
    assert torch.equal(ops.linear_wgrad_mx8(x8, dyd).cpu(), want)
    out = dev(first.clone())
    ops.linear_wgrad_mx8(x8, dyd, out=out)
    assert torch.equal(out.cpu(), want + first)
    assert torch.equal(ops.linear_wgrad_mx8(x8, dyd, out=out, accumulate=False).cpu(), want)


def check_nan_blocks(ops, rows, n, k, act, dev):
    """A NaN in the last block of a row and the first of another reaches those rows' outputs and no others."""
    x, w = exact4(rows, k, 1), exact4(n, k, 2)
    x[1, k - 1], w[9, 0], w[20, k - 1] = math.nan, math.inf, math.nan
    want = torch.zeros(rows, n, dtype=torch.bool)
    want[1], want[:, 9], want[:, 20] = True, True, True
    xa = ops.mx4_quantize(dev(x)) if act == "mx4" else dev(x.to(bf))
    assert torch.equal(torch.isnan(ops.mx4_linear(xa, ops.mx4_quantize(dev(w)))).cpu(), want)


NAN_MX4 = [(290, 900, 96), (290, 900, 160), (290, 900, 520), (290, 901, 2100), (1030, 1410, 160), (2050, 4104, 96)]
NAN_BF16 = [(300, 3200, 96), (300, 3200, 100), (500, 10230, 72), (130, 70, 160)]
