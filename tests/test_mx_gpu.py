"""The block-scaled operators on the GPU against oracle/mx_ref.py (float64): the bodies of tests/_mx_cases.py at sizes from one row
to full tiles, other streams, captured graphs, offsets past 32 bits, and the operators together as a fine-tuning step uses them."""
import math

import pytest
import torch

import _mx_cases as mx
from conftest import same_bits, seeded
from ldm import ops
from oracle import mx_ref

pytestmark = pytest.mark.gpu
bf = torch.bfloat16


def dev(t):
    return t.cuda()


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dtype", [torch.float32, bf])
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 31), (3, 33), (2, 1280), (154, 765), (77, 768), (1000, 320), (4096, 1280), (33, 8191)])
def test_quantize(rows, cols, dtype, bits):
    mx.check_quantize(ops, mx.activations(rows, cols, 3, dtype), bits, dev)


@pytest.mark.parametrize("bits", [4, 8])
def test_quantize_every_exponent_and_special(bits):
    rows = []
    for e in range(-149, 128):
        r = seeded((32,), e + 500).double()
        rows.append((r / r.abs().max() * 1.93 * 2.0 ** e).clamp(-3.4e38, 3.4e38).float())
    x = torch.stack(rows)
    sp = seeded((6, 64), 9)
    sp[0, 3], sp[1, 40], sp[2, 0] = math.inf, -math.inf, math.nan
    sp[3, :32], sp[4] = 0.0, -0.0
    sp[5, 32:] = torch.finfo(torch.float32).max
    for t in (x, x.to(bf), sp, sp.to(bf)):
        mx.check_quantize(ops, t, bits, dev)


@pytest.mark.parametrize("bits", [4, 8])
def test_quantize_every_bfloat16(bits):
    """Every finite bfloat16 as the largest magnitude of its block, and every one as a small member of a block."""
    every = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(bf)
    every = every[torch.isfinite(every.float())]
    lone = torch.zeros(every.numel(), 32, dtype=bf)
    lone[:, 5] = every
    mx.check_quantize(ops, lone, bits, dev)
    mates = every[: every.numel() // 31 * 31].view(-1, 31)
    mates = torch.cat((mates, torch.full((mates.shape[0], 1), 1.75, dtype=bf)), dim=1)
    mx.check_quantize(ops, mates, bits, dev)


def test_quantize_column_slices():
    wide = mx.activations(300, 2000, 4)
    w = wide.cuda()
    for lo, hi in ((0, 640), (8, 1288), (3, 67), (1000, 2000), (1999, 2000)):
        q = ops.mx4_quantize(w[:, lo:hi])
        assert torch.equal(ops.mx_dequantize(q, torch.float32).cpu().double(), mx_ref.quantize(wide[:, lo:hi], 4)[2])
    q = ops.mx8_quantize(w.view(3, 100, 2000))
    assert q.shape == (3, 100, 2000)
    assert torch.equal(ops.mx_dequantize(q, bf).cpu().double().view(300, 2000), mx_ref.quantize(wide, 8)[2])


@pytest.mark.parametrize("rows,n,k", [(65, 33, 1), (65, 130, 32), (100, 136, 320), (129, 257, 520), (257, 640, 640), (300, 1280, 768), (1024, 1290, 765),
                                      (70, 64, 4097), (128, 128, 128), (500, 96, 384), (2048, 4104, 352), (4099, 2560, 320)])
@pytest.mark.parametrize("out_dtype", [bf, torch.float32])
def test_product_both_4bit(rows, n, k, out_dtype):
    mx.check_linear(ops, rows, n, k, 11, "mx4", out_dtype, True, dev)


@pytest.mark.parametrize("act", ["mx4", "bf16"])
@pytest.mark.parametrize("rows,n,k", [(1, 1, 1), (1, 1280, 320), (1, 1280, 1280), (2, 17, 33), (8, 5120, 1280), (16, 40, 130), (17, 33, 96), (33, 20, 1100),
                                      (64, 160, 64), (5, 12, 77), (16, 8200, 2048), (48, 640, 8191), (64, 8200, 96)])
def test_product_few_rows(rows, n, k, act):
    mx.check_linear(ops, rows, n, k, 13, act, torch.float32 if n % 2 else None, rows != 2, dev)


@pytest.mark.parametrize("rows,n,k", [(65, 64, 96), (90, 50, 77), (1000, 1280, 640), (4096, 320, 1280)])
def test_product_many_bf16_rows(rows, n, k):
    mx.check_linear(ops, rows, n, k, 15, "bf16", bf, True, dev)


@pytest.mark.parametrize("rows,n,k", [(66, 200, 2100), (130, 70, 7777), (1100, 1300, 300), (1030, 1410, 4100), (2050, 4104, 2000), (2050, 4104, 2050), (4100, 4000, 3000)])
def test_product_both_4bit_tiles(rows, n, k):
    """Outputs of every tile's choice -- 64 x 64 with its columns split, 128 x 128, 256 x 128, 256 x 256 -- with more steps than LDS has slots."""
    mx.check_linear(ops, rows, n, k, 21, "mx4", bf if n % 4 else torch.float32, True, dev)


@pytest.mark.parametrize("rows,n,k", [(300, 3200, 200), (1300, 1000, 77), (300, 130, 1300), (66, 130, 1300), (70, 33, 8), (154, 1290, 5001), (1030, 1000, 2000), (500, 10230, 1000), (1000, 10230, 1000)])
def test_product_bf16_tiles(rows, n, k):
    """Likewise for bfloat16 activations: 64 x 64, 128 x 128, 128 x 160, 256 x 160."""
    mx.check_linear(ops, rows, n, k, 22, "bf16", bf if n % 3 else torch.float32, True, dev)


@pytest.mark.parametrize("act", ["mx4", "bf16"])
@pytest.mark.parametrize("rows,n,k", [(5, 24, 9000), (3, 20, 2049), (20, 18, 3100), (40, 18, 3100), (3, 4100, 300), (2, 12300, 700), (2, 16500, 640),
                                      (20, 4100, 1360), (40, 4100, 1360), (16, 10240, 4096)])
def test_product_few_rows_variants(rows, n, k, act):
    """Fragments of the weights a workgroup from one to four, rings that wrap, an odd number of columns."""
    mx.check_linear(ops, rows, n, k, 23, act, bf if n % 3 else torch.float32, True, dev)


@pytest.mark.parametrize("rows,n,k", [(3, 40, 160), (70, 72, 96), (70, 72, 160), (70, 72, 520), (70, 72, 1100), (1030, 1100, 520), (2050, 4104, 520)])
def test_product_nan_block_of_a_neighbouring_row(rows, n, k):
    """The last block of a row and the first of the next lie side by side, and so do their scales: a NaN in one of them stays there."""
    x, w = seeded((rows, k), 1), seeded((n, k), 2)
    x[1, k - 1], w[9, 0], w[20, k - 1] = math.nan, math.inf, math.nan
    want = torch.zeros(rows, n, dtype=torch.bool)
    want[1], want[:, 9], want[:, 20] = True, True, True
    wq = ops.mx4_quantize(w.cuda())
    assert torch.equal(torch.isnan(ops.mx4_linear(ops.mx4_quantize(x.cuda()), wq)).cpu(), want)
    assert torch.equal(torch.isnan(ops.mx4_linear(x.to(bf).cuda(), wq)).cpu(), want)


def test_product_leading_dimensions_and_unaligned_rows():
    w, x = seeded((40, 64), 5) / 8, seeded((1 + 6 * 64,), 6).to(bf)
    off = x.cuda()[1:].view(2, 3, 64)
    y = ops.mx4_linear(off, ops.mx4_quantize(w.cuda()))
    assert y.shape == (2, 3, 40)
    assert mx.product_error(y.view(6, 40), x[1:].view(6, 64).double(), mx_ref.quantize(w, 4)[2]) <= 0
    yq = ops.mx4_linear(ops.mx4_quantize(off), ops.mx4_quantize(w.cuda()), out_dtype=torch.float32)
    assert yq.shape == (2, 3, 40)
    assert ops.mx4_linear(off[:0], ops.mx4_quantize(w.cuda())).shape == (0, 3, 40)


def test_product_nan_block_reaches_its_rows_only():
    x, w = seeded((100, 96), 1), seeded((72, 96), 2)
    x[7, 40] = math.nan
    w[9, 3] = math.inf
    y = ops.mx4_linear(ops.mx4_quantize(x.cuda()), ops.mx4_quantize(w.cuda())).cpu()
    want = torch.zeros(100, 72, dtype=torch.bool)
    want[7], want[:, 9] = True, True
    assert torch.equal(torch.isnan(y), want)


@pytest.mark.parametrize("rows,n,k", [(1, 32, 8), (70, 96, 64), (154, 1290, 765), (5, 200, 300), (1024, 5120, 640)])
def test_input_gradient(rows, n, k):
    mx.check_dgrad(ops, rows, n, k, 17, dev)


@pytest.mark.parametrize("rows,n,k", [(7, 4097, 96), (300, 2049, 640), (1030, 2560, 1000), (4100, 640, 1280)])
def test_input_gradient_of_long_sums_and_odd_columns(rows, n, k):
    mx.check_dgrad(ops, rows, n, k, 18, dev)


def test_input_gradient_against_differences():
    """d/dx of sum(dy * (x W^T)) by central differences of the forward product (weights as stored, float32 output)."""
    w, dy = ops.mx4_quantize(seeded((48, 64), 1).cuda()), seeded((3, 48), 2).to(bf)
    dx = ops.mx4_linear_dgrad(dy.cuda(), w).cpu().double()
    x = seeded((3, 64), 3).to(bf)
    for col in (0, 31, 32, 63):
        plus, minus = x.clone(), x.clone()
        plus[:, col] += 1.0
        minus[:, col] -= 1.0
        f = [(ops.mx4_linear(t.cuda(), w, out_dtype=torch.float32).cpu().double() * dy.double()).sum(dim=1) for t in (plus, minus)]
        diff = (f[0] - f[1]) / (plus[:, col].double() - minus[:, col].double())
        # 64 + 16 roundings of sums of |x w| <= 64 * 4 * 6, times 48 |dy| <= 4, and half a bf16 step of dx
        assert float((dx[:, col] - diff).abs().max()) <= 80 * 2.0 ** -23 * 64 * 24 * 48 * 4 + 2.0 ** -8 * float(diff.abs().max())


@pytest.mark.parametrize("act", ["geglu", "swiglu"])
@pytest.mark.parametrize("dtype", [torch.float32, bf])
@pytest.mark.parametrize("rows,ff,recompute", [(1, 16, False), (5, 48, True), (77, 256, True), (154, 5120, False), (2048, 1280, True)])
def test_gated_activation(rows, ff, recompute, dtype, act):
    mx.check_glu(ops, rows, ff, 19, act, dtype, recompute, dev)


@pytest.mark.parametrize("act", ["geglu", "swiglu"])
def test_gated_activation_against_differences(act):
    """The backward pass against central differences of the forward pass at the checkpoint's values (float32)."""
    h = seeded((4, 64), 31)
    _, h8 = ops.glu_forward_mx8(h.cuda(), act)
    hv, d = ops.mx_dequantize(h8, torch.float32), seeded((4, 32), 32).cuda()
    dh = ops.glu_backward_mx8(h8, d, act)
    eps = 2.0 ** -6
    for col in (0, 15, 16, 31, 40, 63):
        e = torch.zeros_like(hv)
        e[:, col] = eps
        f = [(ops.glu_forward_mx8(hv + s * e, act)[0].double() * d.double()).sum(dim=1) for s in (1, -1)]
        diff = (f[0] - f[1]) / (2 * eps)
        # third derivative of a factor |a'''| <= 3, |v|, |d| <= 5: eps^2 / 6 * 75; rounding 2^-23 * 32 sums * 25 / eps
        assert float((dh[:, col].double() - diff).abs().max()) <= eps ** 2 / 6 * 75 + 2.0 ** -23 * 32 * 25 / eps


@pytest.mark.parametrize("rows,n,k,acc", [(1, 8, 1, False), (33, 16, 40, True), (70, 264, 300, False), (154, 1290, 765, False), (97, 56, 320, True),
                                          (4097, 24, 40, False), (4096, 640, 320, True), (1000, 320, 640, False), (8192, 1280, 96, False)])
def test_weight_gradient(rows, n, k, acc):
    mx.check_wgrad(ops, rows, n, k, 23, dev, accumulate=acc)


@pytest.mark.parametrize("rows", [700, 2900, 5200])
def test_weight_gradient_of_many_splits(rows):
    """Two, eleven and twenty ranges of rows, added up by the second kernel."""
    mx.check_wgrad(ops, rows, 24, 40, 24, dev, accumulate=rows == 2900)


def test_gradients_of_rows_at_any_alignment():
    x, flat = mx.activations(100, 72, 3), seeded((1 + 100 * 40,), 4).to(bf)
    off, dy = flat.cuda()[1:].view(100, 40), flat[1:].view(100, 40)
    assert off.data_ptr() % 16
    x8, w = ops.mx8_quantize(x.cuda()), ops.mx4_quantize(seeded((40, 72), 5).cuda())
    assert same_bits(ops.linear_wgrad_mx8(x8, off), ops.linear_wgrad_mx8(x8, dy.cuda()))
    first = seeded((40, 72), 6).cuda()
    a, b = first.clone(), first.clone()
    ops.linear_wgrad_mx8(x8, off, out=a)
    ops.linear_wgrad_mx8(x8, dy.cuda(), out=b)
    # sums of both take the first values in at another place: half a float32 step of it and of the sum each
    assert float((a - b).abs().max()) <= 2.0 ** -23 * float(b.abs().max() + first.abs().max())
    assert same_bits(ops.mx4_linear_dgrad(off, w), ops.mx4_linear_dgrad(dy.cuda(), w))


def test_repeated_calls_give_the_same_bits():
    x, dy = mx.activations(4096, 320, 1).cuda(), seeded((4096, 640), 2).to(bf).cuda()
    w = ops.mx4_quantize(seeded((640, 320), 3).cuda())
    runs = []
    for _ in range(3):
        x8 = ops.mx8_quantize(x)
        runs.append((ops.linear_wgrad_mx8(x8, dy), ops.mx4_linear(ops.mx4_quantize(x), w), ops.mx4_linear(x[:3], w), ops.mx4_linear_dgrad(dy, w)))
    for other in runs[1:]:
        assert all(same_bits(a, b) for a, b in zip(runs[0], other))


def _fine_tuning_step(x, dout, w1, w2, b1, act):
    """A gated feed-forward of two frozen 4-bit layers in training: what a fine-tuning step keeps of it is the 8-bit checkpoint of
    the pre-activation and of the input; returns the output, the input's gradient and the dense weight gradients that adapters of either
    layer are trained with."""
    x8 = ops.mx8_quantize(x)
    h = ops.mx4_linear(ops.mx4_quantize(x), w1, bias=b1)
    y, h8 = ops.glu_forward_mx8(h, act)
    out = ops.mx4_linear(ops.mx4_quantize(y), w2)
    dy = ops.mx4_linear_dgrad(dout, w2)
    dh, again = ops.glu_backward_mx8(h8, dy, act, recompute=True)
    dw2 = ops.linear_wgrad_mx8(ops.mx8_quantize(again), dout)
    dw1 = ops.linear_wgrad_mx8(x8, dh)
    dx = ops.mx4_linear_dgrad(dh, w1)
    return out, dx, dw1, dw2


def _step_inputs(seed, rows=300, c=320, ff=640):
    x, dout = seeded((rows, c), seed).to(bf).cuda(), seeded((rows, c), seed + 1).to(bf).cuda()
    return x, dout


def _step_weights(c=320, ff=640):
    w1, w2 = seeded((2 * ff, c), 71) / math.sqrt(c), seeded((c, ff), 72) / math.sqrt(ff)
    return w1, w2, seeded((2 * ff,), 73)


def test_fine_tuning_step_together():
    """Against float64 with the same roundings at the same places (formats and bfloat16 tensors between the operators): each output's
    error is that of its last operator on inputs that are equal up to bfloat16 steps of the ones before."""
    w1, w2, b1 = _step_weights()
    x, dout = _step_inputs(5)
    out, dx, dw1, dw2 = _fine_tuning_step(x, dout, ops.mx4_quantize(w1.cuda()), ops.mx4_quantize(w2.cuda()), b1.cuda(), "geglu")
    q4 = lambda t: mx_ref.quantize(t, 4)[2]                      # noqa: E731
    q8 = lambda t: mx_ref.quantize(t, 8)[2]                      # noqa: E731
    xd, dd, w1v, w2v = x.cpu(), dout.cpu().double(), q4(w1), q4(w2)
    h = (q4(xd) @ w1v.t() + b1.double()).to(bf)
    y = mx_ref.glu(h.double(), "geglu").to(bf)
    want_out = q4(y) @ w2v.t()
    dy = (dd @ w2v).to(bf).double()
    hv = q8(h)
    dh = mx_ref.glu_backward(hv, dy, "geglu").to(bf).double()
    again = mx_ref.glu(hv, "geglu").to(bf)
    # a bfloat16 tensor between two operators may differ by one step (2^-7) where a sum lands next to a rounding border; a 4-bit element
    # by one of its steps (2^-1) then.  Both happen to few elements: bound the norms with 1 % of them moved.
    def near(a, b, rel):
        assert float((a.cpu().double() - b).norm()) <= rel * float(b.norm())

    near(out, want_out, 2.0 ** -8 + 0.1 * 2.0 ** -1)
    near(dx, dh @ w1v, 2.0 ** -8 + 2.0 ** -7)
    near(dw1, dh.t() @ q8(xd), 2.0 ** -8)
    near(dw2, dd.t() @ q8(again), 2.0 ** -8)


def test_captured_step_replays_on_new_inputs():
    w1, w2, b1 = _step_weights()
    w1q, w2q, b1 = ops.mx4_quantize(w1.cuda()), ops.mx4_quantize(w2.cuda()), b1.cuda()
    x, dout = _step_inputs(5)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _fine_tuning_step(x, dout, w1q, w2q, b1, "swiglu")
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = _fine_tuning_step(x, dout, w1q, w2q, b1, "swiglu")
    for seed in (5, 21, 43, 5):
        nx, nd = _step_inputs(seed)
        x.copy_(nx)
        dout.copy_(nd)
        graph.replay()
        torch.cuda.synchronize()
        eager = _fine_tuning_step(nx, nd, w1q, w2q, b1, "swiglu")
        assert all(same_bits(a, b) for a, b in zip(captured, eager)), seed


def test_single_token_product_captured():
    w = ops.mx4_quantize(seeded((1280, 320), 3).cuda())
    x = seeded((1, 320), 4).to(bf).cuda()
    ops.mx4_linear(x, w)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = ops.mx4_linear(x, w)
        yq = ops.mx4_linear(ops.mx4_quantize(x), w)
    for seed in (1, 2, 3):
        x.copy_(seeded((1, 320), seed).to(bf))
        graph.replay()
        torch.cuda.synchronize()
        assert same_bits(y, ops.mx4_linear(x, w)) and same_bits(yq, ops.mx4_linear(ops.mx4_quantize(x), w))


def test_two_streams_at_once():
    """The same operators on two streams without synchronisation between them: workspaces are per stream."""
    w1, w2, b1 = _step_weights()
    w1q, w2q, b1 = ops.mx4_quantize(w1.cuda()), ops.mx4_quantize(w2.cuda()), b1.cuda()
    ins = [_step_inputs(s, rows=1500) for s in (5, 6)]
    want = [_fine_tuning_step(*i, w1q, w2q, b1, "geglu") for i in ins]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in ins]
    got = [None, None]
    for _ in range(3):
        for j, (st, i) in enumerate(zip(streams, ins)):
            with torch.cuda.stream(st):
                got[j] = _fine_tuning_step(*i, w1q, w2q, b1, "geglu")
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert all(same_bits(u, v) for u, v in zip(a, b))


def test_offsets_past_32_bits():
    """Matrices of more than 2^31 elements: the rows behind that border."""
    rows, cols = (1 << 20) + 5, 2080
    x = torch.zeros(rows, cols, dtype=bf, device="cuda")
    tail = mx.activations(7, cols, 5)
    x[-7:] = tail.cuda()
    for bits, quantize in ((4, ops.mx4_quantize), (8, ops.mx8_quantize)):
        q = quantize(x)
        assert torch.equal(ops.mx_dequantize(q, bf)[-7:].cpu().double(), mx_ref.quantize(tail, bits)[2])
        assert not q.data[:-7].any()
        if bits == 4:
            xq = q
    w = seeded((2080, 64), 6) / 8
    a = ops.MxTensor(xq.data[:, :32].contiguous(), torch.nn.functional.pad(xq.scale[:, :2], (0, 2)), 64)
    y = ops.mx4_linear(a, ops.mx4_quantize(w.cuda()))                                     # (2^20 + 5) x 2080 outputs
    assert mx.product_error(y[-7:], mx_ref.quantize(tail, 4)[2][:, :64], mx_ref.quantize(w, 4)[2]) <= 0
    assert not y[:-7].any()
    del y, a, xq, q
    x8 = ops.mx8_quantize(x[:, :64])
    dw = ops.linear_wgrad_mx8(x8, x)                                                      # dy = x: zero rows but the last
    want = tail.double().t() @ mx_ref.quantize(tail[:, :64], 8)[2]
    size = tail.double().abs().t() @ mx_ref.quantize(tail[:, :64], 8)[2].abs()
    assert float(((dw.cpu().double() - want).abs() - 71 * 2.0 ** -23 * size).max()) <= 0


def test_rows_behind_the_last_stay_as_they_were():
    """Outputs given as the front of a longer buffer through the C entries: nothing is written behind them."""
    from ldm import _lib
    lib = _lib.load()
    x = mx.activations(37, 72, 8).cuda()
    data, scale = torch.full((40, 48), 77, dtype=torch.uint8, device="cuda"), torch.full((40, 4), 77, dtype=torch.uint8, device="cuda")
    st = torch.cuda.current_stream().cuda_stream
    _lib.check(lib.ldm_mx_quantize(x.data_ptr(), 1, 37, 72, 72, 4, data.data_ptr(), scale.data_ptr(), st))
    y = torch.full((40, 130), 5.0, dtype=bf, device="cuda")
    w = ops.mx4_quantize(seeded((130, 72), 9).cuda())
    _lib.check(lib.ldm_mx4_linear(data.data_ptr(), scale.data_ptr(), w.data.data_ptr(), w.scale.data_ptr(), 0, y.data_ptr(), 1, 37, 130, 72, st))
    big = torch.full((140, 130), 5.0, dtype=bf, device="cuda")
    xb = ops.mx4_quantize(mx.activations(133, 72, 8).cuda())
    _lib.check(lib.ldm_mx4_linear(xb.data.data_ptr(), xb.scale.data_ptr(), w.data.data_ptr(), w.scale.data_ptr(), 0, big.data_ptr(), 1, 133, 130, 72, st))
    torch.cuda.synchronize()
    assert (data[37:] == 77).all() and (scale[37:] == 77).all() and (y[37:] == 5.0).all() and (big[133:] == 5.0).all()
