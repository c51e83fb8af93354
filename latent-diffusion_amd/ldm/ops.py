"""Thin torch-tensor front ends of the C-ABI kernels (include/ldm_amd.h).

torch supplies device memory and the current HIP stream; every computation below happens in libldm_amd.so.
Activations are NHWC: a tensor of shape (B, H, W, C) or (B, L, C), contiguous.
"""
from __future__ import annotations

import ctypes as C
import operator
from typing import Optional

import torch

from . import _lib
from ._lib import BF16, F32, ConvGemmDesc

EPI_BIAS, EPI_ROWVEC, EPI_RESIDUAL, EPI_SILU = _lib.EPI_BIAS, _lib.EPI_ROWVEC, _lib.EPI_RESIDUAL, _lib.EPI_SILU
EPI_GEGLU, EPI_SWIGLU = _lib.EPI_GEGLU, _lib.EPI_SWIGLU


def dt_code(dtype: torch.dtype) -> int:
    if dtype == torch.float32:
        return F32
    if dtype == torch.bfloat16:
        return BF16
    raise TypeError(f"unsupported dtype {dtype} (float32 or bfloat16)")


def _gpu(*ts):
    for t in ts:
        if t is not None and not t.is_cuda:
            raise RuntimeError("ldm_amd: tensors must live on an AMD GPU (there is no CPU fallback)")


def _stream(t: torch.Tensor) -> int:
    # the raw handle: 0.1 us a call against 2 us for building torch.cuda.current_stream(t.device) around it
    return torch._C._cuda_getCurrentRawStream(t.get_device())


def _ptr(t: Optional[torch.Tensor]) -> int:
    return 0 if t is None else t.data_ptr()


# The kernels read their side operands (norm affine parameters, biases, raw filters, statistics) as dense float32 arrays of a
# length implied by the other arguments, and their activations in ONE dtype.  A tensor of another dtype or length would be read
# past its end (round 2's GPU fault: a bf16 bias read as float32), so every front end checks before it hands out a pointer.
def _f32_dense(what: str, t: Optional[torch.Tensor], numel: int) -> None:
    if t is None:
        return
    if t.dtype != torch.float32 or t.numel() != numel or not t.is_contiguous():
        raise TypeError(f"{what} must be a contiguous float32 tensor of {numel} elements "
                        f"(got {t.dtype}, shape {tuple(t.shape)}, contiguous={t.is_contiguous()})")


def _same_dtype_dense(what: str, ref: torch.Tensor, *others: Optional[torch.Tensor]) -> None:
    if not ref.is_contiguous():
        raise ValueError(f"{what}: operands must be contiguous")
    for t in others:
        if t is None:
            continue
        if t.dtype != ref.dtype:
            raise TypeError(f"{what}: operands must share one dtype (got {ref.dtype} and {t.dtype})")
        if not t.is_contiguous():
            raise ValueError(f"{what}: operands must be contiguous")


def _rows3(what: str, t: torch.Tensor, dtype: torch.dtype, batch: int, rows: int, cols: int) -> None:
    """A (B, L, C) operand of the attention kernels: unit column stride, rows `stride(1)` apart, samples L rows apart (a dense
    tensor or a column slice of one, e.g. q / k|v inside the fused q|k|v buffer)."""
    if t.dtype != dtype:
        raise TypeError(f"{what}: dtype {t.dtype} does not match the query's {dtype}")
    if t.dim() != 3 or tuple(t.shape) != (batch, rows, cols):
        raise ValueError(f"{what}: expected shape {(batch, rows, cols)}, got {tuple(t.shape)}")
    if t.numel() and (t.stride(2) != 1 or t.stride(1) < cols or (batch > 1 and t.stride(0) != rows * t.stride(1))):
        raise ValueError(f"{what}: must be a row-strided (B, L, C) view with unit column stride (strides {t.stride()})")


def pack_weight(w: torch.Tensor, dtype: torch.dtype, glu_pairs: bool = False, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """float32 [O, I, kh, kw] or [O, I]  ->  [O', kh*kw*I] K-contiguous filter in `dtype` (into `out` when given)."""
    _gpu(w, out)
    w = w.detach().to(torch.float32).contiguous()
    if w.dim() == 2:
        o, i, kh, kw = w.shape[0], w.shape[1], 1, 1
    elif w.dim() == 1:
        o, i, kh, kw = w.shape[0], 1, 1, 1
    else:
        o, i, kh, kw = w.shape
    if out is None:
        out = torch.empty((o, kh * kw * i), dtype=dtype, device=w.device)
    elif out.dtype != dtype or out.numel() != o * kh * kw * i or not out.is_contiguous():
        raise ValueError("pack_weight: out must be a contiguous tensor of the packed size and dtype")
    with torch.cuda.device(w.device):
        _lib.check(_lib.load().ldm_pack_weight(w.data_ptr(), out.data_ptr(), dt_code(dtype), o, i, kh, kw,
                                               1 if glu_pairs else 0, _stream(w)), "ldm_pack_weight")
    return out


def pack_weight_pair(w: torch.Tensor, dtype: torch.dtype, *, glu_pairs: bool = False, fwd: Optional[torch.Tensor] = None,
                     dgrad: Optional[torch.Tensor] = None, want_dgrad: bool = True):
    """One pass over a float32 checkpoint filter [O, I, kh, kw] / [O, I] -> (fwd [O', kh*kw*I], dgrad [kh*kw*I, O'] with the
    taps rotated: the filter of the input-gradient pass).  ``fwd`` / ``dgrad`` may be row / column ranges of fused
    buffers (q|k|v, the time projections): fwd a contiguous row range, dgrad a column range (its row pitch is kept)."""
    _gpu(w, fwd, dgrad)
    w = w.detach()
    if w.dtype != torch.float32 or not w.is_contiguous():
        w = w.to(torch.float32).contiguous()
    if w.dim() == 2:
        o, i, kh, kw = w.shape[0], w.shape[1], 1, 1
    else:
        o, i, kh, kw = w.shape
    k = kh * kw * i
    if fwd is None:
        fwd = torch.empty((o, k), dtype=dtype, device=w.device)
    if dgrad is None and want_dgrad:
        dgrad = torch.empty((k, o), dtype=dtype, device=w.device)
    if fwd.shape != (o, k) or not fwd.is_contiguous() or fwd.dtype != dtype:
        raise ValueError("pack_weight_pair: fwd must be a contiguous (O, K) row range in the packed dtype")
    ld = 0
    if dgrad is not None:
        if dgrad.shape != (k, o) or dgrad.stride(1) != 1 or dgrad.dtype != dtype:
            raise ValueError("pack_weight_pair: dgrad must be a (K, O) column range with unit column stride")
        ld = dgrad.stride(0)
    with torch.cuda.device(w.device):
        _lib.check(_lib.load().ldm_pack_weight_pair(w.data_ptr(), fwd.data_ptr(), _ptr(dgrad), dt_code(dtype), o, i, kh, kw,
                                                    1 if glu_pairs else 0, ld, _stream(w)), "ldm_pack_weight_pair")
    if dgrad is not None and dgrad.is_contiguous():
        dgrad = dgrad.view(i, kh * kw * o)          # the K-contiguous filter of the dgrad GEMM: N = Cin, K = taps * Cout
    return fwd, dgrad


class PackPlan:
    """The repack of MANY filters as one launch per tap count (ldm_pack_weight_pair_batch): the training step rebuilds every
    derived filter after each optimizer step, ~250 of them.  ``jobs``: (w float32 checkpoint filter, fwd (O, K) row range,
    dgrad (K, O) column range or None, glu_pairs).  The destinations are kept and rewritten in place by every ``run()``; jobs
    the batch kernel does not take (float32 destinations, dimensions that are not multiples of 4) go through
    pack_weight_pair one by one."""

    def __init__(self, jobs, dtype: torch.dtype):
        self.dtype = dtype
        self.single = []
        self.groups = {}                       # taps -> (device job table, njobs, total blocks)
        self._keep = []                        # the tensors the device tables point into
        by_taps = {1: [], 9: []}
        for w, fwd, dgrad, glu in jobs:
            _gpu(w, fwd, dgrad)
            wd = w.detach()
            o, i = wd.shape[0], wd.shape[1]
            taps = 1 if wd.dim() == 2 else wd.shape[2] * wd.shape[3]
            k = taps * i
            ld = 0 if dgrad is None else dgrad.stride(0)
            ok = (dtype == torch.bfloat16 and wd.dtype == torch.float32 and wd.is_contiguous() and taps in by_taps
                  and o % 4 == 0 and i % 4 == 0 and ld % 4 == 0 and fwd.data_ptr() % 8 == 0
                  and (dgrad is None or dgrad.data_ptr() % 8 == 0) and (not glu or o % 32 == 0))
            if fwd.shape != (o, k) or not fwd.is_contiguous() or fwd.dtype != dtype:
                raise ValueError("PackPlan: fwd must be a contiguous (O, K) row range in the packed dtype")
            if dgrad is not None and (dgrad.shape != (k, o) or dgrad.stride(1) != 1 or dgrad.dtype != dtype):
                raise ValueError("PackPlan: dgrad must be a (K, O) column range with unit column stride")
            self._keep.append((w, fwd, dgrad))
            if ok:
                by_taps[taps].append((wd, fwd, dgrad, glu, o, i, ld))
            else:
                self.single.append((w, fwd, dgrad, glu))
        for taps, lst in by_taps.items():
            if not lst:
                continue
            arr = (_lib.PackJob * len(lst))()
            first = 0
            for n, (wd, fwd, dgrad, glu, o, i, ld) in enumerate(lst):
                bx, by = (o + 31) // 32, (i + 31) // 32
                arr[n] = _lib.PackJob(src=wd.data_ptr(), fwd=fwd.data_ptr(), dgrad=_ptr(dgrad), dgrad_ld=ld, cout=o, cin=i,
                                      glu_pairs=1 if glu else 0, blocks_x=bx, blocks_y=by, first_block=first)
                first += bx * by
            host = torch.frombuffer(bytearray(bytes(arr)), dtype=torch.uint8)
            table = host.to(lst[0][0].device)
            self.groups[taps] = (table, len(lst), first)
        self.sources = tuple(w.data_ptr() for w, _, _ in self._keep)

    def run(self):
        lib = _lib.load()
        for taps, (table, n, blocks) in self.groups.items():
            with torch.cuda.device(table.device):
                _lib.check(lib.ldm_pack_weight_pair_batch(table.data_ptr(), n, blocks, taps,
                                                          torch.cuda.current_stream(table.device).cuda_stream),
                           "ldm_pack_weight_pair_batch")
        for w, fwd, dgrad, glu in self.single:
            pack_weight_pair(w, self.dtype, glu_pairs=glu, fwd=fwd, dgrad=dgrad, want_dgrad=dgrad is not None)

    def still_valid(self) -> bool:
        """The checkpoint tensors the device tables point at have not moved (optimizers update parameters in place)."""
        return self.sources == tuple(w.data_ptr() for w, _, _ in self._keep)


def conv_gemm(a0: torch.Tensor, w: torch.Tensor, *, a1: Optional[torch.Tensor] = None, ksize: int = 1, stride: int = 1,
              upsample: bool = False, bias: Optional[torch.Tensor] = None, rowvec: Optional[torch.Tensor] = None,
              residual: Optional[torch.Tensor] = None, silu: bool = False, glu: Optional[str] = None,
              out_dtype: Optional[torch.dtype] = None, out_hw=None, rowstats: bool = False, ln=None,
              glu_preact: bool = False):
    """Implicit-GEMM conv / linear.  a0 (and a1): (B, H, W, C) NHWC, or (..., C) matrices for ksize == 1.
    w: packed [N, ksize*ksize*(C0+C1)].  Returns NHWC (B, Hout, Wout, N') / (..., N').
    upsample: False, True (nearest 2x, unet.py:316) or "zero" (zero-insertion 2x: input gradient of a stride-2 conv).
    LayerNorm fold (bf16; include/ldm_amd.h LDM_EPI_ROWSTATS / LDM_EPI_LNFOLD): ``rowstats=True`` returns (out, stats) with
    stats (M, N / 80, 2) float32 = per-row partial (sum, sumsq) of the output; ``ln=(stats, colsum, eps)`` treats a0 as the
    INPUT of a LayerNorm whose statistics are ``stats``: w must be the gamma-scaled filter, colsum its row sums, and bias
    must already contain W beta (``fold_layernorm`` builds the three).
    ``glu_preact=True`` (GLU epilogues, bf16): returns (out, pre) with pre (..., N) the biased pre-activation in the filter's
    paired column order -- what the training forward keeps for ``glu_backward``."""
    _gpu(a0, a1, w, bias, rowvec, residual)
    if not a0.is_contiguous() or (a1 is not None and not a1.is_contiguous()):
        raise ValueError("conv_gemm: activations must be contiguous NHWC")
    c0 = a0.shape[-1]
    c1 = 0 if a1 is None else a1.shape[-1]
    if ksize == 1 and not upsample and stride == 1:
        lead = a0.shape[:-1]
        rows = a0.numel() // c0
        batch, hin, win = rows, 1, 1
        if rowvec is not None:  # per-sample vector: keep the sample structure
            batch = a0.shape[0]
            hin, win = rows // batch, 1
        hout, wout = hin, win
        out_lead = lead
    else:
        if a0.dim() != 4:
            raise ValueError("conv_gemm: 3x3 / strided / upsampled convs take (B, H, W, C) inputs")
        batch, hin, win = a0.shape[0], a0.shape[1], a0.shape[2]
        hs, ws = (2 * hin, 2 * win) if upsample else (hin, win)
        pad = ksize // 2
        hout = (hs + 2 * pad - ksize) // stride + 1
        wout = (ws + 2 * pad - ksize) // stride + 1
        if out_hw is not None:      # zero insertion: the forward input may have had an odd extent
            hout, wout = out_hw
        out_lead = (batch, hout, wout)
    if a1 is not None and a1.shape[:-1] != a0.shape[:-1]:
        raise ValueError("conv_gemm: the two sources must agree in all but the channel dimension")
    n = w.shape[0]
    if w.shape[1] != ksize * ksize * (c0 + c1):
        raise ValueError(f"conv_gemm: filter K={w.shape[1]} does not match {ksize}x{ksize}x({c0}+{c1})")
    epi = 0
    if bias is not None:
        epi |= EPI_BIAS
    if rowvec is not None:
        epi |= EPI_ROWVEC
    if residual is not None:
        epi |= EPI_RESIDUAL
    if silu:
        epi |= EPI_SILU
    if glu == "geglu":
        epi |= EPI_GEGLU
    elif glu == "swiglu":
        epi |= EPI_SWIGLU
    elif glu is not None:
        raise ValueError(f"Unsupported activation function: {glu}")
    if bias is not None and (bias.dtype != torch.float32 or bias.numel() != n or not bias.is_contiguous()):
        raise TypeError(f"conv_gemm: bias must be a contiguous float32 vector of {n} elements (got {bias.dtype}, {tuple(bias.shape)})")
    for name_, t_ in (("rowvec", rowvec), ("residual", residual), ("a1", a1), ("w", w)):
        if t_ is not None and t_.dtype != a0.dtype:
            raise TypeError(f"conv_gemm: {name_} must have the activation dtype {a0.dtype} (got {t_.dtype})")
    if w.dim() != 2 or not w.is_contiguous():
        raise ValueError("conv_gemm: the packed filter must be a contiguous (N, K) matrix")
    if residual is not None and (not residual.is_contiguous() or residual.numel() != batch * hout * wout * n or glu):
        raise ValueError(f"conv_gemm: residual must be a contiguous tensor of the output's {batch * hout * wout} x {n} elements (no GLU)")
    if rowvec is not None and (rowvec.dim() != 2 or rowvec.shape != (batch, n) or rowvec.stride(1) != 1):
        raise ValueError(f"conv_gemm: rowvec must be a (batch, N) = ({batch}, {n}) view with unit column stride, got {tuple(rowvec.shape)}")
    odt = out_dtype or a0.dtype
    nout = n // 2 if glu else n
    out = torch.empty((*out_lead, nout), dtype=odt, device=a0.device)
    d = ConvGemmDesc(a0=a0.data_ptr(), a1=_ptr(a1), c0=c0, c1=c1, batch=batch, hin=hin, win=win, hout=hout, wout=wout,
                     ksize=ksize, stride=stride, upsample=(2 if upsample == "zero" else 1 if upsample else 0), w=w.data_ptr(), n=n, epilogue=epi,
                     bias=_ptr(bias), rowvec=_ptr(rowvec), rowvec_stride=0 if rowvec is None else rowvec.stride(0),
                     residual=_ptr(residual), out=out.data_ptr(), dtype=dt_code(a0.dtype), out_dtype=dt_code(odt))
    pre = None
    if glu_preact:
        if not glu or a0.dtype != torch.bfloat16 or odt != torch.bfloat16 or n % 32:
            raise ValueError("conv_gemm(glu_preact=True): GLU epilogue, bf16 in and out, N a multiple of 32")
        pre = torch.empty((*out_lead, n), dtype=odt, device=a0.device)
        d.glu_preact = pre.data_ptr()
    stats = None
    if rowstats:
        if n % 160 or (c0 + c1) % 64 or c0 % 64 or a0.dtype != torch.bfloat16 or glu or odt != torch.bfloat16:
            raise ValueError("conv_gemm(rowstats=True): bf16 in and out, no GLU, N a multiple of 160, channels multiples of 64")
        stats = torch.empty((batch * hout * wout, n // 80, 2), dtype=torch.float32, device=a0.device)
        d.epilogue |= _lib.EPI_ROWSTATS
        d.rowstats = stats.data_ptr()
    if ln is not None:
        ln_stats, ln_colsum, ln_eps = ln
        _gpu(ln_stats, ln_colsum)
        if ln_stats.dtype != torch.float32 or ln_stats.dim() != 3 or ln_stats.shape[0] != batch * hout * wout or \
                ln_stats.shape[2] != 2 or not ln_stats.is_contiguous():
            raise ValueError("conv_gemm(ln=...): stats must be contiguous float32 (M, segments, 2)")
        if ln_stats.shape[1] * 80 != c0 or c1 or ksize != 1:
            raise ValueError(f"conv_gemm(ln=...): {ln_stats.shape[1]} statistics segments of 80 columns do not cover the {c0} "
                             "channels of a0 (the statistics must come from the GEMM that wrote a0)")
        _f32_dense("conv_gemm(ln=...): colsum", ln_colsum, n)
        d.epilogue |= _lib.EPI_LNFOLD
        d.ln_stats, d.ln_colsum, d.ln_segments, d.ln_eps = ln_stats.data_ptr(), ln_colsum.data_ptr(), ln_stats.shape[1], float(ln_eps)
    if a0.dtype == torch.bfloat16 and batch * hout * wout <= _SPLITK_MAX_ROWS and not rowstats and ln is None:
        ws = _splitk_workspace(a0.device)   # small-M layers may split K; ordered by the current stream like `out`
        d.workspace, d.workspace_bytes = ws.data_ptr(), ws.numel() * 4
    with torch.cuda.device(a0.device):
        if _launch_log is None:
            _lib.check(_lib.load().ldm_conv_gemm(C.byref(d), _stream(a0)), "ldm_conv_gemm")
        else:  # bench.py: bracket the launch with HIP events on the stream it runs on
            tile = (C.c_int * 3)()
            _lib.check(_lib.load().ldm_conv_gemm_tile(C.byref(d), tile), "ldm_conv_gemm_tile")
            e0, e1 = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            e0.record()
            _lib.check(_lib.load().ldm_conv_gemm(C.byref(d), _stream(a0)), "ldm_conv_gemm")
            e1.record()
            m = batch * hout * wout
            _launch_log.append((f"conv_gemm_{'bf16' if a0.dtype == torch.bfloat16 else 'f32'}_kernel<{tile[0]},{tile[1]},{tile[2]}>",
                                2.0 * m * n * ksize * ksize * (c0 + c1), e0, e1,
                                (m, n, ksize * ksize * (c0 + c1), ksize, stride, int(bool(upsample)), c1, epi)))
    if glu_preact:
        return out, pre
    return (out, stats) if rowstats else out


def ln_fold_supported(channels: int, dtype: torch.dtype) -> bool:
    """The LayerNorm fold needs bf16 and a producer whose rows are whole 80-column wave tiles of BN = 160, BK = 64 GEMM
    tiles: channel counts in multiples of lcm(160, 64) = 320 (320 / 640 / 1280 in the SD-1.5-shaped model)."""
    return dtype == torch.bfloat16 and channels % 320 == 0 and channels <= 1280   # <= 16 statistics segments per row


def fold_layernorm_terms(w: torch.Tensor, bias: Optional[torch.Tensor], gamma: torch.Tensor, beta: torch.Tensor, dtype: torch.dtype):
    """Pure torch (any device; tests/test_ln_fold_cpu.py): the three tensors of the identity
        LayerNorm(x) W^T + bias  ==  rstd (x W'^T - mean * colsum) + bias'
    W' = W * gamma [N, K] float32 (to be rounded to ``dtype`` by the packer), colsum[n] = sum_k round(W')[n][k], bias' =
    bias + W beta, float32."""
    with torch.autocast(w.device.type, enabled=False):   # packing may run inside the caller's bf16 autocast region: keep float32
        w32 = w.detach().to(torch.float32)
        ws = w32 * gamma.detach().to(torch.float32)[None, :]
        colsum = ws.to(dtype).to(torch.float32).sum(dim=1)        # of the ROUNDED filter: what the matrix core multiplies with
        b2 = (w32 * beta.detach().to(torch.float32)[None, :]).sum(dim=1)
        if bias is not None:
            b2 = b2 + bias.detach().to(torch.float32)
    assert ws.dtype == colsum.dtype == b2.dtype == torch.float32
    return ws, colsum, b2


def fold_layernorm(w: torch.Tensor, bias: Optional[torch.Tensor], gamma: torch.Tensor, beta: torch.Tensor, dtype: torch.dtype,
                   glu_pairs: bool = False):
    """(packed filter, colsum, bias) of the GEMM  LayerNorm(x) W^T + bias  rewritten on x itself (``fold_layernorm_terms``);
    w: float32 [N, K] checkpoint filter; glu_pairs: interleave value / gate rows in blocks of 16 as
    ``pack_weight(glu_pairs=True)`` does (colsum and bias' in the same order)."""
    ws, colsum, b2 = fold_layernorm_terms(w, bias, gamma, beta, dtype)
    wp = pack_weight(ws, dtype, glu_pairs=glu_pairs)
    if glu_pairs:
        colsum = pack_weight(colsum, torch.float32, glu_pairs=True).flatten()
        b2 = pack_weight(b2, torch.float32, glu_pairs=True).flatten()
    if colsum.dtype != torch.float32 or b2.dtype != torch.float32 or wp.dtype != dtype:
        raise TypeError("fold_layernorm: packed terms came out in the wrong dtype")
    return wp, colsum.contiguous(), b2.contiguous()


_ln_fold_checked = {}


def ln_fold_selfcheck(device) -> bool:
    """Once per process and device, before the first forward that would use the LayerNorm fold: the folded chain (producer
    GEMM with row statistics -> consumer GEMM, plain and GEGLU) against the LayerNorm kernel + the plain GEMMs on random data,
    at a row count that selects the LARGE tiles (256x160 for the producer and the q|k|v projection, 128x128 for GEGLU) -- the
    instantiations the benchmarked batch runs and the small parity cases do not.  A mismatch disables the fold for the process
    (the separate LayerNorm kernel runs instead) and says so; it never falls back to anything but another HIP kernel."""
    device = torch.device(device)
    key = device.index if device.index is not None else (torch.cuda.current_device() if device.type == "cuda" else -1)
    if key in _ln_fold_checked:
        return _ln_fold_checked[key]
    if torch.cuda.is_current_stream_capturing():     # no host sync under capture: decide later, run unfused for now
        return False
    import math
    import warnings
    ok, why = False, ""
    try:
        with torch.no_grad(), torch.autocast("cuda", enabled=False), torch.cuda.device(device):
            g = torch.Generator(device=device).manual_seed(20251111)
            M, Cc = 32768, 320
            bf = torch.bfloat16

            def rnd(*shape):
                return torch.randn(*shape, device=device, generator=g)

            a, res = rnd(M, Cc).to(bf), (rnd(M, Cc) * 0.5 + 0.25).to(bf)
            wp, bp = pack_weight(rnd(Cc, Cc) / math.sqrt(Cc), bf), rnd(Cc)
            x, st = conv_gemm(a, wp, bias=bp, residual=res, rowstats=True)
            x0 = conv_gemm(a, wp, bias=bp, residual=res)
            errs = [float((x.float() - x0.float()).norm() / x0.float().norm())]
            tot = st.sum(dim=1)
            errs.append(float((tot[:, 0] - x.float().sum(dim=1)).abs().max()) / 50.0)     # sums of 320 O(1) values: 1e-2 scale
            gamma, beta = 1 + 0.1 * rnd(Cc), 0.1 * rnd(Cc)
            for N, glu in ((3 * Cc, None), (8 * Cc, "geglu")):
                w, b = rnd(N, Cc) / math.sqrt(Cc), rnd(N)
                wf, cs, b2 = fold_layernorm(w, b, gamma, beta, bf, glu_pairs=bool(glu))
                y = conv_gemm(x, wf, bias=b2, glu=glu, ln=(st, cs, 1e-5))
                b0 = pack_weight(b, torch.float32, glu_pairs=True).flatten() if glu else b
                y0 = conv_gemm(layernorm(x, gamma, beta), pack_weight(w, bf, glu_pairs=bool(glu)), bias=b0, glu=glu)
                errs.append(float((y.float() - y0.float()).norm() / y0.float().norm()))
            ok = all(e == e and e < 1.5e-2 for e in errs)
            why = "relative differences " + ", ".join(f"{e:.2e}" for e in errs)
    except Exception as exc:   # an argument check of the library, an allocation failure: keep the proven path
        why = f"{type(exc).__name__}: {exc}"
    if not ok:
        warnings.warn("ldm_amd: the LayerNorm-fold self-check did not pass (" + why + "); the separate LayerNorm kernel is used "
                      "for this process")
    _ln_fold_checked[key] = ok
    return ok


def pack_weight_dgrad(w: torch.Tensor, dtype: torch.dtype) -> torch.Tensor:
    """Filter of the input-gradient pass: in/out transposed, taps rotated by 180 degrees, then packed K-contiguous
    ([Cin][kh][kw][Cout]) -- so that dX = conv_gemm(dY, this) for a stride-1 conv / linear layer."""
    if w.dim() == 4:
        wd = w.detach().flip(2, 3).transpose(0, 1).contiguous()
    else:
        wd = w.detach().t().contiguous()
    return pack_weight(wd, dtype)


def conv_dgrad(dy: torch.Tensor, wd: torch.Tensor, *, ksize: int = 1, stride: int = 1, upsample: bool = False,
               in_hw=None, residual: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Input gradient of conv_gemm(x, w, ksize, stride, upsample) for all of x's channels (both sources of a concat:
    slice the result).  wd = pack_weight_dgrad(w).  in_hw: spatial extent of x (needed for stride 2).  ``residual`` is
    added to the result (gradient arriving over a skip path)."""
    if ksize == 1 or (stride == 1 and not upsample):
        return conv_gemm(dy, wd, ksize=ksize, residual=residual)
    if stride == 2:
        return conv_gemm(dy, wd, ksize=ksize, upsample="zero", out_hw=in_hw, residual=residual)
    # nearest-2x upsample then conv: gradient at the upsampled extent, then fold every 2x2 block
    du = conv_gemm(dy, wd, ksize=ksize)
    return sum2x2(du, residual=residual)


def sum2x2(x: torch.Tensor, residual: Optional[torch.Tensor] = None) -> torch.Tensor:
    """out[b, h, w, c] = sum of the 2x2 block of x at (2h, 2w): gradient of nearest-2x upsampling (unet.py:316)."""
    _gpu(x, residual)
    B, H, W, Cc = x.shape
    if H % 2 or W % 2 or Cc % 8 or not x.is_contiguous():
        raise ValueError("sum2x2: contiguous (B, even H, even W, C % 8 == 0) input")
    if residual is not None and (residual.dtype != x.dtype or tuple(residual.shape) != (B, H // 2, W // 2, Cc)
                                 or not residual.is_contiguous()):
        raise ValueError("sum2x2: residual must be a contiguous tensor of the output's shape and dtype")
    out = torch.empty((B, H // 2, W // 2, Cc), dtype=x.dtype, device=x.device)
    with torch.cuda.device(x.device):
        _lib.check(_lib.load().ldm_sum2x2(x.data_ptr(), _ptr(residual), out.data_ptr(), dt_code(x.dtype), B, H // 2, W // 2, Cc,
                                          _stream(x)), "ldm_sum2x2")
    return out


def conv_wgrad(a0: torch.Tensor, dy: torch.Tensor, *, a1: Optional[torch.Tensor] = None, ksize: int = 1, stride: int = 1,
               upsample: bool = False, out: Optional[torch.Tensor] = None, accumulate: Optional[bool] = None) -> torch.Tensor:
    """Weight gradient of conv_gemm(a0, w, a1=..., ksize=..., stride=..., upsample=...): float32, checkpoint layout
    ([N, C0+C1, k, k], or [N, C] for ksize == 1 matrices).  ``out``: an existing gradient to accumulate into, or
    (accumulate=False) a buffer to overwrite, e.g. the parameter's slice of a flat gradient bucket."""
    _gpu(a0, a1, dy, out)
    if a0.dtype != dy.dtype or (a1 is not None and a1.dtype != a0.dtype):
        raise TypeError("conv_wgrad: activations and output gradients must share one dtype")
    if not a0.is_contiguous() or not dy.is_contiguous() or (a1 is not None and not a1.is_contiguous()):
        raise ValueError("conv_wgrad: activations and dy must be contiguous")
    c0 = a0.shape[-1]
    c1 = 0 if a1 is None else a1.shape[-1]
    n = dy.shape[-1]
    if ksize == 1 and not upsample and stride == 1:
        rows = a0.numel() // c0
        batch, hin, win, hout, wout = rows, 1, 1, 1, 1
        shape = (n, c0 + c1)
    else:
        if a0.dim() != 4:
            raise ValueError("conv_wgrad: 3x3 / strided / upsampled convs take (B, H, W, C) inputs")
        batch, hin, win = a0.shape[0], a0.shape[1], a0.shape[2]
        hs, ws = (2 * hin, 2 * win) if upsample else (hin, win)
        pad = ksize // 2
        hout = (hs + 2 * pad - ksize) // stride + 1
        wout = (ws + 2 * pad - ksize) // stride + 1
        shape = (n, c0 + c1, ksize, ksize)
    if dy.numel() != batch * hout * wout * n:
        raise ValueError(f"conv_wgrad: dy has {dy.numel()} elements, expected {batch * hout * wout}x{n}")
    if accumulate is None:
        accumulate = out is not None
    if out is None:
        accumulate = False
        out = torch.empty(shape, dtype=torch.float32, device=a0.device)
    elif out.dtype != torch.float32 or tuple(out.shape) != shape or not out.is_contiguous():
        raise ValueError(f"conv_wgrad: out must be a contiguous float32 tensor of shape {shape}")
    d = ConvGemmDesc(a0=a0.data_ptr(), a1=_ptr(a1), c0=c0, c1=c1, batch=batch, hin=hin, win=win, hout=hout, wout=wout,
                     ksize=ksize, stride=stride, upsample=1 if upsample else 0, n=n, dtype=dt_code(a0.dtype),
                     out_dtype=dt_code(a0.dtype))
    lib = _lib.load()
    need = lib.ldm_conv_wgrad_workspace_bytes(C.byref(d))
    ws = _wgrad_workspace(a0.device, need)
    with torch.cuda.device(a0.device):
        if _launch_log is None:
            _lib.check(lib.ldm_conv_wgrad(C.byref(d), dy.data_ptr(), out.data_ptr(), 1 if accumulate else 0, ws.data_ptr(),
                                          ws.numel() * 4, _stream(a0)), "ldm_conv_wgrad")
        else:  # bench.py --train: bracket the launch (kernel + fold) with HIP events on its stream
            e0, e1 = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            e0.record()
            _lib.check(lib.ldm_conv_wgrad(C.byref(d), dy.data_ptr(), out.data_ptr(), 1 if accumulate else 0, ws.data_ptr(),
                                          ws.numel() * 4, _stream(a0)), "ldm_conv_wgrad")
            e1.record()
            m, k = batch * hout * wout, ksize * ksize * (c0 + c1)
            _launch_log.append((f"conv_wgrad_{'bf16' if a0.dtype == torch.bfloat16 else 'f32'}_kernel(+fold)", 2.0 * m * n * k, e0, e1,
                                (m, n, k, ksize, stride, int(bool(upsample)), c1, 0)))
    return out


_wgrad_ws = {}


def _wgrad_workspace(device, nbytes: int) -> torch.Tensor:
    """Per-(device, stream) scratch for the pixel-split partial tiles of ldm_conv_wgrad; grows to the largest layer."""
    key = (device.index, torch.cuda.current_stream(device).cuda_stream)
    ws = _wgrad_ws.get(key)
    if ws is None or ws.numel() * 4 < nbytes:
        ws = _wgrad_ws[key] = torch.empty(max(nbytes // 4 + 1, 1 << 20), dtype=torch.float32, device=device)
    return ws


_launch_log = None

_SPLITK_MAX_ROWS = 4096                 # only layers this small are ever offered the workspace
_SPLITK_WORKSPACE_FLOATS = 16 << 20     # 64 MiB per device: 8 splits of a 2048 x 1280 output
_splitk_ws = {}


def _splitk_workspace(device) -> torch.Tensor:
    """Per-(device, stream) scratch lent to ldm_conv_gemm for split-K partial sums (struct LdmConvGemm.workspace)."""
    key = (device.index, torch.cuda.current_stream(device).cuda_stream)
    ws = _splitk_ws.get(key)
    if ws is None:
        ws = _splitk_ws[key] = torch.empty(_SPLITK_WORKSPACE_FLOATS, dtype=torch.float32, device=device)
    return ws


def set_launch_log(log):
    """bench.py hook: a list that receives (kernel name, algorithmic FLOPs, start event, end event,
    (M, N, K, ksize, stride, upsample, c1, epilogue flags)) per GEMM launch."""
    global _launch_log
    _launch_log = log


_gn_ws = {}


def _gn_workspace(device, batch: int, groups: int) -> torch.Tensor:
    need = _lib.load().ldm_groupnorm_workspace_floats(batch, groups)
    key = (device.index, torch.cuda.current_stream(device).cuda_stream)   # per stream: micro-batches run concurrently
    ws = _gn_ws.get(key)
    if ws is None or ws.numel() < need:
        ws = torch.empty(need, dtype=torch.float32, device=device)
        _gn_ws[key] = ws
    return ws


def _groupnorm_call(a0, gamma, beta, groups, a1, silu, eps):
    _gpu(a0, a1, gamma, beta)
    B = a0.shape[0]
    c0 = a0.shape[-1]
    c1 = 0 if a1 is None else a1.shape[-1]
    _same_dtype_dense("groupnorm", a0, a1)
    if a1 is not None and a1.shape[:-1] != a0.shape[:-1]:
        raise ValueError("groupnorm: the two sources must agree in all but the channel dimension")
    if groups < 1 or (c0 + c1) % groups:
        raise ValueError(f"groupnorm: {c0 + c1} channels do not divide into {groups} groups")
    _f32_dense("groupnorm: gamma", gamma, c0 + c1)
    _f32_dense("groupnorm: beta", beta, c0 + c1)
    hw = a0.numel() // (B * c0) if B else 1
    stats = torch.empty((B, groups, 2), dtype=torch.float32, device=a0.device)
    out = torch.empty((*a0.shape[:-1], c0 + c1), dtype=a0.dtype, device=a0.device)
    lib = _lib.load()
    code = dt_code(a0.dtype)
    with torch.cuda.device(a0.device):
        st = _stream(a0)
        ws = _gn_workspace(a0.device, B, groups)
        _lib.check(lib.ldm_groupnorm(a0.data_ptr(), _ptr(a1), c0, c1, code, B, hw, groups, eps, gamma.data_ptr(),
                                     beta.data_ptr(), 1 if silu else 0, out.data_ptr(), stats.data_ptr(), ws.data_ptr(), st),
                   "ldm_groupnorm")
    return out, stats


def groupnorm(a0: torch.Tensor, gamma: torch.Tensor, beta: torch.Tensor, groups: int, *, a1: Optional[torch.Tensor] = None,
              silu: bool = False, eps: float = 1e-5) -> torch.Tensor:
    """GroupNorm (+SiLU) over NHWC (B, H, W, C) / (B, L, C); two sources are normalised as their channel concat."""
    return _groupnorm_call(a0, gamma, beta, groups, a1, silu, eps)[0]


def groupnorm_with_stats(a0, gamma, beta, groups, *, a1=None, silu=False, eps=1e-5):
    """groupnorm() that also returns the (B, groups, 2) mean/rstd tensor the backward needs."""
    return _groupnorm_call(a0, gamma, beta, groups, a1, silu, eps)


_bwd_ws = {}


def _bwd_workspace(device, nfloats: int) -> torch.Tensor:
    """Per-(device, stream) float32 scratch of the HBM-bound backward kernels; grows to the largest request."""
    key = (device.index, torch.cuda.current_stream(device).cuda_stream)
    ws = _bwd_ws.get(key)
    if ws is None or ws.numel() < nfloats:
        ws = _bwd_ws[key] = torch.empty(max(int(nfloats), 1 << 20), dtype=torch.float32, device=device)
    return ws


def groupnorm_backward(a0, stats, gamma, beta, groups, dy, *, a1=None, silu=False, add=None, dgamma=None, dbeta=None,
                       split=False, accumulate=None):
    """Backward of groupnorm(a0, ..., a1=a1, silu=silu): returns (dx over all c0+c1 channels [+ add], dgamma, dbeta).
    dgamma / dbeta given: accumulated into (float32), or overwritten with accumulate=False.  split (two sources): dx is the pair (dx0 (.., c0), dx1 (.., c1)),
    each dense -- the concat gradient is split where it is produced."""
    _gpu(a0, a1, stats, gamma, beta, dy, add, dgamma, dbeta)
    B = a0.shape[0]
    c0 = a0.shape[-1]
    c1 = 0 if a1 is None else a1.shape[-1]
    hw = a0.numel() // (B * c0) if B else 1
    _same_dtype_dense("groupnorm_backward", a0, a1)
    if not dy.is_contiguous() or dy.shape[-1] != c0 + c1 or dy.dtype != a0.dtype or dy.numel() != B * hw * (c0 + c1):
        raise ValueError("groupnorm_backward: dy must be contiguous (.., c0+c1) in the activation dtype")
    if add is not None and (not add.is_contiguous() or add.shape != dy.shape or add.dtype != dy.dtype):
        raise ValueError("groupnorm_backward: add must be contiguous with dy's shape and dtype")
    _f32_dense("groupnorm_backward: stats", stats, B * groups * 2)
    _f32_dense("groupnorm_backward: gamma", gamma, c0 + c1)
    _f32_dense("groupnorm_backward: beta", beta, c0 + c1)
    _f32_dense("groupnorm_backward: dgamma", dgamma, c0 + c1)
    _f32_dense("groupnorm_backward: dbeta", dbeta, c0 + c1)
    if (dgamma is None) != (dbeta is None):
        raise ValueError("groupnorm_backward: pass both dgamma and dbeta or neither")
    if accumulate is None:
        accumulate = dgamma is not None
    if dgamma is None:
        accumulate = False
        dgamma = torch.empty(c0 + c1, dtype=torch.float32, device=a0.device)
        dbeta = torch.empty(c0 + c1, dtype=torch.float32, device=a0.device)
    if split and a1 is not None:
        dx = torch.empty_like(a0)
        dx1 = torch.empty_like(a1)
    else:
        dx, dx1 = torch.empty_like(dy), None
    lib = _lib.load()
    with torch.cuda.device(a0.device):
        ws = _bwd_workspace(a0.device, lib.ldm_groupnorm_backward_workspace_floats(B, c0 + c1, groups))
        _lib.check(lib.ldm_groupnorm_backward(a0.data_ptr(), _ptr(a1), c0, c1, dt_code(a0.dtype), B, hw, groups, stats.data_ptr(),
                                              gamma.data_ptr(), beta.data_ptr(), 1 if silu else 0, dy.data_ptr(), _ptr(add),
                                              dx.data_ptr(), _ptr(dx1), dgamma.data_ptr(), dbeta.data_ptr(),
                                              1 if accumulate else 0, ws.data_ptr(), _stream(a0)), "ldm_groupnorm_backward")
    return ((dx, dx1) if dx1 is not None else dx), dgamma, dbeta


def layernorm_backward(x, gamma, dy, *, eps: float = 1e-5, add=None, dgamma=None, dbeta=None, accumulate=None):
    """Backward of layernorm(x, gamma, beta): returns (dx [+ add], dgamma, dbeta)."""
    _gpu(x, gamma, dy, add, dgamma, dbeta)
    cols = x.shape[-1]
    rows = x.numel() // cols
    _same_dtype_dense("layernorm_backward", x, dy, add)
    if dy.shape != x.shape or (add is not None and add.shape != x.shape):
        raise ValueError("layernorm_backward: dy (and add) must have x's shape")
    _f32_dense("layernorm_backward: gamma", gamma, cols)
    _f32_dense("layernorm_backward: dgamma", dgamma, cols)
    _f32_dense("layernorm_backward: dbeta", dbeta, cols)
    if (dgamma is None) != (dbeta is None):
        raise ValueError("layernorm_backward: pass both dgamma and dbeta or neither")
    if accumulate is None:
        accumulate = dgamma is not None
    if dgamma is None:
        accumulate = False
        dgamma = torch.empty(cols, dtype=torch.float32, device=x.device)
        dbeta = torch.empty(cols, dtype=torch.float32, device=x.device)
    dx = torch.empty_like(x)
    lib = _lib.load()
    with torch.cuda.device(x.device):
        ws = _bwd_workspace(x.device, lib.ldm_layernorm_backward_workspace_floats(cols))
        _lib.check(lib.ldm_layernorm_backward(x.data_ptr(), dy.data_ptr(), dt_code(x.dtype), rows, cols, eps, gamma.data_ptr(),
                                              _ptr(add), dx.data_ptr(), dgamma.data_ptr(), dbeta.data_ptr(),
                                              1 if accumulate else 0, ws.data_ptr(), _stream(x)), "ldm_layernorm_backward")
    return dx, dgamma, dbeta


def colsum(x: torch.Tensor, segments: int = 1, out: Optional[torch.Tensor] = None, accumulate: Optional[bool] = None) -> torch.Tensor:
    """float32 column sums per segment of consecutive rows: (segments, n).  out given: accumulated into (or overwritten
    with accumulate=False)."""
    _gpu(x, out)
    n = x.shape[-1]
    rows = x.numel() // n
    if rows % segments:
        raise ValueError("colsum: rows not divisible by segments")
    if not x.is_contiguous():
        raise ValueError("colsum: x must be contiguous")
    if accumulate is None:
        accumulate = out is not None
    if out is None:
        accumulate = False
        out = torch.empty((segments, n), dtype=torch.float32, device=x.device)
    elif out.dtype != torch.float32 or out.numel() != segments * n or not out.is_contiguous():
        raise ValueError("colsum: out must be a contiguous float32 tensor of segments * n elements")
    lib = _lib.load()
    with torch.cuda.device(x.device):
        ws = _bwd_workspace(x.device, lib.ldm_colsum_workspace_floats(segments, n))
        _lib.check(lib.ldm_colsum(x.data_ptr(), dt_code(x.dtype), segments, rows // segments, n, out.data_ptr(),
                                  1 if accumulate else 0, ws.data_ptr(), _stream(x)), "ldm_colsum")
    return out


def glu_forward(h: torch.Tensor, act: str) -> torch.Tensor:
    """Training form of GEGLU / SwiGLU: h = packed-order pre-activation (.., 2*ff) -> (.., ff)."""
    _gpu(h)
    ff = h.shape[-1] // 2
    _same_dtype_dense("glu_forward", h)
    out = torch.empty((*h.shape[:-1], ff), dtype=h.dtype, device=h.device)
    with torch.cuda.device(h.device):
        _lib.check(_lib.load().ldm_glu_forward(h.data_ptr(), out.data_ptr(), dt_code(h.dtype), h.numel() // (2 * ff), ff,
                                               1 if act == "geglu" else 0, _stream(h)), "ldm_glu_forward")
    return out


def glu_backward(h: torch.Tensor, dout: torch.Tensor, act: str) -> torch.Tensor:
    _gpu(h, dout)
    ff = h.shape[-1] // 2
    _same_dtype_dense("glu_backward", h, dout)
    if dout.numel() * 2 != h.numel():
        raise ValueError("glu_backward: dout must have half of h's columns")
    dh = torch.empty_like(h)
    with torch.cuda.device(h.device):
        _lib.check(_lib.load().ldm_glu_backward(h.data_ptr(), dout.data_ptr(), dh.data_ptr(), dt_code(h.dtype),
                                                h.numel() // (2 * ff), ff, 1 if act == "geglu" else 0, _stream(h)),
                   "ldm_glu_backward")
    return dh


def _rows_view(t: torch.Tensor):
    """(rows, cols, row stride) of a tensor that is a dense matrix or a column slice of one."""
    cols = t.shape[-1]
    rows = t.numel() // cols if cols else 0
    if t.stride(-1) != 1:
        raise ValueError("operand must have unit column stride")
    ld = t.stride(-2) if t.dim() > 1 else cols
    exp = ld
    for d in range(t.dim() - 2, -1, -1):      # leading dimensions must be a plain row enumeration
        if t.shape[d] != 1 and t.stride(d) != exp:
            raise ValueError("operand must be a row-strided matrix view")
        exp *= t.shape[d]
    return rows, cols, ld


def add(a: torch.Tensor, b: torch.Tensor) -> torch.Tensor:
    """a + b -> dense tensor; a and b may be column slices of wider matrices (halves of a concat gradient)."""
    _gpu(a, b)
    if a.shape != b.shape or a.dtype != b.dtype:
        raise ValueError("add: operands must have equal shape and dtype")
    rows, cols, lda = _rows_view(a)
    _, _, ldb = _rows_view(b)
    out = torch.empty(a.shape, dtype=a.dtype, device=a.device)
    with torch.cuda.device(a.device):
        _lib.check(_lib.load().ldm_add(a.data_ptr(), lda, b.data_ptr(), ldb, out.data_ptr(), dt_code(a.dtype), rows, cols,
                                       _stream(a)), "ldm_add")
    return out


def silu_backward(x: torch.Tensor, dy: torch.Tensor) -> torch.Tensor:
    _gpu(x, dy)
    _same_dtype_dense("silu_backward", x, dy)
    if dy.numel() != x.numel():
        raise ValueError("silu_backward: dy must have x's element count")
    dx = torch.empty_like(x)
    with torch.cuda.device(x.device):
        _lib.check(_lib.load().ldm_silu_backward(x.data_ptr(), dy.data_ptr(), dx.data_ptr(), dt_code(x.dtype), x.numel(),
                                                 _stream(x)), "ldm_silu_backward")
    return dx


def layernorm(x: torch.Tensor, gamma: torch.Tensor, beta: torch.Tensor, eps: float = 1e-5) -> torch.Tensor:
    _gpu(x, gamma, beta)
    cols = x.shape[-1]
    _same_dtype_dense("layernorm", x)
    _f32_dense("layernorm: gamma", gamma, cols)
    _f32_dense("layernorm: beta", beta, cols)
    out = torch.empty_like(x)
    with torch.cuda.device(x.device):
        _lib.check(_lib.load().ldm_layernorm(x.data_ptr(), dt_code(x.dtype), x.numel() // cols, cols, eps, gamma.data_ptr(),
                                             beta.data_ptr(), out.data_ptr(), _stream(x)), "ldm_layernorm")
    return out


def attention(q: torch.Tensor, kv: torch.Tensor, heads: int) -> torch.Tensor:
    """q: (B, Lq, C); kv: (B, Lk, 2C) with K in the first C columns and V in the last (unet.py:656-657).
    Returns (B, Lq, C) with heads merged."""
    _gpu(q, kv)
    B, Lq, Cq = q.shape
    Lk = kv.shape[1]
    if kv.shape[2] != 2 * Cq or Cq % heads:
        raise ValueError("attention: kv must have 2*C columns and C must divide into heads")
    d = Cq // heads
    _rows3("attention: q", q, q.dtype, B, Lq, Cq)
    _rows3("attention: kv", kv, q.dtype, B, Lk, 2 * Cq)
    out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    es = q.element_size()
    with torch.cuda.device(q.device):
        _lib.check(_lib.load().ldm_attention(q.data_ptr(), q.stride(1), kv.data_ptr(), kv.data_ptr() + Cq * es, kv.stride(1),
                                             out.data_ptr(), out.stride(1), dt_code(q.dtype), B, heads, Lq, Lk, d,
                                             _stream(q)), "ldm_attention")
    return out


def attention_train(q: torch.Tensor, kv: torch.Tensor, heads: int):
    """attention() that also returns lse (B, heads, Lq) float32 = log2 sum exp2 of the scaled scores, for the backward."""
    _gpu(q, kv)
    B, Lq, Cq = q.shape
    Lk = kv.shape[1]
    if kv.shape[2] != 2 * Cq or Cq % heads:
        raise ValueError("attention: kv must have 2*C columns and C must divide into heads")
    d = Cq // heads
    _rows3("attention: q", q, q.dtype, B, Lq, Cq)
    _rows3("attention: kv", kv, q.dtype, B, Lk, 2 * Cq)
    out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    lse = torch.empty((B, heads, Lq), dtype=torch.float32, device=q.device)
    es = q.element_size()
    with torch.cuda.device(q.device):
        _lib.check(_lib.load().ldm_attention_train(q.data_ptr(), q.stride(1), kv.data_ptr(), kv.data_ptr() + Cq * es,
                                                   kv.stride(1), out.data_ptr(), out.stride(1), dt_code(q.dtype), B, heads,
                                                   Lq, Lk, d, lse.data_ptr(), _stream(q)), "ldm_attention_train")
    return out, lse


def attention_backward(q, kv, out, dout, lse, heads, dq=None, dkv=None):
    """Gradients of attention(q, kv): returns (dq (B, Lq, C), dkv (B, Lk, 2C): dK first, dV second).  dq / dkv may be
    preallocated (row-strided) views, e.g. the column slices of one (B, L, 3C) buffer for the fused q|k|v projection."""
    _gpu(q, kv, out, dout, lse, dq, dkv)
    B, Lq, Cq = q.shape
    Lk = kv.shape[1]
    d = Cq // heads
    if dq is None:
        dq = torch.empty((B, Lq, Cq), dtype=q.dtype, device=q.device)
    if dkv is None:
        dkv = torch.empty((B, Lk, 2 * Cq), dtype=q.dtype, device=q.device)
    if kv.dim() != 3 or kv.shape[2] != 2 * Cq or Cq % heads:
        raise ValueError("attention_backward: kv must have 2*C columns and C must divide into heads")
    for nm, t, rows, cols in (("q", q, Lq, Cq), ("kv", kv, Lk, 2 * Cq), ("out", out, Lq, Cq), ("dout", dout, Lq, Cq),
                              ("dq", dq, Lq, Cq), ("dkv", dkv, Lk, 2 * Cq)):
        _rows3("attention_backward: " + nm, t, q.dtype, B, rows, cols)
    _f32_dense("attention_backward: lse", lse, B * heads * Lq)
    delta = torch.empty((B, heads, Lq), dtype=torch.float32, device=q.device)
    es = q.element_size()
    with torch.cuda.device(q.device):
        _lib.check(_lib.load().ldm_attention_backward(
            q.data_ptr(), q.stride(1), kv.data_ptr(), kv.data_ptr() + Cq * es, kv.stride(1), out.data_ptr(), out.stride(1),
            dout.data_ptr(), dout.stride(1), lse.data_ptr(), dq.data_ptr(), dq.stride(1), dkv.data_ptr(),
            dkv.data_ptr() + Cq * es, dkv.stride(1), delta.data_ptr(), dt_code(q.dtype), B, heads, Lq, Lk, d, _stream(q)),
            "ldm_attention_backward")
    return dq, dkv


def timestep_embedding(t: torch.Tensor, dim: int, dtype: torch.dtype) -> torch.Tensor:
    _gpu(t)
    t = t.to(torch.float32).contiguous()
    out = torch.empty((t.shape[0], dim), dtype=dtype, device=t.device)
    with torch.cuda.device(t.device):
        _lib.check(_lib.load().ldm_timestep_embedding(t.data_ptr(), t.shape[0], dim, out.data_ptr(), dt_code(dtype), _stream(t)),
                   "ldm_timestep_embedding")
    return out


def conv_in(x: torch.Tensor, w: torch.Tensor, bias: torch.Tensor, out_dtype: torch.dtype) -> torch.Tensor:
    """x: NCHW (B, Cin, H, W); w: float32 OIHW; returns NHWC (B, H, W, Cout)."""
    _gpu(x, w, bias)
    x = x.contiguous()
    B, cin, H, W = x.shape
    cout = w.shape[0]
    _f32_dense("conv_in: filter", w, cout * cin * 9)
    _f32_dense("conv_in: bias", bias, cout)
    out = torch.empty((B, H, W, cout), dtype=out_dtype, device=x.device)
    with torch.cuda.device(x.device):
        _lib.check(_lib.load().ldm_conv_in(x.data_ptr(), dt_code(x.dtype), w.data_ptr(), bias.data_ptr(), out.data_ptr(),
                                           dt_code(out_dtype), B, cin, H, W, cout, _stream(x)), "ldm_conv_in")
    return out


def conv_out(x: torch.Tensor, w: torch.Tensor, bias: torch.Tensor, out_dtype: torch.dtype) -> torch.Tensor:
    """x: NHWC (B, H, W, Cin); w: float32 OIHW; returns NCHW (B, Cout, H, W)."""
    _gpu(x, w, bias)
    B, H, W, cin = x.shape
    cout = w.shape[0]
    _same_dtype_dense("conv_out", x)
    _f32_dense("conv_out: filter", w, cout * cin * 9)
    _f32_dense("conv_out: bias", bias, cout)
    out = torch.empty((B, cout, H, W), dtype=out_dtype, device=x.device)
    with torch.cuda.device(x.device):
        _lib.check(_lib.load().ldm_conv_out(x.data_ptr(), dt_code(x.dtype), w.data_ptr(), bias.data_ptr(), out.data_ptr(),
                                            dt_code(out_dtype), B, cin, H, W, cout, _stream(x)), "ldm_conv_out")
    return out


def silu(x: torch.Tensor) -> torch.Tensor:
    _gpu(x)
    x = x.contiguous()
    out = torch.empty_like(x)
    with torch.cuda.device(x.device):
        _lib.check(_lib.load().ldm_silu(x.data_ptr(), out.data_ptr(), dt_code(x.dtype), x.numel(), _stream(x)), "ldm_silu")
    return out


def gaussian_noise(seed: int, step: int, row0: int, rows: int, row_shape, device) -> torch.Tensor:
    """float32 (rows, *row_shape) N(0,1) noise of global samples [row0, row0 + rows) at `step` (-1: the initial latents): a
    function of (seed, step, global sample index, element) only (ldm_gaussian_noise, Philox4x32-10 + Box-Muller), so a
    batch-sharded sampler draws just its rows and gets the same rows on any number of ranks."""
    device = torch.device(device)
    if device.type != "cuda":
        raise RuntimeError("ldm_amd: gaussian_noise draws on an AMD GPU (there is no CPU fallback)")
    row_elems = 1
    for d in row_shape:
        row_elems *= int(d)
    out = torch.empty((rows, *row_shape), dtype=torch.float32, device=device)
    with torch.cuda.device(device):
        _lib.check(_lib.load().ldm_gaussian_noise(int(seed) & 0xFFFFFFFFFFFFFFFF, int(step), int(row0), int(rows), row_elems,
                                                  out.data_ptr(), torch.cuda.current_stream(device).cuda_stream),
                   "ldm_gaussian_noise")
    return out


# ----------------------------------------------------------------------------- VAE-decoder leg
def softmax_rows(scores: torch.Tensor, valid_cols: int, scale: float, out_dtype: torch.dtype) -> torch.Tensor:
    """scores: float32 (rows, cols).  softmax(scale * scores) over the first valid_cols columns, zeros after."""
    _gpu(scores)
    if scores.dim() != 2 or scores.dtype != torch.float32 or scores.stride(1) != 1:
        raise ValueError("softmax_rows: float32 (rows, cols) with unit column stride expected")
    rows, cols = scores.shape
    out = torch.empty((rows, cols), dtype=out_dtype, device=scores.device)
    with torch.cuda.device(scores.device):
        _lib.check(_lib.load().ldm_softmax_rows(scores.data_ptr(), scores.stride(0), rows, cols, valid_cols, scale,
                                                out.data_ptr(), dt_code(out_dtype), cols, _stream(scores)), "ldm_softmax_rows")
    return out


def conv1x1_nchw(x: torch.Tensor, w: torch.Tensor, bias: torch.Tensor) -> torch.Tensor:
    """x: NCHW with at most 8 channels; w: float32 (cout, cin[, 1, 1]); returns float32 NCHW."""
    _gpu(x, w, bias)
    x = x.contiguous()
    B, cin, H, W = x.shape
    cout = w.shape[0]
    _f32_dense("conv1x1_nchw: filter", w, cout * cin)
    _f32_dense("conv1x1_nchw: bias", bias, cout)
    out = torch.empty((B, cout, H, W), dtype=torch.float32, device=x.device)
    with torch.cuda.device(x.device):
        _lib.check(_lib.load().ldm_conv1x1_nchw(x.data_ptr(), dt_code(x.dtype), w.data_ptr(), bias.data_ptr(), out.data_ptr(),
                                                B, cin, cout, H * W, _stream(x)), "ldm_conv1x1_nchw")
    return out


def image_to_uint8(x: torch.Tensor) -> torch.Tensor:
    """(255 * (x / 2 + 0.5).clamp(0, 1)).to(uint8) as one kernel (train_latent_diffusion.py:600-601)."""
    _gpu(x)
    x = x.contiguous()
    out = torch.empty(x.shape, dtype=torch.uint8, device=x.device)
    with torch.cuda.device(x.device):
        _lib.check(_lib.load().ldm_image_to_uint8(x.data_ptr(), dt_code(x.dtype), out.data_ptr(), x.numel(), _stream(x)),
                   "ldm_image_to_uint8")
    return out


# ------------------------------------------------------------------------ block-scaled ("microscaled") rows, 4 and 8 bits
class MxTensor:
    """Rows in blocks of 32 columns, each block under one power-of-two scale (include/ldm_amd.h ldm_mx_quantize): what
    mx4_quantize / mx8_quantize return and what the mx operators take.

    data   (*lead, 16 * blocks) uint8 for 4-bit elements, (*lead, 32 * blocks) int8 for 8-bit ones, blocks = ceil(cols / 32)
    scale  (*lead, 4 * ceil(blocks / 4)) uint8: exponent + 127 a block (255: NaN)
    cols   columns of the rows that it stands for: elements behind them and scales behind the last block count for nothing (the
           quantisers leave zeros there)

    Both tensors are plain storage: they may be saved, moved or concatenated along leading dimensions like any other."""

    __slots__ = ("data", "scale", "cols")

    def __init__(self, data: torch.Tensor, scale: torch.Tensor, cols: int):
        cols = operator.index(cols)
        blocks = (cols + 31) // 32
        if cols < 1 or data.dim() < 1 or data.dtype not in (torch.uint8, torch.int8):
            raise TypeError(f"MxTensor: data must be uint8 (4-bit) or int8 (8-bit) rows of at least one column (got {data.dtype})")
        if scale.dtype != torch.uint8:
            raise TypeError(f"MxTensor: scale must be uint8 (got {scale.dtype})")
        width = blocks * (16 if data.dtype == torch.uint8 else 32)
        if scale.dim() < 1 or data.shape[-1] != width or scale.shape[-1] != (blocks + 3) // 4 * 4 or data.shape[:-1] != scale.shape[:-1]:
            raise ValueError(f"MxTensor: {cols} columns need rows of {width} elements' bytes and {(blocks + 3) // 4 * 4} scales "
                             f"(got {tuple(data.shape)} and {tuple(scale.shape)})")
        if data.device != scale.device:
            raise ValueError(f"MxTensor: data on {data.device}, scale on {scale.device}")
        if not data.is_contiguous() or not scale.is_contiguous():
            raise ValueError("MxTensor: data and scale must be contiguous")
        self.data, self.scale, self.cols = data, scale, cols

    @property
    def fmt(self) -> int:
        return _lib.MX4 if self.data.dtype == torch.uint8 else _lib.MX8

    @property
    def shape(self) -> torch.Size:
        return torch.Size((*self.data.shape[:-1], self.cols))

    @property
    def rows(self) -> int:
        return self.scale.numel() // self.scale.shape[-1]

    def __repr__(self):
        return f"MxTensor({'mx4' if self.fmt == _lib.MX4 else 'mx8'}, {tuple(self.shape)}, {self.data.device})"


def _same_device(what: str, ref: torch.Tensor, *others: Optional[torch.Tensor]) -> None:
    index = ref.get_device()
    for t in others:
        if t is not None and t.get_device() != index:
            raise ValueError(f"{what}: operands on {ref.device} and {t.device}")


def _mx(what: str, q, fmt: int) -> None:
    if not isinstance(q, MxTensor) or q.data.dtype != (torch.uint8 if fmt == _lib.MX4 else torch.int8):
        raise TypeError(f"{what} must be an MxTensor with {'4' if fmt == _lib.MX4 else '8'}-bit elements")
    _gpu(q.data, q.scale)


def _mx_empty(lead, cols: int, fmt: int, device) -> MxTensor:
    blocks = (cols + 31) // 32
    q = MxTensor.__new__(MxTensor)          # laid out here: nothing for the constructor to check
    if fmt == _lib.MX4:
        q.data = torch.empty((*lead, blocks * 16), dtype=torch.uint8, device=device)
    else:
        q.data = torch.empty((*lead, blocks * 32), dtype=torch.int8, device=device)
    q.scale = torch.empty((*lead, (blocks + 3) // 4 * 4), dtype=torch.uint8, device=device)
    q.cols = cols
    return q


def _call(t: torch.Tensor, entry: str, *args) -> None:
    """The C entry on t's device and its current stream.  These calls take a few microseconds on the GPU for few rows, so the device
    is switched only where it is not the current one (1.3 us)."""
    fn = getattr(_lib.load(), entry)
    if 0 <= t.get_device() == torch.cuda.current_device():
        rc = fn(*args, _stream(t))
    else:
        with torch.cuda.device(t.device):
            rc = fn(*args, _stream(t))
    if rc:
        _lib.check(rc, entry)


def _mx_quantize(what: str, x: torch.Tensor, fmt: int) -> MxTensor:
    _gpu(x)
    code = dt_code(x.dtype)
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError(f"{what}: at least one column expected, got shape {tuple(x.shape)}")
    q = _mx_empty(x.shape[:-1], x.shape[-1], fmt, x.device)
    if x.numel() == 0:
        return q
    rows, cols, ld = _rows_view(x)
    if rows > 1 and ld < cols:
        raise ValueError(f"{what}: rows overlap (row stride {ld} for {cols} columns)")
    _call(x, "ldm_mx_quantize", x.data_ptr(), code, rows, cols, max(ld, cols), fmt, q.data.data_ptr(), q.scale.data_ptr())
    return q


def mx4_quantize(x: torch.Tensor) -> MxTensor:
    """x (*lead, cols) float32 / bfloat16 (a dense tensor or a column slice of one) in 4-bit floats, one power-of-two scale per 32
    columns: 4.25 bits a value.  Weights for mx4_linear, and its left operand.  A block with an infinity or a NaN becomes NaN."""
    return _mx_quantize("mx4_quantize", x, _lib.MX4)


def mx8_quantize(x: torch.Tensor) -> MxTensor:
    """x (*lead, cols) float32 / bfloat16 in 8-bit whole numbers, one power-of-two scale per 32 columns: 8.25 bits a value, off by at
    most a 64th of the block's largest magnitude.  The checkpoint that linear_wgrad_mx8 and glu_backward_mx8 read."""
    return _mx_quantize("mx8_quantize", x, _lib.MX8)


def mx_dequantize(q: MxTensor, dtype: torch.dtype) -> torch.Tensor:
    """The values q stands for, float32 or bfloat16 (both hold them exactly)."""
    if not isinstance(q, MxTensor):
        raise TypeError("mx_dequantize: an MxTensor expected")
    _gpu(q.data, q.scale)
    code = dt_code(dtype)
    out = torch.empty((*q.data.shape[:-1], q.cols), dtype=dtype, device=q.data.device)
    if out.numel():
        _call(out, "ldm_mx_dequantize", q.data.data_ptr(), q.scale.data_ptr(), q.fmt, q.rows, q.cols, out.data_ptr(), code, q.cols)
    return out


def _mx4_widen_once(rows: int, n: int, k: int) -> bool:
    """bf16 activations: whether the weights are widened once to memory, or in registers, by workgroups of 64 rows and 16 outputs.
    In registers up to 256 rows (k = 128 .. 8192, us: 1280 outputs 5.7 .. 28 against 8.9 .. 35, 8192 outputs 11 .. 66 / 9.8 .. 77); beyond,
    while such workgroups are few (k = 1280: 512 rows on 1280 outputs 13.6 / 14.7, on 1920 17.0 / 16.1, on 2560 21.2 / 19.2) and so is what
    they read of x again for every 16 outputs but the first (512 rows on 1280: k = 2560 18.9 / 20.4, k = 8192 40 / 35; 4096 rows on 160: k = 320
    9.8 / 9.4, k = 1280 18.1 / 13.1, k = 8192 76 / 31; 8000 rows on 32: k = 1280 9.6 / 13.0, k = 5120 25.7 / 24.9; 30000 rows on 16: k = 5120
    57 / 63).  The product behind the widening takes 2^21 columns, the other 2^22."""
    down, across = (rows + 63) // 64, (n + 15) // 16
    return rows > 256 and k <= 1 << 21 and (down * across > 960 or down * (across - 1) * rows * k > 1_300_000_000)


def _pad_cols(t: torch.Tensor, cols: int) -> torch.Tensor:
    """bfloat16 (rows, c) -> (rows, cols) zero-padded copy for operands that are fetched 16 bytes at a time; t itself if it can be."""
    if t.shape[-1] == cols and t.data_ptr() % 16 == 0:
        return t
    out = torch.empty((t.shape[0], cols), dtype=t.dtype, device=t.device)
    _call(t, "ldm_pad_columns_bf16", t.data_ptr(), out.data_ptr(), t.shape[0], t.shape[1], cols)
    return out


def _widening_workspace(x: torch.Tensor, rows: int, inner: int, outer: int):
    """(workspace, bytes) of ldm_mx4_linear_wide / ldm_mx4_linear_dgrad: the widened weights, and x's rows where they cannot be fetched 16
    bytes at a time."""
    inner8 = (inner + 7) // 8 * 8
    size = inner8 * (outer + (rows if inner8 != inner or x.data_ptr() % 16 else 0))
    return torch.empty(size, dtype=torch.bfloat16, device=x.device), 2 * size


def mx4_linear(x, w: MxTensor, bias: Optional[torch.Tensor] = None, out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """x W^T + bias for 4-bit weights w (n, k): (*lead, n), float32 sums.  x: an MxTensor with 4-bit elements (*lead, k) -- both
    operands go to the matrix cores as they are -- or bfloat16 (*lead, k), contiguous, multiplied as it is with the weights widened
    (exactly) to bfloat16.  bias: float32 (n,).  out_dtype: bfloat16 (default) or float32."""
    _mx("mx4_linear: w", w, _lib.MX4)
    if w.data.dim() != 2 or w.data.shape[0] < 1:
        raise ValueError(f"mx4_linear: w must be (n, k) with at least one row, got {tuple(w.shape)}")
    n, k = w.data.shape[0], w.cols
    mx = isinstance(x, MxTensor)
    if mx:
        _mx("mx4_linear: x", x, _lib.MX4)
        xt, xk = x.data, x.cols
    else:
        _gpu(x)
        if x.dtype != torch.bfloat16:
            raise TypeError(f"mx4_linear: x must be bfloat16 or an MxTensor (got {x.dtype})")
        if not x.is_contiguous():
            raise ValueError("mx4_linear: x must be contiguous")
        xt, xk = x, x.shape[-1] if x.dim() else 0
    if xk != k:
        raise ValueError(f"mx4_linear: x {tuple(x.shape)} does not match w {tuple(w.shape)}")
    odt = out_dtype or torch.bfloat16
    code = dt_code(odt)
    if bias is not None:
        _gpu(bias)
        _f32_dense("mx4_linear: bias", bias, n)
    _same_device("mx4_linear", xt, w.data, bias)
    lead = xt.shape[:-1]
    rows = xt.numel() // xt.shape[-1]
    if not mx and _mx4_widen_once(rows, n, k):
        out = torch.empty((*lead, n), dtype=odt, device=x.device)
        ws, need = _widening_workspace(x, rows, k, n)
        _call(x, "ldm_mx4_linear_wide", x.data_ptr(), w.data.data_ptr(), w.scale.data_ptr(), _ptr(bias), out.data_ptr(), code, rows, n, k,
              ws.data_ptr(), need)
        return out
    out = torch.empty((*lead, n), dtype=odt, device=xt.device)
    if rows:
        _call(xt, "ldm_mx4_linear", xt.data_ptr(), x.scale.data_ptr() if mx else 0, w.data.data_ptr(), w.scale.data_ptr(), _ptr(bias),
              out.data_ptr(), code, rows, n, k)
    return out


def mx4_linear_dgrad(dy: torch.Tensor, w: MxTensor) -> torch.Tensor:
    """Input gradient of mx4_linear(x, w): dy W, (*lead, n) -> (*lead, k), bfloat16, float32 sums.  The weights themselves have no
    gradient: they are frozen (what is trained around them -- biases, norms, added low-rank layers -- has its own operators)."""
    _mx("mx4_linear_dgrad: w", w, _lib.MX4)
    if w.data.dim() != 2 or w.data.shape[0] < 1:
        raise ValueError(f"mx4_linear_dgrad: w must be (n, k) with at least one row, got {tuple(w.shape)}")
    _gpu(dy)
    n, k = w.data.shape[0], w.cols
    if dy.dtype != torch.bfloat16:
        raise TypeError(f"mx4_linear_dgrad: dy must be bfloat16 (got {dy.dtype})")
    if dy.dim() < 1 or dy.shape[-1] != n or not dy.is_contiguous():
        raise ValueError(f"mx4_linear_dgrad: dy must be a contiguous (..., {n}) tensor, got {tuple(dy.shape)}")
    _same_device("mx4_linear_dgrad", dy, w.data)
    rows = dy.numel() // n
    out = torch.empty((*dy.shape[:-1], k), dtype=dy.dtype, device=dy.device)
    if rows:
        ws, need = _widening_workspace(dy, rows, n, k)
        _call(dy, "ldm_mx4_linear_dgrad", dy.data_ptr(), w.data.data_ptr(), w.scale.data_ptr(), out.data_ptr(), rows, n, k, ws.data_ptr(), need)
    return out


def _glu_kind(what: str, act: str) -> int:
    if act not in ("geglu", "swiglu"):
        raise ValueError(f"{what}: Unsupported activation function: {act}")
    return 1 if act == "geglu" else 0


def glu_forward_mx8(h: torch.Tensor, act: str):
    """glu_forward that leaves an 8-bit checkpoint of h for the backward pass: (out (.., ff), h in mx8), one pass over h.
    h (.., 2 ff) in the packed (paired) column order, ff a multiple of 16; out is computed from h itself."""
    gelu = _glu_kind("glu_forward_mx8", act)
    _gpu(h)
    code = dt_code(h.dtype)
    _same_dtype_dense("glu_forward_mx8", h)
    if h.dim() < 1 or h.shape[-1] < 32 or h.shape[-1] % 32:
        raise ValueError(f"glu_forward_mx8: h needs a multiple of 32 columns, got {tuple(h.shape)}")
    ff = h.shape[-1] // 2
    out = torch.empty((*h.shape[:-1], ff), dtype=h.dtype, device=h.device)
    q = _mx_empty(h.shape[:-1], 2 * ff, _lib.MX8, h.device)
    _call(h, "ldm_glu_forward_mx8", h.data_ptr(), out.data_ptr(), q.data.data_ptr(), q.scale.data_ptr(), code, h.numel() // (2 * ff), ff,
          gelu)
    return out, q


def glu_backward_mx8(h8: MxTensor, dout: torch.Tensor, act: str, recompute: bool = False):
    """Gradient of the gated activation from its checkpoint alone: dh (.., 2 ff) in dout's dtype.  recompute=True: (dh, out) with out
    the activation of the checkpoint, the next layer's input for its weight gradient."""
    gelu = _glu_kind("glu_backward_mx8", act)
    _mx("glu_backward_mx8: h8", h8, _lib.MX8)
    _gpu(dout)
    code = dt_code(dout.dtype)
    _same_dtype_dense("glu_backward_mx8", dout)
    if h8.cols % 32 or dout.dim() < 1 or dout.shape[-1] != h8.cols // 2 or dout.shape[:-1] != h8.data.shape[:-1]:
        raise ValueError(f"glu_backward_mx8: dout {tuple(dout.shape)} does not match the checkpoint {tuple(h8.shape)}")
    _same_device("glu_backward_mx8", dout, h8.data)
    ff = h8.cols // 2
    dh = torch.empty((*dout.shape[:-1], h8.cols), dtype=dout.dtype, device=dout.device)
    out = torch.empty(dout.shape, dtype=dout.dtype, device=dout.device) if recompute else None
    _call(dout, "ldm_glu_backward_mx8", h8.data.data_ptr(), h8.scale.data_ptr(), dout.data_ptr(), dh.data_ptr(), _ptr(out), code, h8.rows,
          ff, gelu)
    return (dh, out) if recompute else dh


def _wgrad_mx8(x8: MxTensor, dy: torch.Tensor, out: torch.Tensor, rows: int, n: int, k: int, accumulate: int) -> None:
    need = _lib.load().ldm_linear_wgrad_mx8_workspace_bytes(rows, n, k)
    # from the allocator, not kept: a graph that captured the call owns its own, and no other call or graph writes to it
    ws = torch.empty(need, dtype=torch.uint8, device=dy.device) if need else None
    _call(dy, "ldm_linear_wgrad_mx8", x8.data.data_ptr(), x8.scale.data_ptr(), dy.data_ptr(), out.data_ptr(), rows, n, k, accumulate, _ptr(ws),
          need)


def linear_wgrad_mx8(x8: MxTensor, dy: torch.Tensor, *, out: Optional[torch.Tensor] = None, accumulate: Optional[bool] = None) -> torch.Tensor:
    """Weight gradient dY^T X (n, k) float32 of a linear layer whose input was kept as an 8-bit checkpoint x8 (*lead, k); dy (*lead, n)
    bfloat16.  ``out`` / ``accumulate`` as conv_wgrad: an existing gradient to accumulate into, or a buffer to overwrite."""
    _mx("linear_wgrad_mx8: x8", x8, _lib.MX8)
    _gpu(dy, out)
    if dy.dtype != torch.bfloat16:
        raise TypeError(f"linear_wgrad_mx8: dy must be bfloat16 (got {dy.dtype})")
    if dy.dim() < 1 or dy.shape[-1] < 1 or dy.shape[:-1] != x8.data.shape[:-1] or not dy.is_contiguous():
        raise ValueError(f"linear_wgrad_mx8: dy must be a contiguous {(*x8.shape[:-1], 'n')} tensor, got {tuple(dy.shape)}")
    _same_device("linear_wgrad_mx8", dy, x8.data, out)
    n, k, rows = dy.shape[-1], x8.cols, x8.rows
    if out is not None and (out.dtype != torch.float32 or tuple(out.shape) != (n, k) or not out.is_contiguous()):
        raise ValueError(f"linear_wgrad_mx8: out must be a contiguous float32 tensor of shape {(n, k)}")
    accumulate = out is not None and (accumulate is None or bool(accumulate))
    npad = (n + 7) // 8 * 8
    if rows and (npad != n or dy.data_ptr() % 16):      # the kernel fetches dy in 16-byte pieces: other rows go through a padded copy
        full = torch.empty((npad, k), dtype=torch.float32, device=dy.device)
        _wgrad_mx8(x8, _pad_cols(dy.view(rows, n), npad), full, rows, npad, k, 0)
        full = full[:n]
        if out is None:
            return full
        # as storage, which is how the kernel writes into the ones of other widths: out may require a gradient itself
        out.detach().add_(full) if accumulate else out.detach().copy_(full)
        return out
    if out is None:
        out = torch.empty((n, k), dtype=torch.float32, device=dy.device)
    if rows == 0:
        if not accumulate:
            out.detach().zero_()
        return out
    _wgrad_mx8(x8, dy, out, rows, n, k, 1 if accumulate else 0)
    return out
