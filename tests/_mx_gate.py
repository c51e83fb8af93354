"""The gated activation far in the gate's negative tail, where the result itself is below the absolute error that a common approximation of
erfc has: relative bounds.  Body of tests/test_mx_gate_cpu.py and tests/test_mx_gate_gpu.py."""
import torch

from oracle import mx_ref

bf = torch.bfloat16


def check_tail(ops, act, dtype, dev):
    """Gates -2 .. -12.5 in eighths, values 1 .. 15 in eighths: both are 8-bit values of blocks under 2^3, so the checkpoint is h itself.
    Off by: half a step of the type, twice where a factor was rounded before; erfc's fit 2^-12; the exponential, whose argument is off by
    two roundings and which carries them on times the argument, g^2 / 2 (|g| for the sigmoid); 16 roundings or one-step instructions besides.
    a' = Phi + g phi there is at least 0.6 of |g| phi (g <= -2), so its two terms' errors count at most twice; for the sigmoid's, 1 + g (1 - s) is
    at least half of |g|."""
    g = -torch.arange(16, 101, dtype=torch.float64) / 8
    g = torch.cat((g, torch.full((11,), -3.0).double())).view(6, 16)
    v = 15 - torch.arange(96, dtype=torch.float64).view(6, 16) / 8
    h = mx_ref.join_pairs(v, g)
    d = torch.where(torch.arange(96) % 2 == 0, 1.0, -0.75).double().view(6, 16)
    out, h8 = ops.glu_forward_mx8(dev(h.to(dtype)), act)
    assert torch.equal(ops.mx_dequantize(h8, torch.float32).cpu().double(), h)
    dh, again = ops.glu_backward_mx8(h8, dev(d.to(dtype)), act, recompute=True)
    half = 2.0 ** -8 if dtype == bf else 2.0 ** -24
    fit = 2.0 ** -12 if dtype == bf and act == "geglu" else 0.0
    rel = half + fit + 2.0 ** -24 * (16 + 4 * (g * g if act == "geglu" else g.abs()))
    assert float(((out.cpu().double() - mx_ref.glu(h, act)).abs() / mx_ref.glu(h, act).abs() - rel).max()) <= 0
    assert torch.equal(again.cpu(), out.cpu())
    dv, dg = mx_ref.split_pairs((dh.cpu().double() / mx_ref.glu_backward(h, d, act) - 1).abs())
    assert float((dv - rel).max()) <= 0
    assert float((dg - 2 * rel).max()) <= 0
