"""The kernels of the block-scaled products: which call runs which (their launches noted, not run, at every size), and exact sums in each of
them on the host emulator."""
import ctypes as C
import os
import sys

import pytest
import torch

HERE = os.path.dirname(os.path.abspath(__file__))
sys.path.insert(0, os.path.join(HERE, "emu"))
sys.path.insert(0, os.path.join(os.path.dirname(HERE), "tools"))

import _mx_paths as paths  # noqa: E402
import isa_audit  # noqa: E402
from harness import Guarded, emu_lib, emulated  # noqa: E402

bf = torch.bfloat16
OUT = {torch.float32: "float", bf: "unsigned short"}


def _empty4(ops, rows, cols):
    blocks = (cols + 31) // 32
    return ops.MxTensor(torch.empty(rows, 16 * blocks, dtype=torch.uint8), torch.empty(rows, (blocks + 3) // 4 * 4, dtype=torch.uint8), cols)


def _empty8(ops, rows, cols):
    blocks = (cols + 31) // 32
    return ops.MxTensor(torch.empty(rows, 32 * blocks, dtype=torch.int8), torch.empty(rows, (blocks + 3) // 4 * 4, dtype=torch.uint8), cols)


def _linear(ops, act, rows, n, k, dtype):
    x = _empty4(ops, rows, k) if act == "mx4" else torch.empty(rows, k, dtype=bf)
    ops.mx4_linear(x, _empty4(ops, n, k), out_dtype=dtype)


@pytest.fixture
def launched():
    """launched(fn): the names of the kernels that fn launches; none is executed."""
    lib = emu_lib()
    lib.emu_launch_histogram.argtypes, lib.emu_launch_histogram.restype = [C.c_char_p, C.c_longlong, C.c_int], C.c_longlong
    buf = C.create_string_buffer(1 << 16)

    def names(fn, *args):
        lib.emu_launch_histogram(buf, len(buf), 1)
        lib.emu_set_dry_run(1)
        try:
            fn(*args)
        finally:
            lib.emu_set_dry_run(0)
        lib.emu_launch_histogram(buf, len(buf), 1)
        text = [line.split("\t")[1].replace("void ", "") for line in buf.value.decode().splitlines()]
        return {t[len("ldm::"):].split("(")[0] for t in text}

    return names


def _products(launched, ops):
    """{case: kernels} of every case, both output types."""
    out = {}
    for dtype in OUT:
        for act, cases in (("mx4", paths.MX4 + paths.MX4_LARGE), ("bf16", paths.BF16 + paths.BF16_LARGE)):
            for rows, n, k, kernel in cases:
                out[act, rows, n, k, f"{kernel}, {OUT[dtype]}>"] = launched(_linear, ops, act, rows, n, k, dtype)
    for rows, n, k, kernel in paths.DGRAD + paths.DGRAD_LARGE:
        out["dgrad", rows, n, k, f"{kernel}, unsigned short>"] = launched(ops.mx4_linear_dgrad, torch.empty(rows, n, dtype=bf), _empty4(ops, n, k))
    for rows, n, k, kernel in paths.WGRAD + paths.WGRAD_LARGE:
        out["wgrad", rows, n, k, kernel] = launched(ops.linear_wgrad_mx8, _empty8(ops, rows, k), torch.empty(rows, n, dtype=bf))
    return out


def test_every_case_runs_the_kernel_it_is_there_for(launched):
    with emulated() as ops:
        products = _products(launched, ops)
    assert not {case: names for case, names in products.items() if case[-1] not in names}
    for case, names in products.items():
        if case[0] == "wgrad":
            assert ("wgrad_mx8_fold_kernel" in names) == (case[1] >= paths.SPLIT_ROWS), case


def test_every_kernel_of_the_library_has_a_case(launched, tmp_path):
    have = set()
    for name in ("mx_gemm.hip.o", "mx_wgrad.hip.o"):
        path = os.path.join(isa_audit.BUILD, name)
        if not os.path.exists(path):
            pytest.skip("objects not built (make -C latent-diffusion_amd/csrc)")
        have |= {r["kernel"].replace("void ", "").replace("ldm::", "") for r in isa_audit.audit(path, str(tmp_path))}
    with emulated() as ops:
        reached = set().union(*_products(launched, ops).values())
    assert len(have) > 40 and not have - reached, sorted(have - reached)


def test_long_rows_run_in_registers(launched):
    """The product of widened weights takes 2^21 columns, the one in registers 2^22."""
    with emulated() as ops:
        k = (1 << 21) + 8
        assert launched(_linear, ops, "bf16", 257, 1, k, bf) == {"mx4_rows_kernel<false, 4, 1, 4, 2, true, unsigned short>"}
        for rows, n in ((257, 1), (300, 4096), (100000, 4096)):
            assert not ops._mx4_widen_once(rows, n, k) and ops._mx4_widen_once(rows, max(n, 4096), k - 8)


def _both_dma(cases):
    """(rows, n, k, DMA completion model): both models where that takes seconds."""
    return [(*c[:3], dma) for c in cases for dma in ("lazy", "eager") if dma == "lazy" or c[0] * c[1] * c[2] < 5e8]


@pytest.mark.parametrize("rows,n,k,dma", _both_dma(paths.MX4))
def test_exact_product_both_4bit(rows, n, k, dma):
    with Guarded() as g, emulated(dma, guard=True) as ops:
        paths.check_linear(ops, rows, n, k, "mx4", g.like, (bf,) if n % 2 else (torch.float32,))


@pytest.mark.parametrize("rows,n,k,dma", _both_dma(paths.BF16))
def test_exact_product_bf16_rows(rows, n, k, dma):
    with Guarded() as g, emulated(dma, guard=True) as ops:
        paths.check_linear(ops, rows, n, k, "bf16", g.like, (bf,) if n % 2 else (torch.float32,))


@pytest.mark.parametrize("rows,n,k,dma", _both_dma(paths.DGRAD))
def test_exact_input_gradient(rows, n, k, dma):
    with Guarded() as g, emulated(dma, guard=True) as ops:
        paths.check_dgrad(ops, rows, n, k, g.like)


@pytest.mark.parametrize("rows,n,k,dma", _both_dma(paths.WGRAD))
def test_exact_weight_gradient(rows, n, k, dma):
    with Guarded() as g, emulated(dma, guard=True) as ops:
        paths.check_wgrad(ops, rows, n, k, g.like)


@pytest.mark.parametrize("act,rows,n,k", [("mx4", *c) for c in paths.NAN_MX4] + [("bf16", *c) for c in paths.NAN_BF16])
def test_nan_blocks(rows, n, k, act):
    with Guarded() as g, emulated(guard=True) as ops:
        paths.check_nan_blocks(ops, rows, n, k, act, g.like)


def test_the_exact_check_finds_one_lost_column():
    """Planted in the operand on the CPU: the sum without its last column differs, in bfloat16 too where it is not rounded away."""
    x, w = paths.exact4(4, 9000, 1), paths.exact4(8, 9000, 2)
    x[:, -1], w[:, -1] = 4.0, 6.0
    assert ((x @ w.t()) - (x[:, :-1] @ w[:, :-1].t()) == 24.0).all()
    assert torch.equal((x @ w.t()).double(), x.double() @ w.double().t())
