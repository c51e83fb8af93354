"""Limits of the block-scaled operators that the host or the compiler checks (no GPU)."""
import os
import subprocess
import sys

import pytest
import torch

HERE = os.path.dirname(os.path.abspath(__file__))
sys.path.insert(0, os.path.join(HERE, "emu"))

import build_emu  # noqa: E402
from ldm import _lib  # noqa: E402


@pytest.mark.parametrize("slots,fine", [(5, True), (6, False)])
def test_ring_of_the_few_row_kernel(slots, fine, tmp_path):
    """Scales are fetched four steps at a time into two places: a ring of six steps would fetch those of step 8 over step 3's."""
    path = os.path.join(build_emu.CSRC, "mx_gemm.hip")
    with open(path) as f:
        text = build_emu.translate(f.read(), "mx_gemm.hip")
    src = tmp_path / "ring.cpp"
    src.write_text(text + f"\ntemplate void ldm::mx4_rows_kernel<true, 1, 1, 1, {slots}, true, float>(const ldm::Mx4Params);\n")
    r = subprocess.run([build_emu.CLANG, "-std=c++20", "-fsyntax-only", "-w", "-march=native", "-I", os.path.join(HERE, "emu", "shim"), "-I",
                        os.path.join(HERE, "emu"), "-I", build_emu.CSRC, "-x", "c++", str(src)], capture_output=True, text=True)
    assert (r.returncode == 0) == fine, r.stderr[-2000:]
    assert fine or "static assertion" in r.stderr


INT_MAX = 2 ** 31 - 1


def test_products_of_too_many_outputs_are_refused():
    """Column counts whose tiles do not fit an int, and outputs beyond the 2^32 threads of a launch: refused before anything is launched."""
    lib = _lib.load()
    a = torch.zeros(4096, dtype=torch.uint8)
    p = (a.data_ptr() + 15) // 16 * 16

    def bad(rc):
        return rc == -1 and any(why in lib.ldm_last_error() for why in (b"outputs are too many", b"bad sizes"))

    for n in (INT_MAX, INT_MAX - 62, INT_MAX - 63, (1 << 30) + 1):
        for rows in (1, 64, 65, 5000):
            assert bad(lib.ldm_mx4_linear(p, p, p, p, 0, p, 0, rows, n, 32, 0)), (rows, n)
            assert bad(lib.ldm_mx4_linear(p, 0, p, p, 0, p, 0, rows, n, 32, 0)), (rows, n)
            assert bad(lib.ldm_linear_bf16(p, p, 0, p, 1, rows, n, 8, 0)), (rows, n)
    assert bad(lib.ldm_mx4_linear(p, p, p, p, 0, p, 0, 64, 1 << 30, 32, 0))              # 2^25 workgroups of 256 threads
    assert bad(lib.ldm_mx4_linear(p, 0, p, p, 0, p, 0, 64 * 65535, 1 << 20, 32, 0))      # 2^31 workgroups
    assert bad(lib.ldm_mx4_linear(p, p, p, p, 0, p, 0, 1 << 20, 1 << 19, 32, 0))         # 2^25 tiles of 128 x 128
    assert bad(lib.ldm_linear_bf16(p, p, 0, p, 1, 1 << 20, 1 << 19, 8, 0))
    assert bad(lib.ldm_mx4_linear_wide(p, p, p, 0, p, 1, 1 << 20, 1 << 19, 32, p, 1 << 60, 0))
    assert bad(lib.ldm_mx4_linear_dgrad(p, p, p, p, 1 << 20, 32, 1 << 19, p, 1 << 60, 0))


def test_weight_gradient_of_rows_past_31_bits_is_refused():
    """64 rows of dY are fetched under one 31-bit byte count."""
    lib = _lib.load()
    a = torch.zeros(4096, dtype=torch.uint8)
    p = (a.data_ptr() + 15) // 16 * 16
    widest = (1 << 24) - 8                                                                 # 64 rows: 2^31 - 1024 bytes
    assert lib.ldm_linear_wgrad_mx8(p, p, p, p, 64, widest + 8, 32, 0, 0, 0, 0) == -1
    assert b"bad sizes" in lib.ldm_last_error()
    assert lib.ldm_linear_wgrad_mx8_workspace_bytes(1 << 20, widest + 8, 32) == 0
    assert lib.ldm_linear_wgrad_mx8(p + 1, p, p, p, 64, widest, 32, 0, 0, 0, 0) == -1      # the sizes are fine, the pointer is not
    assert b"unaligned" in lib.ldm_last_error()
