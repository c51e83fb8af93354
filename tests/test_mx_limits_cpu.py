"""Limits of the block-scaled operators that the host or the compiler checks (no GPU)."""
import os
import subprocess
import sys

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))
sys.path.insert(0, os.path.join(HERE, "emu"))

import build_emu  # noqa: E402


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
