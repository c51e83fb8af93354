"""Corners of the block-scaled operators' Python front ends (host emulator)."""
import os
import sys

import pytest
import torch

HERE = os.path.dirname(os.path.abspath(__file__))
sys.path.insert(0, os.path.join(HERE, "emu"))

from conftest import seeded  # noqa: E402
from harness import emu_lib, emulated  # noqa: E402

bf = torch.bfloat16


def test_weights_without_rows_are_refused():
    with emulated() as ops:
        w = ops.mx4_quantize(torch.zeros(0, 64))
        before = emu_lib().emu_launch_count()
        for call in (lambda: ops.mx4_linear(torch.zeros(3, 64, dtype=bf), w), lambda: ops.mx4_linear(torch.zeros(0, 64, dtype=bf), w),
                     lambda: ops.mx4_linear_dgrad(torch.zeros(3, 0, dtype=bf), w)):
            with pytest.raises(ValueError, match="at least one row"):
                call()
        assert emu_lib().emu_launch_count() == before
