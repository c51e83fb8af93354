"""The gate's tail on the host emulator."""
import os
import sys

import pytest
import torch

HERE = os.path.dirname(os.path.abspath(__file__))
sys.path.insert(0, os.path.join(HERE, "emu"))

import _mx_gate as gate  # noqa: E402
from harness import Guarded, emulated  # noqa: E402


@pytest.mark.parametrize("act", ["geglu", "swiglu"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_tail(act, dtype):
    with Guarded() as g, emulated(guard=True) as ops:
        gate.check_tail(ops, act, dtype, g.like)
