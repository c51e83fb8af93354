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


@pytest.mark.parametrize("rows,n", [(5, 16), (5, 13), (0, 16)])
def test_weight_gradient_into_a_tensor_that_requires_grad(rows, n):
    """Every width writes into ``out`` the way conv_wgrad does: as storage, whatever autograd knows of it."""
    x, dy = seeded((rows, 40), 1).to(bf), seeded((rows, n), 2).to(bf)
    with emulated() as ops:
        x8 = ops.mx8_quantize(x)
        want = ops.linear_wgrad_mx8(x8, dy)
        out = torch.ones(n, 40, requires_grad=True)
        assert ops.linear_wgrad_mx8(x8, dy, out=out, accumulate=False).data_ptr() == out.data_ptr()
        assert torch.equal(out.detach(), want)
        ops.linear_wgrad_mx8(x8, dy, out=out)
        assert torch.equal(out.detach(), want + want)
        assert out.is_leaf and out.requires_grad


def test_mx_tensor_refuses_a_scalar_scale_and_a_fractional_width():
    with emulated() as ops:
        data, scale = torch.zeros(16, dtype=torch.uint8), torch.zeros(4, dtype=torch.uint8)
        assert ops.MxTensor(data, scale, 32).shape == (32,)
        with pytest.raises(ValueError):
            ops.MxTensor(data, scale[0], 32)
        with pytest.raises(TypeError):
            ops.MxTensor(data, scale, 32.0)
