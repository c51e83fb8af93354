"""The gate's tail."""
import pytest
import torch

import _mx_gate as gate
from ldm import ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("act", ["geglu", "swiglu"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_tail(act, dtype):
    gate.check_tail(ops, act, dtype, lambda t: t.cuda())
