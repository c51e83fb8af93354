"""Exact sums in every kernel of the block-scaled products (tests/test_mx_paths_cpu.py holds the cases against the dispatch)."""
import pytest

import _mx_paths as paths
from ldm import ops

pytestmark = pytest.mark.gpu


def dev(t):
    return t.cuda()


@pytest.mark.parametrize("rows,n,k", [c[:3] for c in paths.MX4 + paths.MX4_LARGE])
def test_exact_product_both_4bit(rows, n, k):
    paths.check_linear(ops, rows, n, k, "mx4", dev)


@pytest.mark.parametrize("rows,n,k", [c[:3] for c in paths.BF16 + paths.BF16_LARGE])
def test_exact_product_bf16_rows(rows, n, k):
    paths.check_linear(ops, rows, n, k, "bf16", dev)


@pytest.mark.parametrize("rows,n,k", [c[:3] for c in paths.DGRAD + paths.DGRAD_LARGE])
def test_exact_input_gradient(rows, n, k):
    paths.check_dgrad(ops, rows, n, k, dev)


@pytest.mark.parametrize("rows,n,k", [c[:3] for c in paths.WGRAD + paths.WGRAD_LARGE])
def test_exact_weight_gradient(rows, n, k):
    paths.check_wgrad(ops, rows, n, k, dev)


@pytest.mark.parametrize("act,rows,n,k", [("mx4", *c) for c in paths.NAN_MX4] + [("bf16", *c) for c in paths.NAN_BF16])
def test_nan_blocks(rows, n, k, act):
    paths.check_nan_blocks(ops, rows, n, k, act, dev)
