"""Storage behind a row's last column counts for nothing, in every kernel that reads block-scaled rows (host emulator)."""
import os
import sys

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))
sys.path.insert(0, os.path.join(HERE, "emu"))

import _mx_storage as storage  # noqa: E402
from harness import Guarded, emulated  # noqa: E402


@pytest.mark.parametrize("act", ["mx4", "bf16"])
@pytest.mark.parametrize("rows,n,k", [(3, 40, 1), (3, 40, 45), (17, 20, 96), (40, 36, 264), (70, 72, 333), (300, 3300, 77)])
def test_product_few_rows(rows, n, k, act):
    with Guarded() as g, emulated(guard=True) as ops:
        storage.check_product(ops, rows, n, k, act, g.like)


@pytest.mark.parametrize("dma", ["lazy", "eager"])
@pytest.mark.parametrize("rows,n,k", [(290, 900, 77), (290, 900, 160), (290, 901, 333)])
def test_product_tiles_with_columns_split(rows, n, k, dma):
    with Guarded() as g, emulated(dma, guard=True) as ops:
        storage.check_product(ops, rows, n, k, "mx4", g.like)


# 128 x 128, 256 x 128
@pytest.mark.parametrize("rows,n,k,dma", [(1030, 1410, 45, "lazy"), (1030, 1410, 297, "eager"), (1030, 1410, 352, "lazy"), (2050, 4104, 70, "lazy"),
                                          (2050, 4104, 96, "eager")])
def test_product_tiles(rows, n, k, dma):
    with Guarded() as g, emulated(dma, guard=True) as ops:
        storage.check_exact_product(ops, rows, n, k, g.like)


def test_product_largest_tile():
    """256 x 256, taken for sums of 2048 columns and more."""
    with Guarded() as g, emulated(guard=True) as ops:
        storage.check_exact_product(ops, 2050, 4104, 2057, g.like)


def test_other_readers():
    with Guarded() as g, emulated(guard=True) as ops:
        storage.check_other_readers(ops, g.like)
