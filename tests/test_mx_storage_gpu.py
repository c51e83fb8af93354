"""Storage behind a row's last column counts for nothing, in every kernel that reads block-scaled rows."""
import pytest

import _mx_storage as storage
from ldm import ops

pytestmark = pytest.mark.gpu


def dev(t):
    return t.cuda()


@pytest.mark.parametrize("act", ["mx4", "bf16"])
@pytest.mark.parametrize("rows,n,k", [(1, 1, 1), (3, 40, 45), (17, 20, 96), (40, 36, 264), (70, 72, 333), (300, 3300, 77), (16, 8200, 2057), (290, 900, 77),
                                      (290, 901, 3333), (290, 900, 160), (1030, 1410, 45), (1030, 1410, 297), (2050, 4104, 70), (2050, 4104, 96),
                                      (2050, 4104, 2057)])
def test_product(rows, n, k, act):
    storage.check_product(ops, rows, n, k, act, dev)


@pytest.mark.parametrize("rows,n,k", [(3, 40, 45), (290, 901, 3333), (1030, 1410, 297), (2050, 4104, 70), (2050, 4104, 2057)])
def test_exact_product(rows, n, k):
    storage.check_exact_product(ops, rows, n, k, dev)


def test_other_readers():
    storage.check_other_readers(ops, dev)
