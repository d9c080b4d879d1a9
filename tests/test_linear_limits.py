"""Extents at which the products with quantized weights refuse a call, before any CUDA call is made."""
import pytest

from cubek_b200 import ElemType, QuantScheme, QuantStore, QuantValue, grouped_linear, linear
from cubek_b200 import _ffi
from tests.test_linear_refusals import fake, status, weight

BF = ElemType.BF16
BYTES = QuantScheme(value=QuantValue.Q8S, store=QuantStore.Native)


@pytest.mark.parametrize("rows", [2 ** 31 - 511, 2 ** 31 - 1, 2 ** 31])
@pytest.mark.parametrize("n,k", [(1, 8), (16, 8)])
def test_rows(rows, n, k):
    """Row counts that, rounded up to a tile, have no 32-bit integer."""
    x, y = fake((rows, k), 2), fake((rows, n), 2)
    assert status(linear.launch, x, weight((n, k), BYTES), y, BF) == _ffi.QK_ERR_TOO_LARGE
    assert status(linear.launch_backward, y, weight((n, k), BYTES), x, BF) == _ffi.QK_ERR_TOO_LARGE
    assert status(grouped_linear.launch, x, fake((3,), 4), weight((2, n, k), BYTES), y, BF) == _ffi.QK_ERR_TOO_LARGE


def test_tiles():
    """More tiles than a 32-bit integer counts: a row for each of 1024 experts, and rows of the longest gradient."""
    far = 2 ** 26 - 64
    off = fake((1025,), 4)
    x, y = fake((1024, 64), 2), fake((1024, far), 2)
    assert status(grouped_linear.launch, x, off, weight((1024, far, 64), BYTES), y, BF) == _ffi.QK_ERR_TOO_LARGE
    g, gx = fake((2 ** 20, 64), 2), fake((2 ** 20, far), 2)
    assert status(grouped_linear.launch_backward, g, off, weight((1024, 64, far), BYTES), gx, BF) == _ffi.QK_ERR_TOO_LARGE
