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
