"""Arguments of the row routing, the linears with adapters and an evaluator's adapters that are checked on the host; no GPU."""
import ctypes

import numpy as np
import pytest

from symmetrix_b200 import _lib
from symmetrix_b200.mace import _adapter_ids
from tests.test_adapters import P, _adapter_call, _status


@pytest.mark.parametrize("fn", ["smx_adapter_forward", "smx_adapter_backward"])
def test_status_off_its_boundary_is_refused(fn):
    status, text = _status(getattr(_lib.load(), fn), ctypes.byref(_adapter_call(status=P + 2)))
    assert status == _lib.SMX_ERR_INVALID_ARGUMENT and "multiple" in text


@pytest.mark.parametrize("ids,want", [
    ([0, 2, -1], [0, 2, -1]),
    (np.array([2 ** 32, 2 ** 32 + 1, -2 ** 32 + 1, 2 ** 31, 2 ** 31 - 1, 1]), [-1, -1, -1, -1, 2 ** 31 - 1, 1]),
    (np.array([2 ** 64 - 1, 2 ** 63, 3], dtype=np.uint64), [-1, -1, 3]),
    (np.array([2 ** 32 - 1, 2 ** 31], dtype=np.uint32), [-1, -1]),
    (np.array([[1.0, -1.0], [np.inf, 1e300]]), [[1, -1], [-1, -1]]),
    (np.array([True, False]), [1, 0]),
    ([], []),
])
def test_ids_beyond_32_bits_are_no_adapters(ids, want):
    got = _adapter_ids(ids)
    assert got.dtype == np.int32 and got.flags.c_contiguous
    np.testing.assert_array_equal(got, np.array(want, dtype=np.int32))


@pytest.mark.parametrize("ids", [np.array([0.5, 1.0]), np.array([np.nan, 1.0]), ["a", "b"], np.array([1j]), np.zeros((2, 2, 2)), 3])
def test_ids_that_are_no_numbers_of_adapters_are_refused(ids):
    with pytest.raises(ValueError):
        _adapter_ids(ids)
