"""Arguments of the row routing, the linears with adapters and an evaluator's adapters that are checked on the host; no GPU."""
import ctypes

import pytest

from symmetrix_b200 import _lib
from tests.test_adapters import P, _adapter_call, _status


@pytest.mark.parametrize("fn", ["smx_adapter_forward", "smx_adapter_backward"])
def test_status_off_its_boundary_is_refused(fn):
    status, text = _status(getattr(_lib.load(), fn), ctypes.byref(_adapter_call(status=P + 2)))
    assert status == _lib.SMX_ERR_INVALID_ARGUMENT and "multiple" in text
