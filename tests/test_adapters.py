"""Refusals of the row routing and of the adapter linears that need no GPU: every bad argument is an error before any launch."""
import ctypes

import pytest
import torch

from symmetrix_b200 import AdapterLinear, RowRouting, SymmetrixError, _lib

P = 1 << 20          # stands for a device pointer: nothing dereferences it on the host


def _status(fn, *args):
    err = ctypes.create_string_buffer(256)
    return fn(*args, err, 256), err.value.decode()


def test_plan_sizes():
    lib = _lib.load()
    assert lib.smx_route_plan_bytes(0, 1, 1) == 0
    assert lib.smx_route_plan_bytes(8192, 1, 1024) == 0
    assert lib.smx_route_plan_bytes(8193, 1, 3) == 4 * (5 + 1) * 4            # counts of five chunks and a total for each of four bins
    for bad in [(-1, 1, 1), (1, 0, 1), (1, 65, 1), (1, 1, 0), (1, 1, 1025), (1 << 31, 1, 1), ((1 << 31) - 1, 1, 4), (1 << 26, 64, 4)]:
        assert lib.smx_route_plan_bytes(*bad) == -1


@pytest.mark.parametrize("args,message", [
    ((P, -1, 1, 1, P, P, P, None, 0), "negative"),
    ((P, 4, 0, 1, P, P, P, None, 0), "slots"),
    ((P, 4, 1, 0, P, P, P, None, 0), "groups"),
    ((P, 4, 1, 2000, P, P, P, None, 0), "groups"),
    ((P, 1 << 31, 1, 1, P, P, P, None, 0), "32-bit"),
    ((None, 4, 1, 1, P, P, P, None, 0), "null"),
    ((P, 4, 1, 1, P, P, None, None, 0), "null"),
    ((P, 9000, 1, 1, P, P, P, P, 8), "workspace"),
    ((P, 9000, 1, 1, P, P, P, None, 1 << 20), "workspace"),
    ((P, 9000, 1, 1, P, P, P, P, -1), "workspace"),
])
def test_plan_refusals(args, message):
    status, text = _status(_lib.load().smx_route_plan, *args, None)
    assert status == _lib.SMX_ERR_INVALID_ARGUMENT and message in text


@pytest.mark.parametrize("name,args,message", [
    ("smx_route_dispatch", (16, P, 8, 4, 1, 8, P, P, 1, P, 0, None), "precision"),
    ("smx_route_dispatch", (32, P, -8, 4, 1, 8, P, P, 1, P, 0, None), "stride"),
    ("smx_route_dispatch", (32, P, 8, 4, 1, -1, P, P, 1, P, 0, None), "width"),
    ("smx_route_dispatch", (64, P, 8, 4, 1, 1 << 40, P, P, 1, P, 0, None), "width"),
    ("smx_route_dispatch", (64, None, 8, 4, 1, 8, P, P, 1, P, 0, None), "null"),
    ("smx_route_dispatch", (64, P, 8, 4, 99, 8, P, P, 1, P, 0, None), "slots"),
    ("smx_route_combine", (1, P, P, 4, 1, 8, None, None, 0, P, 8, None), "precision"),
    ("smx_route_combine", (32, P, P, 4, 1, 8, None, None, 0, P, 7, None), "overlap"),
    ("smx_route_combine", (32, P, P, 4, 1, 8, None, P, -1, P, 8, None), "stride"),
    ("smx_route_combine", (32, P, None, 4, 1, 8, None, None, 0, P, 8, None), "null"),
    ("smx_route_combine_backward", (3, P, 8, P, P, P, 1, 4, 1, 8, None, P, P, 0, None), "precision"),
    ("smx_route_combine_backward", (32, P, 8, None, P, P, 1, 4, 1, 8, None, P, P, 0, None), "null"),
    ("smx_route_combine_backward", (32, P, 8, P, P, P, 1, 4, 1, 8, None, None, P, 0, None), "null"),
    ("smx_route_combine_backward", (32, P, -1, P, P, P, 1, 4, 1, 8, None, P, P, 0, None), "stride"),
])
def test_row_refusals(name, args, message):
    status, text = _status(getattr(_lib.load(), name), *args)
    assert status == _lib.SMX_ERR_INVALID_ARGUMENT and message in text


def _adapter_call(**over):
    c = _lib.AdapterCall()
    c.precision, c.num_degrees, c.num_groups, c.rank, c.slots, c.num_rows = 64, 2, 3, 4, 1, 10
    for q in range(8):
        d = c.degrees[q]
        d.components, d.in_channels, d.out_channels, d.shared, d.down, d.up = 2 * q + 1, 8, 8, P, P, P
    c.tiles = c.order = c.position = c.offsets = c.x = c.y = c.grad_y = c.grad_x = c.workspace = P
    c.x_stride = c.y_stride = c.grad_y_stride = c.grad_x_stride = 32
    c.workspace_bytes = 1 << 40
    for k, v in over.items():
        if k.startswith("degree_"):
            setattr(c.degrees[1], k[7:], v)
        else:
            setattr(c, k, v)
    return c


@pytest.mark.parametrize("over,message", [
    ({"precision": 16}, "precision"), ({"num_degrees": 0}, "degrees"), ({"num_degrees": 9}, "degrees"), ({"rank": 0}, "rank"), ({"rank": 65}, "rank"),
    ({"num_groups": 0}, "groups"), ({"num_groups": 1025}, "groups"), ({"slots": 0}, "slots"), ({"num_rows": -1}, "negative"),
    ({"num_rows": 1 << 31}, "32-bit"), ({"degree_components": 0}, "components"), ({"degree_in_channels": 0}, "channels"),
    ({"degree_out_channels": (1 << 20) + 1}, "channels"), ({"tiles": None}, "tiles"), ({"order": None}, "plan"), ({"offsets": None}, "plan"),
    ({"tiles": P + 8}, "16-byte"), ({"hidden": P + 4}, "16-byte"), ({"workspace": P + 8}, "16-byte"), ({"x": None}, "null x"), ({"y": None}, "null y"), ({"y_stride": 31}, "stride of y"), ({"x_stride": -1}, "stride of x"),
])
def test_forward_refusals(over, message):
    c = _adapter_call(**over)
    status, text = _status(_lib.load().smx_adapter_forward, ctypes.byref(c))
    assert status == _lib.SMX_ERR_INVALID_ARGUMENT and message in text


@pytest.mark.parametrize("over,message", [
    ({"slots": 2, "workspace_bytes": 0}, "workspace"), ({"workspace_bytes": 0}, "workspace"), ({"workspace": None}, "workspace"),
    ({"grad_y": None}, "grad_y"), ({"grad_x_stride": 31}, "grad_x"), ({"degree_grad_down": P}, "come together"),
    ({"degree_grad_down": P, "degree_grad_up": P}, "all degrees or none"), ({"grad_weights": P, "x": None}, "null x"),
])
def test_backward_refusals(over, message):
    c = _adapter_call(**over)
    status, text = _status(_lib.load().smx_adapter_backward, ctypes.byref(c))
    assert status == _lib.SMX_ERR_INVALID_ARGUMENT and message in text


def test_arrays_off_their_elements_boundaries_are_refused():
    lib, odd = _lib.load(), P + 4
    row = {"smx_route_plan": (P + 2, 4, 1, 2, P, P, P, None, 0, None),
           "smx_route_dispatch": (64, odd, 8, 4, 1, 8, P, P, 1, P, 0, None),
           "smx_route_combine": (64, P, P, 4, 1, 8, odd, None, 0, P, 8, None),
           "smx_route_combine_backward": (64, P, 8, P, P, P, 1, 4, 1, 8, None, odd, P, 0, None)}
    for name, args in row.items():
        status, text = _status(getattr(lib, name), *args)
        assert status == _lib.SMX_ERR_INVALID_ARGUMENT and "multiple" in text, name
    for over in ({"x": odd}, {"y": odd}, {"weights": odd}, {"order": P + 2}, {"offsets": P + 1}):
        status, text = _status(lib.smx_adapter_forward, ctypes.byref(_adapter_call(**over)))
        assert status == _lib.SMX_ERR_INVALID_ARGUMENT and "multiple" in text, over
    for over in ({"grad_y": odd}, {"grad_x": odd}, {"grad_weights": odd}, {"degree_grad_down": odd, "degree_grad_up": P}):
        status, text = _status(lib.smx_adapter_backward, ctypes.byref(_adapter_call(**over)))
        assert status == _lib.SMX_ERR_INVALID_ARGUMENT and "multiple" in text, over
    for over in ({"degree_shared": odd}, {"degree_down": odd}, {"degree_up": odd}):
        status, text = _status(lib.smx_adapter_prepare, ctypes.byref(_adapter_call(**over)), 3)
        assert status == _lib.SMX_ERR_INVALID_ARGUMENT and "multiple" in text, over


def test_prepare_refusals_and_null_calls():
    lib = _lib.load()
    assert _status(lib.smx_adapter_prepare, ctypes.byref(_adapter_call(degree_down=None)), 2)[0] == _lib.SMX_ERR_INVALID_ARGUMENT
    assert _status(lib.smx_adapter_prepare, ctypes.byref(_adapter_call(tiles=None)), 2)[0] == _lib.SMX_ERR_INVALID_ARGUMENT
    assert "part" in _status(lib.smx_adapter_prepare, ctypes.byref(_adapter_call()), 4)[1]
    for fn in (lib.smx_adapter_forward, lib.smx_adapter_backward):
        assert _status(fn, None)[0] == _lib.SMX_ERR_INVALID_ARGUMENT
    for size in (lambda c: lib.smx_adapter_tiles_bytes(c), lambda c: lib.smx_adapter_hidden_elements(c), lambda c: lib.smx_adapter_workspace_bytes(c, 1)):
        assert size(None) == -1
        assert size(ctypes.byref(_adapter_call(rank=0))) == -1
        assert size(ctypes.byref(_adapter_call())) > 0
    assert lib.smx_adapter_hidden_elements(ctypes.byref(_adapter_call(slots=2))) == 10 * 2 * 4 * 4


def test_python_refuses_what_is_not_on_a_gpu():
    with pytest.raises(ValueError, match="CUDA"):
        RowRouting(torch.zeros(4, dtype=torch.int32), 2)
    with pytest.raises(ValueError, match="CUDA"):
        AdapterLinear(None, [torch.zeros(2, 4, 3)], [torch.zeros(2, 3, 4)])
    with pytest.raises(ValueError, match="degrees"):
        AdapterLinear(None, [], [])
    assert issubclass(SymmetrixError, RuntimeError)
