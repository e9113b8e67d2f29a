"""Arguments of the linears of routed rows, the embeddings and the clipping of gradients that are checked on the host; no GPU."""
import ctypes

import pytest
import torch

from symmetrix_b200 import Embedding, EmbeddingPlan, GradientSet, GroupedLinear, _lib, clip_gradients, gradient_norm
from tests.test_adapters import P, _status

CPU = torch.zeros


def grouped_call(**over):
    c = _lib.GroupedCall()
    c.precision, c.num_degrees, c.num_groups, c.num_rows = 64, 2, 3, 10
    for q in range(8):
        d = c.degrees[q]
        d.components, d.in_channels, d.out_channels, d.weight, d.grad_weight = 2 * q + 1, 8, 8, P, P
    c.offsets = c.x = c.y = c.grad_y = c.grad_x = c.workspace = P
    c.x_stride = c.y_stride = c.grad_y_stride = c.grad_x_stride = 32
    c.workspace_bytes = 1 << 40
    for k, v in over.items():
        if k.startswith("degree_"):
            setattr(c.degrees[1], k[7:], v)
        else:
            setattr(c, k, v)
    return c


BAD_CALLS = [
    (dict(precision=16), "precision"), (dict(num_degrees=0), "degrees"), (dict(num_degrees=9), "degrees"), (dict(num_groups=0), "groups"),
    (dict(num_groups=1025), "groups"), (dict(num_rows=-1), "negative"), (dict(num_rows=1 << 31), "32-bit"), (dict(degree_components=0), "components"),
    (dict(degree_components=1025), "components"), (dict(degree_in_channels=0), "channels"), (dict(degree_out_channels=(1 << 20) + 1), "channels"),
    (dict(offsets=None), "plan"), (dict(offsets=P + 2), "multiple"), (dict(status=P + 2), "multiple"), (dict(x=P + 4), "multiple"),
    (dict(degree_weight=P + 4), "multiple"), (dict(precision=32, grad_y=P + 2), "multiple"),
]


@pytest.mark.parametrize("fn", ["smx_grouped_forward", "smx_grouped_backward"])
@pytest.mark.parametrize("over,message", BAD_CALLS)
def test_grouped_refusals(fn, over, message):
    status, text = _status(getattr(_lib.load(), fn), ctypes.byref(grouped_call(**over)))
    assert status == _lib.SMX_ERR_INVALID_ARGUMENT and message in text


@pytest.mark.parametrize("fn,over,message", [
    ("smx_grouped_forward", dict(x=None), "null x"), ("smx_grouped_forward", dict(y=None), "null y"), ("smx_grouped_forward", dict(degree_weight=None), "null weight"),
    ("smx_grouped_forward", dict(y_stride=31), "stride of y"), ("smx_grouped_forward", dict(x_stride=-1), "stride of x"),
    ("smx_grouped_backward", dict(grad_y=None), "null grad_y"), ("smx_grouped_backward", dict(grad_x_stride=31), "stride of grad_x"),
    ("smx_grouped_backward", dict(grad_x=None, x=None), "null x"), ("smx_grouped_backward", dict(degree_grad_weight=None), "all degrees or none"),
    ("smx_grouped_backward", dict(degree_weight=None), "null weight"),
])
def test_grouped_refusals_of_one_direction(fn, over, message):
    status, text = _status(getattr(_lib.load(), fn), ctypes.byref(grouped_call(**over)))
    assert status == _lib.SMX_ERR_INVALID_ARGUMENT and message in text


def test_grouped_null_calls_and_sizes():
    lib = _lib.load()
    assert lib.smx_grouped_workspace_bytes(None, 0) == -1
    assert lib.smx_grouped_workspace_bytes(ctypes.byref(grouped_call(num_groups=0)), 1) == -1
    for backward in (0, 1):
        assert lib.smx_grouped_workspace_bytes(ctypes.byref(grouped_call()), backward) >= 0
    for fn in (lib.smx_grouped_forward, lib.smx_grouped_backward):
        status, text = _status(fn, None)
        assert status == _lib.SMX_ERR_INVALID_ARGUMENT and "null" in text


@pytest.mark.parametrize("args,message", [
    ((P, -1, 1, 4, P, P, None, 0), "negative"), ((P, 4, 0, 4, P, P, None, 0), "slots"), ((P, 4, 65, 4, P, P, None, 0), "slots"), ((P, 4, 1, 0, P, P, None, 0), "table rows"),
    ((P, 4, 1, 1 << 20, P, P, P, 1 << 40), "table rows"), ((P, 1 << 31, 1, 4, P, P, None, 0), "32-bit"), ((None, 4, 1, 4, P, P, None, 0), "null"),
    ((P, 4, 1, 4, None, P, None, 0), "null"), ((P, 4, 1, 4, P, None, None, 0), "null"), ((P, 4, 1, 4, P + 2, P, None, 0), "multiple"),
    ((P, 9000, 1, 4, P, P, None, 0), "workspace"), ((P, 9000, 1, 4, P, P, P, 8), "workspace"), ((P, 9000, 1, 4, P, P, P, -1), "workspace"),
    ((P, 4, 1, 5000, P, P, P, 8), "workspace"),
])
def test_embedding_plan_refusals(args, message):
    status, text = _status(_lib.load().smx_embedding_plan, *args, None)
    assert status == _lib.SMX_ERR_INVALID_ARGUMENT and message in text


def test_embedding_sizes():
    lib = _lib.load()
    assert lib.smx_embedding_plan_bytes(0, 1, 1) == 0 and lib.smx_embedding_plan_bytes(8192, 1, 1023) == 0
    assert lib.smx_embedding_plan_bytes(100, 2, 5000) >= 800             # the order of the lower digits
    for bad in [(-1, 1, 1), (1, 0, 1), (1, 65, 1), (1, 1, 0), (1, 1, 1 << 20), (1 << 31, 1, 1)]:
        assert lib.smx_embedding_plan_bytes(*bad) == -1
    assert lib.smx_embedding_backward_bytes(32, 0, 1, 8) == 0
    for bad in [(16, 1, 1, 8), (32, -1, 1, 8), (32, 1, 0, 8), (32, 1, 1, -1), (32, 1, 1, 65535 * 32 + 1)]:
        assert lib.smx_embedding_backward_bytes(*bad) == -1


@pytest.mark.parametrize("name,args,message", [
    ("smx_embedding_forward", (16, P, 8, 4, P, 4, 1, 8, None, 1.0, P, 8, None), "precision"),
    ("smx_embedding_forward", (32, P, 8, 0, P, 4, 1, 8, None, 1.0, P, 8, None), "table rows"),
    ("smx_embedding_forward", (32, P, -1, 4, P, 4, 1, 8, None, 1.0, P, 8, None), "stride"),
    ("smx_embedding_forward", (32, P, 8, 4, P, 4, 1, 8, None, 1.0, P, 7, None), "stride"),
    ("smx_embedding_forward", (32, P, 8, 4, P, 4, 1, -8, None, 1.0, P, 8, None), "width"),
    ("smx_embedding_forward", (32, P, 1 << 31, 4, P, 4, 1, (1 << 30) + 1, None, 1.0, P, 1 << 31, None), "width"),
    ("smx_embedding_forward", (32, P, 8, 4, P, 4, 99, 8, None, 1.0, P, 8, None), "slots"),
    ("smx_embedding_forward", (32, None, 8, 4, P, 4, 1, 8, None, 1.0, P, 8, None), "null"),
    ("smx_embedding_forward", (64, P + 4, 8, 4, P, 4, 1, 8, None, 1.0, P, 8, None), "multiple"),
    ("smx_embedding_forward", (64, P, 8, 4, P + 2, 4, 1, 8, None, 1.0, P, 8, None), "multiple"),
    ("smx_embedding_backward", (16, P, 8, P, 8, 4, P, P, 4, 1, 8, None, 1.0, P, P, P, 1 << 30, None), "precision"),
    ("smx_embedding_backward", (32, P, -1, P, 8, 4, P, P, 4, 1, 8, None, 1.0, P, P, P, 1 << 30, None), "stride"),
    ("smx_embedding_backward", (32, None, 8, P, 8, 4, P, P, 4, 1, 8, None, 1.0, P, P, P, 1 << 30, None), "null"),
    ("smx_embedding_backward", (32, P, 8, None, 8, 4, P, P, 4, 1, 8, None, 1.0, P, P, P, 1 << 30, None), "table"),
    ("smx_embedding_backward", (32, P, 8, P, 8, 4, None, P, 4, 1, 8, None, 1.0, P, P, P, 1 << 30, None), "null"),
    ("smx_embedding_backward", (32, P, 8, P, 8, 4, P, P, 4, 1, 8, None, 1.0, P, P, P, -1, None), "workspace"),
    ("smx_embedding_backward", (32, P, 8, P, 8, 4, P, P, 4, 1, 8, None, 1.0, P, None, P, 8, None), "workspace"),
    ("smx_embedding_backward", (32, P, 8, P, 8, 4, P, P, 4, 1, 8, None, 1.0, P, None, P + 8, 1 << 30, None), "16-byte"),
    ("smx_embedding_backward", (32, P, 8, P, 8, 4, P, P, 4, 1, 8, None, 1.0, P + 2, None, P, 1 << 30, None), "multiple"),
])
def test_embedding_refusals(name, args, message):
    status, text = _status(getattr(_lib.load(), name), *args)
    assert status == _lib.SMX_ERR_INVALID_ARGUMENT and message in text


def gradient_list(*entries):
    return (_lib.Gradient * len(entries))(*[_lib.Gradient(*e) for e in entries])


@pytest.mark.parametrize("entries,max_norm,workspace,message", [
    ([(P, P, 8, 16)], 1.0, (P, 1 << 20), "precision"), ([(P, P, -1, 32)], 1.0, (P, 1 << 20), "number of values"), ([(P, P, (1 << 40) + 1, 32)], 1.0, (P, 1 << 40), "number of values"),
    ([(None, P, 8, 32)], 1.0, (P, 1 << 20), "null"), ([(P, None, 8, 32)], 1.0, (P, 1 << 20), "null"), ([(P + 2, P, 8, 32)], 1.0, (P, 1 << 20), "multiple"),
    ([(P, P + 4, 8, 64)], 1.0, (P, 1 << 20), "multiple"), ([(P, P, 8, 64)], -1.0, (P, 1 << 20), "largest norm"), ([(P, P, 8, 64)], float("nan"), (P, 1 << 20), "largest norm"),
    ([(P, P, 8, 64)], 1.0, (P, 8), "workspace"), ([(P, P, 8, 64)], 1.0, (None, 1 << 20), "workspace"), ([(P, P, 8, 64)], 1.0, (P, -1), "workspace"),
    ([(P, P, 8, 64)], 1.0, (P + 4, 1 << 20), "multiple"),
])
def test_clip_refusals(entries, max_norm, workspace, message):
    entries = gradient_list(*entries)
    status, text = _status(_lib.load().smx_gradient_clip, entries, len(entries), max_norm, None, *workspace, None)
    assert status == _lib.SMX_ERR_INVALID_ARGUMENT and message in text


def test_gradient_norm_refusals_and_sizes():
    lib = _lib.load()
    entries = gradient_list((P, None, 8, 64))
    status, text = _status(lib.smx_gradient_norm, entries, 1, None, P, 1 << 20, None)
    assert status == _lib.SMX_ERR_INVALID_ARGUMENT and "null norm" in text
    status, text = _status(lib.smx_gradient_norm, None, 1, P, P, 1 << 20, None)
    assert status == _lib.SMX_ERR_INVALID_ARGUMENT and "list" in text
    assert lib.smx_gradient_workspace_bytes(entries, 1) >= 8 and lib.smx_gradient_workspace_bytes(entries, -1) == -1
    # a single tensor of the largest size
    assert lib.smx_gradient_workspace_bytes(gradient_list((P, P, 1 << 40, 64)), 1) > 0


def test_tensors_on_the_host_are_refused():
    with pytest.raises(ValueError, match="CUDA"):
        GroupedLinear([CPU(2, 3, 4)])
    with pytest.raises(ValueError, match="degrees"):
        GroupedLinear([])
    with pytest.raises(ValueError, match="CUDA"):
        Embedding(CPU(2, 3))
    with pytest.raises(ValueError, match="CUDA"):
        EmbeddingPlan(CPU(2, dtype=torch.int32), 3)
    with pytest.raises(ValueError, match="CUDA"):
        GradientSet([CPU(3)])
    with pytest.raises(ValueError, match="at least one"):
        gradient_norm([])
    with pytest.raises(ValueError, match="expected 1"):
        clip_gradients([CPU(3)], 1.0, out=[])
