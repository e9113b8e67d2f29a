"""float32 linears with adapters whose rows have few values: every CTA then walks many tiles of one chunk of 32 inner values each.

The kernel's warps work up to four such tiles apart; sizes here give each of a B200's 148 CTAs five tiles of 128 rows and more.
Bounds are those of ``tests/test_gpu_adapters.py``.
"""
import pytest
import torch

from symmetrix_b200 import RowRouting
from tests.test_gpu_adapters import Case, everything

pytestmark = pytest.mark.gpu

ROWS = 148 * 128


@pytest.mark.parametrize("components,in_channels,out_channels", [
    ([3], [32], [64]), ([3], [16], [64]), ([1, 3], [32, 16], [128, 64]), ([1, 3], [33, 32], [64, 64]), ([3], [1], [64]), ([3], [64], [32]),
])
@pytest.mark.parametrize("slots", [1, 2])
@pytest.mark.parametrize("shared", [True, False])
def test_up_to_32_channels(components, in_channels, out_channels, slots, shared):
    """Columns by 64 let all rows leave directly, which is the variant with the longest look-ahead; 64 -> 32 takes it on the way back."""
    case = Case(torch.float32, components, in_channels, out_channels, 6 * ROWS // sum(components) + 77, slots, 5, 7, shared=shared)
    _, _, y, grads = everything(case)
    case.check(y, grads)


@pytest.mark.parametrize("rank", [4, 24, 40, 64])
def test_ranks(rank):
    case = Case(torch.float32, [3], [32], [64], 6 * ROWS // 3 + 5, 1, 3, rank, kind="skewed")
    _, _, y, grads = everything(case)
    case.check(y, grads)


@pytest.mark.parametrize("in_channels,out_channels", [([16, 16], [40, 24]), ([32, 32], [32, 32]), ([40, 72], [16, 32])])
@pytest.mark.parametrize("slots", [1, 2])
def test_products_without_an_output(in_channels, out_channels, slots):
    """Backward passes that make hidden rows only: those of x where they were not kept, those of grad_y where no gradient of x is wanted."""
    case = Case(torch.float32, [1, 3], in_channels, out_channels, 6 * ROWS // (4 * slots) + 31, slots, 4, 6)
    layer, routing = case.layer(), RowRouting(case.ids, case.groups)
    _, hidden = layer.forward(case.x, routing, case.weights, keep_hidden=True)
    case.check(None, layer.backward(case.x, case.gy, routing, case.weights))
    case.check(None, layer.backward(case.x, case.gy, routing, case.weights, hidden=hidden, want_x=False))
    case.check(None, layer.backward(case.x, case.gy, routing, case.weights, want_x=False))
