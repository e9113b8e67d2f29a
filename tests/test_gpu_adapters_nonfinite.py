"""NaN and infinities in the operands of linears with adapters: what they touch by the formulas is not finite, all else keeps its bits.

The NaN of the GPU's own float32 arithmetic has all bits of its mantissa set (0x7fffffff), torch's constant only the first; both signs count.
"""
import numpy as np
import pytest
import torch

from symmetrix_b200 import RowRouting
from tests.test_gpu_adapters import Case, host

pytestmark = pytest.mark.gpu

BITS = {torch.float32: {"nan": 0x7FC00000, "computed": 0x7FFFFFFF, "negative": -1, "inf": 0x7F800000, "-inf": -0x800000},
        torch.float64: {"nan": 0x7FF8 << 48, "computed": 0x7FFFFFFFFFFFFFFF, "negative": -1, "inf": 0x7FF0 << 48, "-inf": -(1 << 52)}}


def outputs(case):
    layer, routing = case.layer(), RowRouting(case.ids, case.groups)
    y, hidden = layer.forward(case.x, routing, case.weights, keep_hidden=True)
    grads = layer.backward(case.x, case.gy, routing, case.weights, hidden=hidden)
    again = layer.backward(case.x, case.gy, routing, case.weights, want_x=False)
    return [y, grads.x, *grads.down, *grads.up, grads.weights, *again.down, *again.up, again.weights]


@pytest.mark.filterwarnings("ignore:invalid value", "ignore:overflow")
@pytest.mark.parametrize("dtype", [torch.float32, torch.float64])
@pytest.mark.parametrize("value", ["nan", "computed", "negative", "inf", "-inf"])
@pytest.mark.parametrize("place", ["x", "gy", "weights", "down", "up", "shared"])
@pytest.mark.parametrize("shape", [
    # channels, slots, rank: rows that leave directly and through shared memory, one slot and several
    (64, 1, 8), (64, 2, 16), (40, 2, 7), (130, 1, 33),
], ids=str)
def test_what_is_not_finite_stays_so(dtype, value, place, shape):
    channels, slots, rank = shape
    for shared in ((True,) if place == "shared" else (True, False)):
        case = Case(dtype, [1, 3], [channels, channels], [channels, channels], 300, slots, 3, rank, shared=shared)
        case.ids[17] = 1
        clean = outputs(case)
        integers = torch.int32 if dtype is torch.float32 else torch.int64
        target, at = {"x": (case.x, (17, channels + 5)), "gy": (case.gy, (17, 3)), "weights": (case.weights, (17, slots - 1)),
                      "down": (case.down[1], (1, 9, rank - 1)), "up": (case.up[0], (1, rank - 1, 11)),
                      "shared": (case.shared[1] if shared else None, (6, 2))}[place]
        target.view(integers)[at] = BITS[dtype][value]
        assert not torch.isfinite(target[at])
        y, gx, gds, gus, gw = case.reference()
        for got, before, want in zip(outputs(case), clean, [y, gx, *gds, *gus, gw, *gds, *gus, gw]):
            touched = ~np.isfinite(want)
            found = np.isnan(host(got)) if "inf" not in value else ~np.isfinite(host(got))
            np.testing.assert_array_equal(found, touched)
            keep = torch.as_tensor(~touched).cuda()
            assert torch.equal(got[keep], before[keep])


@pytest.mark.parametrize("shared", [True, False])
def test_nan_made_by_arithmetic(shared):
    """As an earlier kernel leaves it: infinity less infinity, computed on the GPU."""
    case = Case(torch.float32, [1], [64], [64], 200, 1, 2, 8, kind="skewed", shared=shared)
    layer, routing = case.layer(), RowRouting(case.ids, case.groups)
    clean = layer.forward(case.x, routing, case.weights)
    big = torch.full_like(case.x[:1], float("inf"))
    case.x[5:6] = big - big
    case.ids[5] = 1
    routing.update(case.ids)
    got = layer.forward(case.x, routing, case.weights)
    assert torch.isnan(got[5]).all()
    assert torch.equal(got[:5], clean[:5]) and torch.equal(got[6:], clean[6:])


@pytest.mark.filterwarnings("ignore:invalid value")
@pytest.mark.parametrize("shared", [True, False])
@pytest.mark.parametrize("rank", [1, 2, 3, 5, 6, 7, 9, 61])
def test_infinities_in_float64(rank, shared):
    """Positive factors: an infinite value makes positive infinities, and no NaN from the columns that pad the rank. (The reference says where; without
    shared weights it has zeros in their place, which make NaN there.)"""
    case = Case(torch.float64, [1, 3], [24, 17], [17, 24], 90, 1, 2, rank, shared=shared)
    for m in (*case.down, *case.up, *(case.shared or []), case.weights, case.x, case.gy):
        m.abs_().add_(0.1)
    case.ids[:] = 1
    case.x[17, 30], case.gy[40, 3] = float("inf"), float("inf")
    layer, routing = case.layer(), RowRouting(case.ids, case.groups)
    y, grads = layer.forward(case.x, routing, case.weights), layer.backward(case.x, case.gy, routing, case.weights)
    want_y, want_gx, gds, gus, gw = case.reference()
    for got, want in zip([y, grads.x, *grads.down, *grads.up, grads.weights], [want_y, want_gx, *gds, *gus, gw]):
        assert (host(got)[~np.isfinite(want)] == np.inf).all()
        assert np.isfinite(host(got)[np.isfinite(want)]).all()
