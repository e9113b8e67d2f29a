"""float32 linears of routed rows: waits that run out in the pass of the matrices' gradients alone, and infinities."""
import numpy as np
import pytest
import torch

from symmetrix_b200 import SymmetrixError
from tests.test_gpu_grouped import Case, host

pytestmark = pytest.mark.gpu


def test_waits_of_the_matrices_gradients_that_run_out():
    """The test switch takes B behind its first step from every CTA. A tile of more than 64 component rows is lost, be it a group's only sum or one of several; no CTA has more than
    one tile here (84 for 148 SMs), so what is made of one step or none is right. The call itself reports it."""
    case = Case(torch.float32, [300, 0, 700, 40, 100], [1, 3], [70, 200], [136, 64])
    _, _, want = case.expect()
    layer = case.layer
    layer.check()
    layer._fixed.expire_polls = 20000
    lost = layer.backward(case.x, case.gy, case.routing, want_x=False)
    with pytest.raises(SymmetrixError, match="ran out"):
        layer.check()
    layer._fixed.expire_polls = 0
    layer.check()
    for q, (got, (expect, tol)) in enumerate(zip(lost.weights, want)):
        got = host(got)
        gone = np.isnan(got)
        assert gone[0].all() and gone[2].all()               # several sums of 128 rows
        assert gone[4].all()                                 # 100 and 300 component rows: one sum and three
        np.testing.assert_array_equal(got[1], 0.0)           # no rows
        assert gone[3].all() == (q == 1)                     # 40 component rows are one step, 120 are two
        right = ~gone
        assert right.any() and np.all(np.abs(got - expect)[right] <= tol[right])
    case.check()


@pytest.mark.parametrize("value", [float("inf"), -float("inf")])
def test_infinities_give_nan(value):
    case = Case(torch.float32, [150, 0, 37], [1, 3], [72, 40], [64, 136], tail=0)
    before = [case.x.clone(), case.gy.clone(), [w.clone() for w in case.weights]]
    y, gx, gw = case.expect()
    wide_in, wide_out = [72, 40], [64, 136]

    def check(lost_y, lost_gx, lost_gw):
        """Each a list of (degree, index): NaN there, right everywhere else."""
        got_y = case.blocks(host(case.layer.forward(case.x, case.routing)), wide_out)
        grads = case.layer.backward(case.x, case.gy, case.routing)
        for got, want, lost in [(got_y, y, lost_y), (case.blocks(host(grads.x), wide_in), gx, lost_gx), ([host(w) for w in grads.weights], gw, lost_gw)]:
            for q, (a, (b, tol)) in enumerate(zip(got, want)):
                gone = np.zeros(a.shape, bool)
                for d, at in lost:
                    if d == q:
                        gone[at] = True
                assert np.isnan(a[gone]).all() and np.all(np.abs(a - b)[~gone] <= tol[~gone])
        case.x.copy_(before[0])
        case.gy.copy_(before[1])
        for w, b in zip(case.weights, before[2]):
            w.copy_(b)

    row, group = 140, 0
    case.x[row, 72 + 40 * 2 + 5] = value                     # degree 1, component 2, channel 5
    check([(1, np.s_[row, 2, :])], [], [(1, np.s_[group, 5, :])])
    case.gy[row, 3] = value                                  # degree 0, output 3
    check([], [(0, np.s_[row, 0, :])], [(0, np.s_[group, :, 3])])
    case.weights[1][2, 39, 135] = value
    check([(1, np.s_[150:, :, 135])], [(1, np.s_[150:, :, 39])], [])
