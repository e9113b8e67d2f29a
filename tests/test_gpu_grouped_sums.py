"""The matrices' gradients of groups with many rows in float32: sums over chunks of rows are added without a loss for each of them."""
import numpy as np
import pytest
import torch

from symmetrix_b200 import GroupedLinear, RowRouting

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("outs", [4, 3])
def test_sums_of_many_chunks(outs):
    """x = 1 and small whole numbers in grad_y: every product and every sum over up to 4,096 rows (a chunk) is a whole number below 2^24, and exact. Each chunk's sum ends on the same
    odd bits, which a float32 sum of all chunks would lose again and again (160 units of 2^-24 here). Eight of them are added with at most seven roundings of 2^-24 of the result, the
    rest in 64 bits, and that is rounded once: at most 8 2^-24 of it."""
    rows, chunk = 4096 * 900, 4096
    gy = torch.full((rows, outs), 4000.0, device="cuda")
    gy[::chunk, 0] = 4450.0
    gy[::chunk, 1] = 4470.0
    routing = RowRouting(torch.zeros(rows, dtype=torch.int32, device="cuda"), 2)
    layer = GroupedLinear([torch.zeros(2, 5, outs, device="cuda")], components=[1])
    got = layer.backward(torch.ones(rows, 5, device="cuda"), gy, routing, want_x=False).weights[0].double().cpu().numpy()
    want = gy.double().sum(0).cpu().numpy()
    np.testing.assert_array_equal(got[1], 0.0)
    assert np.all(np.abs(got[0] - want) <= 8 * 2.0 ** -24 * want), np.max(np.abs(got[0] - want) / want) * 2.0 ** 24
