"""The workspace of the linears of routed rows: as many sums of the matrices' gradients as any division of the rows into groups can need, and not many more; no GPU."""
import ctypes
import random

import pytest

from symmetrix_b200 import _lib
from tests.test_operator_arguments import grouped_call


def workspace(rows, groups, comps, ins, outs, precision):
    c = grouped_call(precision=precision, num_degrees=1, num_rows=rows, num_groups=groups)
    c.degrees[0].components, c.degrees[0].in_channels, c.degrees[0].out_channels = comps, ins, outs
    return _lib.load().smx_grouped_workspace_bytes(ctypes.byref(c), 1)


def chunk_of(rows, comps, ins, outs, precision):
    """Rows of a sum: four tiles for each of 148 SMs, 128 to 4,096 rows."""
    tile = 128 if precision == 32 else 64
    steps = -(-rows * comps // 64) * -(-ins // tile) * -(-outs // tile)
    return 64 * max(2, min(64, -(-steps // 592)))


@pytest.mark.parametrize("precision", [32, 64])
@pytest.mark.parametrize("rows,groups,comps,ins,outs", [(98304, 1, 7, 2048, 2048), (98304, 89, 7, 2048, 2048), (5000, 16, 3, 128, 128), (1024, 1024, 1, 64, 64), (300, 2, 1, 16, 16),
                                                        (100000, 1000, 2, 8, 8), (127, 1, 1, 4, 4), (1 << 20, 3, 1, 512, 128)])
def test_sums_that_groups_can_need(rows, groups, comps, ins, outs, precision):
    matrix = ins * outs * (precision // 8)
    chunk = chunk_of(rows, comps, ins, outs, precision)
    have = workspace(rows, groups, comps, ins, outs, precision) // matrix
    rng = random.Random(rows + groups)
    most = 0
    for kind in range(60):
        cuts = sorted(rng.randint(0, rows) for _ in range(groups - 1)) if kind else [rows * g // groups for g in range(1, groups)]
        if kind % 3 == 1:                                               # groups just beyond one sum
            cuts = [min(rows, g * (chunk // comps + 1)) for g in range(1, groups)]
        lengths = [b - a for a, b in zip([0, *cuts], [*cuts, rows])]
        sums = [-(-n * comps // chunk) for n in lengths]
        most = max(most, sum(s for s in sums if s > 1))
    whole = rows * comps // chunk
    rounded_up = 63 * (precision // 8) // matrix                        # (to 64 values)
    assert most <= have <= whole + min(groups, whole) + rounded_up


def test_one_group_needs_one_sum_more_than_fill_the_rows():
    # 98,304 atoms, seven components, 2,048 x 2,048: 2.8 GB, not twice that
    assert workspace(98304, 1, 7, 2048, 2048, 32) == 169 * 2048 * 2048 * 4
