"""Plans of one CTA whose counters take just under 48 KB of shared memory: each as the first plan of its process."""
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu

PROGRAM = """
import sys
import numpy as np, torch
from symmetrix_b200 import RowRouting
from tests.test_gpu_adapters import make_ids, same_plan
pairs, groups = int(sys.argv[1]), int(sys.argv[2])
ids = make_ids(np.random.default_rng(pairs), pairs, 1, groups)
same_plan(RowRouting(ids, groups), ids)
"""


@pytest.mark.parametrize("pairs,groups", [(993, 371), (8192, 371), (961, 382), (350, 1021), (100, 1024)])
def test_first_plan_of_a_process(pairs, groups):
    """Counters are (warps + 1) x (groups + 1) + 1 ints: 49,108 bytes with 32 warps and 371 groups, to which the kernel's own 132 come; the
    launch needs the attribute for more than 49,152 in all, which only a larger plan set before."""
    r = subprocess.run([sys.executable, "-c", PROGRAM, str(pairs), str(groups)], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stdout + r.stderr
