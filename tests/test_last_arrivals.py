"""Barriers at the end of the float32 kernels with specialised warps: whatever arrives at one in a CTA's shared memory arrives before that CTA ends. No GPU."""
import re

import pytest

from symmetrix_b200.build import CSRC


class Barrier:
    """A barrier of one arrival a phase; a wait for a parity returns when the phase at hand has the other one."""
    def __init__(self):
        self.phase = 0

    def wait(self, parity):
        return (self.phase & 1) != parity


@pytest.mark.parametrize("stages", [1, 2, 3, 4, 5])
@pytest.mark.parametrize("count", range(12))
def test_waits_for_the_last_uses_of_all_stages(stages, count):
    """The waits that the kernels end with: use q has stage q % stages and is that stage's phase q / stages. They pass once everything has arrived, and one of them does not as long
    as any stage's last arrival is missing (a stage is used again only behind its arrival before, so no other one can be)."""
    last = range(max(0, count - stages), count)
    assert {q % stages for q in last} == {q % stages for q in range(count)}
    for missing in [None, *last]:
        bars = [Barrier() for _ in range(stages)]
        for q in range(count):
            bars[q % stages].phase += q != missing
        assert all(bars[q % stages].wait((q // stages) & 1) for q in last) == (missing is None)


@pytest.mark.parametrize("file,kernel", [("grouped_f32.cuh", "grouped_f32_kernel"), ("adapters_f32.cuh", "adapter_pass_f32_kernel")])
def test_whoever_commits_products_waits_for_every_barrier_they_arrive_at(file, kernel):
    text = (CSRC / file).read_text()
    body = text[text.index(f" {kernel}("):]
    body = body[:body.index("\n}\n")]
    committed = set(re.findall(r"ts_commit\(&(\w+)", body))
    assert committed and committed <= set(re.findall(r"\bmbar_wait\(&(\w+)", body))
