"""Rules of kernels that start before the one in front of them has ended, checked in their sources; no GPU.

What such a kernel reads of its predecessor's output must not be promised to be constant (``const T* __restrict__`` allows loads through the read-only path, and allows the
compiler to move them across the wait), and it is read behind ``griddepcontrol.wait``."""
import re

import pytest

from symmetrix_b200.build import CSRC

# kernels that wait elsewhere than in their first statement, with the constant arrays that are complete before their predecessor starts
WAITING = {"embedding_join_kernel": ("embedding.cu", {"tokens"}), "gradient_scale_kernel": ("gradients.cu", set()), "grouped_f32_kernel": ("grouped_f32.cuh", set()),
           "grouped_f64_kernel": ("grouped_f64.cuh", set())}


def kernels(text):
    """(name, parameters, body) of every kernel of a file."""
    for m in re.finditer(r"__global__[^;{]*?\b(\w+_kernel)\(", text):
        depth, at = 1, m.end()
        while depth:
            depth += {"(": 1, ")": -1}.get(text[at], 0)
            at += 1
        end = text.index("\n}\n", at)
        yield m.group(1), text[m.end():at - 1], text[at:end]


@pytest.mark.parametrize("name", sorted(WAITING))
def test_what_an_overlapped_kernel_reads_is_not_promised_to_be_constant(name):
    file, complete = WAITING[name]
    found = {n: (p, b) for n, p, b in kernels((CSRC / file).read_text())}
    parameters, body = found[name]
    assert re.search(r'asm volatile\("griddepcontrol\.wait;" ::: "memory"\)', body)
    constant = set(re.findall(r"const\s+\w+\s*\*\s*__restrict__\s+(\w+)", parameters))
    assert constant <= complete


def test_no_other_operator_waits_for_its_predecessor():
    for file in CSRC.glob("*.cu*"):
        text = file.read_text()
        for name, _, body in kernels(text):
            if "griddepcontrol.wait" in body:
                assert name in WAITING and WAITING[name][0] == file.name
