"""The kernels of the attention operators may start while the kernel in front of them still runs: each waits before it reads anything from memory, in every
thread and whatever its arguments. A rule about the sources, checked on the sources: no run can show that a guarantee is missing."""

import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "tilefish_b200", "csrc")
KERNELS = {"rotary.cuh": 2, "paged_attention.cuh": 2}
READS = re.compile(r"p\.\w+(?:\.\w+)?\[|\*reinterpret_cast|\bload_f32\(|\bspan_of<|\bposition_of\(|\bentry_offset\(|\bcos_sin\(|\bcost_of\(")


def kernels(name):
    """(what stands in front of the first statement that is not a declaration of constants, the body) of each kernel."""
    text = re.sub(r"//[^\n]*", "", open(os.path.join(CSRC, name)).read())
    for m in re.finditer(r"__global__", text):
        at = text.index(" {\n", m.end()) + 2
        depth, end = 1, at
        while depth:
            depth += {"{": 1, "}": -1}.get(text[end], 0)
            end += 1
        yield text[at:end]


@pytest.mark.parametrize("name", KERNELS)
def test_nothing_is_read_before_the_wait(name):
    bodies = list(kernels(name))
    assert len(bodies) == KERNELS[name]
    for body in bodies:
        assert body.count("griddep_wait();") == 1
        before = body[:body.index("griddep_wait();")]
        assert before.count("{") == before.count("}"), "the wait stands in a branch or a loop"
        assert not READS.search(before) and "return" not in before and "if (" not in before
