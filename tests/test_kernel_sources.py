"""Rules that every kernel's source keeps and no run can show safely."""

import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "kvengine_b200", "csrc")
SOURCES = sorted(f for f in os.listdir(CSRC) if f.endswith((".cu", ".cuh")))


def kernels(text):
    """(name, body) of each __global__ function, comments removed."""
    text = re.sub(r"//[^\n]*", "", text)
    for m in re.finditer(r"__global__", text):
        start = text.index("{", text.index(")", text.index("(", m.end() + text[m.end():].index("_kernel"))))
        depth, end = 0, start
        for end in range(start, len(text)):
            depth += {"{": 1, "}": -1}.get(text[end], 0)
            if depth == 0:
                break
        yield re.search(r"(\w+_kernel)\b", text[m.end():]).group(1), text[start:end]


def test_the_kernels_are_found():
    found = [k for f in SOURCES for k in kernels(open(os.path.join(CSRC, f)).read())]
    assert sum("tcgen05.alloc" in body for _, body in found) >= 4 and len(found) > 20


@pytest.mark.parametrize("source", SOURCES)
def test_dependents_start_after_tensor_memory_is_allocated(source):
    """An allocation of tensor memory waits, without a limit, for columns that a CTA on the same SM holds. A
    dependent that has allocated and waits for this kernel must therefore not start before this
    kernel's own allocation: griddepcontrol.launch_dependents comes behind it."""
    for name, body in kernels(open(os.path.join(CSRC, source)).read()):
        if "tcgen05.alloc" in body:
            allocs = [m.start() for m in re.finditer(r"tcgen05\.alloc", body)]
            launches = [m.start() for m in re.finditer(r"grid_dep_launch\(\)", body)]
            assert launches and min(launches) > max(allocs), name
