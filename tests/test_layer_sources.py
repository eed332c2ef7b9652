"""The transformer-layer kernels' sources keep what no run can show."""

import pathlib
import re

import pytest

CSRC = pathlib.Path(__file__).resolve().parent.parent / "tensorforge_b200" / "csrc"


def kernels(name):
    """(kernel, body) of each __global__ function of a file."""
    text = re.sub(r"//[^\n]*", "", (CSRC / name).read_text())
    for m in re.finditer(r"__global__", text):
        start = text.index("{", text.index(")", text.index("_kernel(", m.end())))
        depth, end = 0, start
        while True:
            depth += {"{": 1, "}": -1}.get(text[end], 0)
            end += 1
            if depth == 0:
                break
        yield re.search(r"(\w+_kernel)\(", text[m.end():]).group(1), text[start:end]


@pytest.mark.parametrize("name", ["tf_layer.cu", "tf_norm.cu", "tf_linear_slim.cu", "tf_linear_pair.cu"])
def test_every_dependent_launch_waits(name):
    """A kernel that may start before the one ahead of it has ended waits for it once, whatever its
    arguments: what earlier grids wrote is visible only behind a grid's own wait.  What the memory
    holds is not promised to be constant either."""
    found = list(kernels(name))
    assert found
    for kernel, body in found:
        waits = [line.strip() for line in body.splitlines() if "grid_dependency_wait" in line]
        assert waits == ["grid_dependency_wait();"], (kernel, waits)
        before = body[:body.index("grid_dependency_wait")].rstrip()
        assert before[-1] in ";{}", (kernel, "a condition before the wait")
        assert before.count("{") - before.count("}") == 1, (kernel, "the wait is inside a block")
        assert "__ldg" not in body and "__restrict__" not in body, kernel
