"""CPU: rules that the sources of general attention's kernels keep, where a breach would show on
a GPU only now and then."""
import re
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parents[1] / "fastflashattention_b200" / "csrc"
SOURCES = sorted(CSRC.glob("ffa_gen_*.cuh"))


def kernels():
    """(name, parameters, body) of every kernel."""
    for path in SOURCES:
        text = re.sub(r"//[^\n]*", "", path.read_text())
        for m in re.finditer(r"__global__\s+void\s+__launch_bounds__\((?:[^()]|\((?:[^()]|\([^()]*\))*\))*\)\s*(\w+)\(", text):
            ends = []
            for opening, closing, at in (("(", ")", m.end() - 1), ("{", "}", None)):
                at = text.index(opening, ends[-1]) if at is None else at
                depth, end = 0, at
                while True:
                    depth += (text[end] == opening) - (text[end] == closing)
                    end += 1
                    if depth == 0:
                        break
                ends += [at, end]
            yield m.group(1), text[ends[0]:ends[1]], text[ends[2]:ends[3]]


KERNELS = {name: (parameters, body) for name, parameters, body in kernels()}


def test_kernels_are_found():
    assert len(KERNELS) == sum(p.read_text().count("__global__ ") for p in SOURCES) >= 9


@pytest.mark.parametrize("name", sorted(KERNELS))
def test_early_kernels_take_no_constant_pointers(name):
    """A kernel that waits for the one in front of it runs while that one still writes: through a
    `const __restrict__` pointer its loads count as constant and may move above the wait."""
    parameters, body = KERNELS[name]
    if "griddepcontrol.wait" in body:
        assert not re.search(r"const\s+[\w ]+\*\s*__restrict__", parameters)


def functions_with(needle):
    """Bodies of the device functions that contain `needle`."""
    for path in SOURCES:
        text = re.sub(r"//[^\n]*", "", path.read_text())
        for m in re.finditer(r"__device__ __forceinline__ \w+ (\w+)\([^)]*\) \{\n(.*?)\n\}", text, re.S):
            if needle in m.group(2):
                yield m.group(1), m.group(2)


def test_aligned_barriers_find_their_warps_whole():
    """bar.red and barrier.cluster.arrive.aligned want all lanes of a warp at once, and lanes come
    apart in loops and branches by lane: each stands in one function, behind a __syncwarp()."""
    for needle, name in (("named_barrier_and(", "whole_barrier_and"), ("barrier.cluster.arrive", "cluster_barrier")):
        assert sum(p.read_text().count(needle) for p in SOURCES) == 1, needle
        found = dict(functions_with(needle))
        assert list(found) == [name]
        assert found[name].index("__syncwarp();") < found[name].index(needle)
