"""Rules of the dense feed-forward kernels' sources that no run shows: an instruction marked .aligned (and bar.sync, which is) has to
be executed by all lanes of a warp as one. Where lanes part before it - rows behind the last are not stored, columns behind the last
not loaded - only a barrier of the warp brings them together for certain; without one it is the compiler's choice."""
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "vkernels_b200", "csrc")
FILES = sorted(f for f in os.listdir(CSRC) if f.startswith("dense") and f.endswith((".cu", ".cuh")))
BARRIER = re.compile(r"__syncwarp\(\);|__syncthreads\(\);")
# reached by whole warps from code in which no lane parts: set-up and teardown by one warp, behind the block's barrier
WHOLE = ("tcgen05.alloc", "tcgen05.relinquish_alloc_permit", "tcgen05.dealloc", "tcgen05.wait::ld")


def lines_of(name):
    with open(os.path.join(CSRC, name)) as f:
        return [re.sub(r"//.*", "", line).strip() for line in f]


def needs_whole_warp(line, name):
    if "cluster_sync_all();" in line:
        return True
    return (".aligned" in line or "bar.sync" in line) and not any(w in line for w in WHOLE)


@pytest.mark.parametrize("name", FILES)
def test_aligned_instructions_follow_a_barrier_of_the_warp(name):
    lines = [line for line in lines_of(name) if line]
    for i, line in enumerate(lines):
        if needs_whole_warp(line, name):
            before = lines[max(0, i - 2):i]
            before = [b for b in before if b != "asm volatile("]      # the statement's own first line
            if before and before[-1].startswith('"') and needs_whole_warp(before[-1], name):
                continue                                              # two instructions of one statement
            assert before and BARRIER.search(before[-1]), (name, before, line)


def test_the_rule_is_looked_for_where_it_matters():
    assert {"dense_tc.cuh", "dense_math.cuh", "dense_gemm.cu", "dense_narrow.cu"} <= set(FILES)
    found = [line for name in FILES for line in lines_of(name) if needs_whole_warp(line, name)]
    assert any("tcgen05.ld" in line for line in found) and any("bar.sync" in line for line in found) and any("cluster_sync_all" in line for line in found)
