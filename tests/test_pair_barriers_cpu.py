"""Barriers between the two blocks of a pair, read from the kernels' source: an
arrival on another block's barrier has the cluster as its scope, and what is
handed over by it is waited for with an acquire of the cluster.  (A missing
order between blocks shows on no result that a test could count on.)"""

import re
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parents[1] / "ascend-spmm_b200" / "csrc"
SOURCES = sorted([*CSRC.glob("*.cu"), *CSRC.glob("*.cuh")])


@pytest.mark.parametrize("path", SOURCES, ids=[p.name for p in SOURCES])
def test_remote_arrivals_have_the_scope_of_the_cluster(path):
    for found in re.findall(r"mbarrier\.arrive[\w.:]*shared::cluster[\w.:]*", path.read_text()):
        assert re.search(r"\.(release|relaxed)\.cluster\.", found), found


def test_arrivals_that_order_no_memory_stand_behind_a_fence_of_tmem():
    """`bar_arrive_tmem` hands over what fence_before orders, and nothing else does."""
    for path in SOURCES:
        text = path.read_text()
        for call in re.finditer(r"(?<!void )bar_arrive_tmem\(", text):
            before = text[:call.start()]
            last = before.rfind("fence_before();")
            assert last >= 0 and "st_shared" not in before[last:] and "bar_wait" not in before[last:], path.name


@pytest.mark.parametrize("name", ["gemm_tc.cuh", "fp8_gemm.cuh"])
def test_hand_overs_of_a_pair_are_acquired_from_the_cluster(name):
    """Accumulators (full and empty) and landed slices, whose barriers the other block arrives on."""
    text = (CSRC / name).read_text()
    waits = re.findall(r"bar_wait(<PAIR>)?\((acc_full|acc_empty|full) \+[^;{]*abort\)", text)
    assert {barrier for _, barrier in waits} == {"acc_full", "acc_empty", "full"}
    assert all(pair for pair, _ in waits), waits
