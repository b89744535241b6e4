"""Limits of the calls on listed groups and drafted nodes, before anything is launched (no GPU: every pointer is fake)."""
import ctypes as C
import sys

import pytest

import cabi
from test_parts_refusals import B, CAPACITY, FAKE, S, view

sys.path.insert(0, cabi.PKG)
import sjk  # noqa: E402


@pytest.fixture(scope="module")
def lib():
    return sjk.load()


def test_selections_past_the_ring(lib):
    """as the attention over the same place"""
    v = view(lib)
    for B_, N, qpos0, n_q in ((B, B + 513, B + 512, 1), (B, B + 600, B + 500, 13), (S, S + 600, S + 599, 1), (0, S + 600, S + 512, 1)):
        assert lib.sjk_hip_select_groups(C.byref(v), B_, N, qpos0, n_q, 8, FAKE, 2, FAKE, None) == CAPACITY, (B_, N, qpos0)
        assert lib.sjk_hip_attend_groups(C.byref(v), B_, N, qpos0, n_q, 8, FAKE, 0.1, FAKE, 2, sjk.F32, FAKE << 4, None) == CAPACITY, (B_, N, qpos0)
    jobs = (sjk.GroupsJob * 2)(*[sjk.GroupsJob(v, B, n, n - 1, FAKE, FAKE, None) for n in (B + 5, B + 513)])
    assert lib.sjk_hip_select_groups_batch(jobs, 2, 1, 8, 2, None) == CAPACITY
