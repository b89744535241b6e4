"""Limits of the calls on listed groups and drafted nodes, before anything is launched (no GPU: every pointer is fake)."""
import ctypes as C
import sys

import pytest

import cabi
from test_parts_refusals import ARG, B, CAPACITY, FAKE, N, QPOS, S, view

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


def test_a_batch_is_checked_whole(lib):
    """a workspace that is too small, behind more jobs than are handed on at a time: nothing of the batch is launched"""
    small = view(lib, work_bytes=1 << 16)
    g = (sjk.GroupsJob * 70)(*[sjk.GroupsJob(small if k == 69 else view(lib), B, N, QPOS, FAKE, FAKE, FAKE << 4) for k in range(70)])
    assert lib.sjk_hip_attend_groups_batch(g, 70, 1, 8, 0.1, 2, sjk.F32, None) == ARG
    t = (sjk.TreeJob * 70)(*[sjk.TreeJob(small if k == 69 else view(lib), B, N, FAKE, FAKE, FAKE << 4) for k in range(70)])
    assert lib.sjk_hip_attend_tree_batch(t, 70, 4, 4, 8, 0.1, sjk.F32, None) == ARG
