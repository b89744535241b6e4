"""Calls between projections and cache, and those that move pages, that are refused before anything is launched (no GPU; every
device pointer is fake): positions past 32 bits."""
import ctypes as C
import sys

import cabi

sys.path.insert(0, cabi.PKG)
from test_heads_refusals import ARG, FAKE, job, lib, rope, sjk, view  # noqa: E402, F401


def test_head_rows_positions_past_32_bits(lib):  # noqa: F811
    """pos0 + i ends below 2^32 - 1 (no position), as in sjk_hip_store_qkv"""
    def call(n, pos0):
        return lib.sjk_hip_head_rows(C.byref(job(rope=1)), 1, n, 128, C.byref(rope()), pos0, None, None)

    for n, pos0 in ((200, 0xFFFFFF80), (1, 0xFFFFFFFF), (2, 0xFFFFFFFE)):
        assert call(n, pos0) == ARG, (n, pos0)
    assert b"2^32" in lib.sjk_last_error() and call(0, 0xFFFFFFFF) == 0
