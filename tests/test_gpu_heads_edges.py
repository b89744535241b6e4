"""Rows at the edges of the append's and the row call's arithmetic: rows whose rotation or sum of squares overflows, in the
sink and behind it, alone in their wavefront and beside rows with infinities and NaNs. The bytes are those of
sjk_hip_head_rows to fp32 followed by sjk_hip_layer_store, whose bytes the oracle pins."""
import ctypes as C

import numpy as np
import pytest

import cabi  # noqa: F401
from test_gpu_heads import Proj, cache_bytes, dev, from_bits, lib, new_layer, sjk, to_bits  # noqa: F401

pytestmark = pytest.mark.gpu


def same_rows(a, b, what):
    """fp32 rows given as bits: NaN in the same places, the same bits everywhere else"""
    na, nb = np.isnan(from_bits(a, sjk.F32)), np.isnan(from_bits(b, sjk.F32))
    assert np.array_equal(na, nb), what
    assert np.array_equal(a[~na], b[~nb]), what


# finite rows: (channels, value) that overflow in the rotation to infinities alone, to infinities and NaNs, in the sum of
# squares only; the largest values that do not
OVERFLOWS = [((5, 6), 3e38), ((0, 1), -3e38), ((0, 127), 3e38), ((3, 5, 6), 3e38), (range(0, 128, 2), 3e38), (range(128), 3e38),
             (range(128), 1e30), ((7,), 3e38), ((5, 6), 1e19)]


# whole turns, parts, parts by LDS, odd addresses, no turn
@pytest.mark.parametrize("n_rot,pad", [(128, 0), (64, 0), (40, 0), (128, 3), (0, 0)])
@pytest.mark.parametrize("D,t", [(128, sjk.F32), (256, sjk.F32), (128, sjk.BF16), (256, sjk.BF16)])
@pytest.mark.parametrize("staging", [0, 1])
def test_append_of_rows_whose_rotation_overflows(lib, dev, D, t, staging, n_rot, pad):  # noqa: F811
    rng = np.random.default_rng(D + t + n_rot + pad)
    H, n_head, n = 4, 4, 2 * len(OVERFLOWS)
    A, B = (new_layer(lib, D, H, staging, 1) for _ in range(2))
    va, vb = lib.sjk_layer_view(C.byref(A)), lib.sjk_layer_view(C.byref(B))
    try:
        for beside in (None, np.inf, np.nan):
            for pos0 in (300, 128 - n // 2):
                p = Proj(dev, rng, n, n_head, H, D, t, False, n_rot, 0, pad=pad)
                flat, idx = from_bits(p.x.host, t).copy(), p.x.index()
                for i, (channels, value) in enumerate(OVERFLOWS):
                    for head in (1, 4 + i % 4, 8 + (i + 1) % 4):                     # a query, a key, a value
                        flat[idx[2 * i, head, list(channels)]] = value
                    if beside is not None:
                        for head in (4 + (i + 1) % 4, 8 + i % 4):                    # other heads of the position
                            flat[idx[2 * i, head, i]] = beside
                        flat[idx[2 * i + 1, 4 + i % 4, i]] = -beside                 # the same head of the next position
                p.x.host = to_bits(flat, t)
                dev.upload(p.x.d, p.x.host)
                want_q = p.two_steps(lib, vb, pos0)
                q, k, v = p.ptrs()
                sjk.check(lib.sjk_hip_store_qkv(C.byref(va), pos0, n, C.byref(p.m), None, q, k, v, p.q, None), "store_qkv")
                dev.sync()
                same_rows(p.q_out(), want_q, (beside, pos0))
                for got, want in zip(cache_bytes(dev, va), cache_bytes(dev, vb)):
                    assert np.array_equal(got, want), (beside, pos0)
    finally:
        lib.sj_kvarn_layer_free(C.byref(A))
        lib.sj_kvarn_layer_free(C.byref(B))
