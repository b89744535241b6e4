"""Rows at the edges of the append's and the row call's arithmetic: rows whose rotation or sum of squares overflows, in the
sink and behind it, alone in their wavefront and beside rows with infinities and NaNs. The bytes are those of
sjk_hip_head_rows to fp32 followed by sjk_hip_layer_store, whose bytes the oracle pins. Calls of more rows than one launch
holds (2^32 threads)."""
import ctypes as C

import numpy as np
import pytest

import cabi  # noqa: F401
from test_gpu_heads import (EPS, Proj, Set, cache_bytes, check_rows, dev, from_bits, head_job, lib, make_rope,  # noqa: F401
                            new_layer, reference, run_rows, sjk, to_bits, turn_table, untouched)

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


def windows(n, k, rng):
    """first positions of k-position windows: the ends, the middle and places between, where a call may be cut"""
    return [0, n - k, n // 2 - k // 2] + [int(p) for p in rng.integers(0, n - k, 20)]


def test_more_rows_than_a_launch_holds(lib, dev):  # noqa: F811
    """2^29 rows of two channels turned in place, 2 GiB: the rows are those of small calls"""
    rng = np.random.default_rng(29)
    D, n, k, pos0 = 2, (1 << 29) + 7003, 1000, 5
    row = rng.standard_normal((65536 + 8, D)).astype(np.float16).view(np.uint16)      # (no whole number of these rows is n)
    host = np.resize(row, (n, D))
    d = dev.alloc(host.nbytes, zero=False)
    dev.upload(d, host)
    rope = make_rope(dev, {"n_rot": D, "layout": 0, "turns": turn_table(D)})

    def job(ptr):
        return sjk.HeadJob(ptr, ptr, D, D, D, D, sjk.F16, sjk.F16, 1, 1, 0, EPS, None, 0)

    run_rows(lib, dev, [job(d.value)], n, D, rope, pos0=pos0)
    small = dev.alloc(k * D * 2)
    for p in windows(n, k, rng):
        dev.upload(small, host[p:p + k])
        run_rows(lib, dev, [job(small.value)], k, D, rope, pos0=pos0 + p)
        got, want = (dev.get(C.c_void_p(a), k * D * 2, np.uint16) for a in (d.value + p * D * 2, small.value))
        assert np.array_equal(got, want), p


@pytest.mark.parametrize("dyn", [False, True])
def test_append_of_more_rows_than_a_launch_holds(lib, dev, dyn):  # noqa: F811
    """2^27 positions of one head of 128 to tq6_0, a ring of 26 GB, every position from the same projection row: the staged rows
    are those of small calls"""
    rng = np.random.default_rng(27)
    D, k, pos0 = 128, 500, 40
    n = (1 << 27) + 4003
    A = new_layer(lib, D, 1, 0, 0, n_ubatch=512)
    small = lib.sjk_layer_view(C.byref(A))
    try:
        p = Proj(dev, rng, 1, 0, 1, D, sjk.F16, True, D, 0)
        p.m.q_pos = p.m.k_pos = p.m.v_pos = 0
        _, kp, vp = p.ptrs()
        big = sjk.View.from_buffer_copy(small)
        entry = 2 * big.stage_bytes
        big.cap = n
        big.ring, big.sink = dev.alloc(n * entry, zero=False).value, dev.alloc(big.S * 4 * D).value
        if dyn:
            desc = np.zeros(16, np.int32)
            desc[4] = pos0 + big.S
            rc = lib.sjk_hip_store_qkv_dyn(C.byref(big), dev.put(desc), n, C.byref(p.m), None, None, kp, vp, None, None)
        else:
            rc = lib.sjk_hip_store_qkv(C.byref(big), pos0 + big.S, n, C.byref(p.m), None, None, kp, vp, None, None)
        sjk.check(rc, "store_qkv")
        dev.sync()
        for w in windows(n, k, rng):
            at = pos0 + big.S + w
            sjk.check(lib.sjk_hip_store_qkv(C.byref(small), at, k, C.byref(p.m), None, None, kp, vp, None, None), "store_qkv")
            dev.sync()
            want = cache_bytes(dev, small)[1].reshape(small.cap, entry)[(at - small.S + np.arange(k)) % small.cap]
            slot = (at - big.S) % n
            first = min(k, n - slot)                     # the window may wrap
            got = np.concatenate([dev.get(C.c_void_p(big.ring + s * entry), c * entry, np.uint8) for s, c in ((slot, first), (0, k - first)) if c])
            assert np.array_equal(got.reshape(k, entry), want), w
    finally:
        lib.sj_kvarn_layer_free(C.byref(A))


def test_turns_up_to_the_last_position(lib, dev):  # noqa: F811
    """positions up to 2^32 - 2 by pos0; rows that are not turned, or by positions of their own, take any pos0"""
    rng = np.random.default_rng(32)
    D, n = 128, 255
    r = {"n_rot": D, "layout": 0, "turns": turn_table(D)}
    rope = make_rope(dev, r)
    x, o = Set(dev, rng, n, 2, D, sjk.F32), Set(dev, rng, n, 2, D, sjk.F32)
    run_rows(lib, dev, [head_job(x, o, rope=1)], n, D, rope, pos0=0xFFFFFF00)
    ref, err = reference(x.values(), 0xFFFFFF00 + np.arange(n, dtype=np.int64), rope=r)
    check_rows(untouched(o), sjk.F32, ref, err, "last positions")
    run_rows(lib, dev, [head_job(x, o)], n, D, rope, pos0=0xFFFFFFFF)
    assert np.array_equal(untouched(o), x.host[x.index()])
    run_rows(lib, dev, [head_job(x, o, rope=1)], n, D, rope, pos0=0xFFFFFFFF, d_pos=dev.put(np.zeros(n, np.int32)))
    assert np.array_equal(from_bits(untouched(o), sjk.F32), x.values())
