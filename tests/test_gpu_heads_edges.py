"""Rows at the edges of the append's and the row call's arithmetic: rows whose rotation or sum of squares overflows, in the
sink and behind it, alone in their wavefront and beside rows with infinities and NaNs. The bytes are those of
sjk_hip_head_rows to fp32 followed by sjk_hip_layer_store, whose bytes the oracle pins. Calls of more rows than one launch
holds (2^32 threads)."""
import ctypes as C
import os
import re

import numpy as np
import pytest

import cabi
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
    are those of small calls. By descriptor one launch takes what it holds, and more is refused"""
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
            d_desc = dev.put(desc)
            assert lib.sjk_hip_store_qkv_dyn(C.byref(big), d_desc, n, C.byref(p.m), None, None, kp, vp, None, None) == -100
            n -= 4100                                    # the most that one launch holds, and less
            big.cap = n
            rc = lib.sjk_hip_store_qkv_dyn(C.byref(big), d_desc, n, C.byref(p.m), None, None, kp, vp, None, None)
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


@pytest.mark.parametrize("D,n_rot,layout,rotate", [(128, 0, 0, 1), (256, 0, 0, 1), (64, 64, 0, 1), (512, 512, 1, 1), (128, 64, 0, 1), (128, 40, 0, 0),
                                                   (80, 80, 0, 0), (96, 50, 1, 0), (33, 20, 0, 0), (7, 0, 0, 0), (128, 128, 0, 1)])
@pytest.mark.parametrize("t_out", [sjk.F16, sjk.BF16], ids=["f16", "bf16"])
@pytest.mark.parametrize("norm", [False, True])
def test_fp32_rows_to_16_bits(lib, dev, D, n_rot, layout, rotate, t_out, norm):  # noqa: F811
    """the attention's output on its way to the output projection (the rotation alone, to 16 bits), and fp32 rows through every
    other step, in calls of a few positions and of many, on 16-byte accesses and at any address"""
    rng = np.random.default_rng(D + 1000 * n_rot + t_out)
    r = {"n_rot": n_rot, "layout": layout, "turns": turn_table(n_rot)}
    rope = make_rope(dev, r)
    w = (1 + 0.25 * rng.standard_normal(D)).astype(np.float32)
    for n, heads, offset in ((1, 3, 0), (3, 16, 0), (2, 5, 1), (301, 8, 0), (5, 1, 0)):
        x, o = Set(dev, rng, n, heads, D, sjk.F32, offset=offset, scale=2.0), Set(dev, rng, n, heads, D, t_out, offset=offset)
        run_rows(lib, dev, [head_job(x, o, rope=int(n_rot > 0), rotate=rotate, d_norm=dev.put(w).value if norm else None)], n, D, rope, pos0=4000)
        ref, err = reference(x.values(), 4000 + np.arange(n), w=w if norm else None, rope=r, rotate=bool(rotate))
        check_rows(untouched(o), t_out, ref, err, (n, heads, offset))


def test_fp32_rows_past_the_range_of_16_bits(lib, dev):  # noqa: F811
    """values past the type's largest become infinities, values below its smallest zeros or subnormal, NaNs stay NaNs: the one
    rounding to nearest even that numpy makes"""
    rng = np.random.default_rng(16)
    D = 128
    v = np.concatenate([np.float32([65504, 65519.99, 65520, -65520, 1e30, -3.3895e38, 3.4e38, 2 ** -14, 2 ** -24, 2 ** -25, 2.9802326e-08, 1e-45,
                                    np.inf, -np.inf, np.nan, 0.0, -0.0]), (rng.integers(0, 1 << 32, 64 * D, dtype=np.uint64).astype(np.uint32)).view(np.float32)])
    v = np.resize(v, (64, 1, D))
    for t in (sjk.F16, sjk.BF16):
        x, o = Set(dev, rng, 64, 1, D, sjk.F32), Set(dev, rng, 64, 1, D, t)
        x.host[x.index()] = v.view(np.uint32)
        dev.upload(x.d, x.host)
        run_rows(lib, dev, [head_job(x, o)], 64, D)
        got, want = from_bits(untouched(o), t), from_bits(to_bits(v, t), t)
        assert np.array_equal(np.isnan(got), np.isnan(want))
        assert np.array_equal(got[~np.isnan(got)], want[~np.isnan(want)]) and np.array_equal(np.signbit(got[got == 0]), np.signbit(want[want == 0]))


def midpoints():
    text = open(os.path.join(cabi.ROOT, "include", "sjk_tables.h")).read().replace("\\\n", " ")
    bits = re.search(r"define\s+SJK_TQ6_MIDPOINT_BITS_INIT\s*\{(.*?)\}", text, re.S).group(1)
    return np.array([int(x, 0) for x in re.findall(r"0x[0-9A-Fa-f]+", bits)], np.uint32).view(np.float32)


def step_of(x):
    """floats as integers, one apart from one float to the next (both zeros 0)"""
    i = np.asarray(x, np.float32).view(np.int32).astype(np.int64)
    return np.where(i < 0, -(i & 0x7FFFFFFF), i)


def at_step(i):
    return np.uint32(i if i >= 0 else 0x80000000 - i).view(np.float32)


def test_levels_next_to_every_midpoint(lib, dev):  # noqa: F811
    """blocks whose values over their norm are a midpoint, or one of the three floats on either side of it: the codes of
    sjk_hip_layer_store, which searches the midpoints themselves. numpy makes the same fp32 operations, to see that every midpoint
    is met from both sides and exactly"""
    rng = np.random.default_rng(63)
    mids = midpoints()
    D, H = 128, 8

    def block(i, scale):
        """values mid[i] and mids[62 - i] a few floats apart, times scale, and one that brings the sum of squares to 1"""
        x = np.zeros(D, np.float32)
        near = []
        for m in (mids[i], mids[(i + 21) % 63]):
            for k in range(-3, 4):
                near.append(at_step(step_of(m) + k))
        near = np.array(near, np.float32)
        x[1:1 + len(near)] = near
        x[0] = np.sqrt(max(0.0, 1.0 - np.sum(near.astype(np.float64) ** 2)))
        return (x * np.float32(scale)).astype(np.float32)

    blocks = [block(i, 2.0 ** e * (1 + f)) for i in range(63) for e, f in ((0, 0), (3, 0), (-6, 0), (0, 0.1), (0, 0.37), (1, 0.71), (0, 1e-7), (0, -1e-7))]
    blocks += [block(i, s) for i in range(63) for s in rng.uniform(0.5, 8, 24)]
    rows = np.array(blocks + [np.zeros(D, np.float32)] * (-len(blocks) % (2 * H)), np.float32).reshape(-1, 2 * H, D)
    nsq = np.zeros(rows.shape[:2], np.float32)
    for c in range(D):
        nsq += rows[..., c] * rows[..., c]
    inv = np.float32(1) / np.maximum(np.sqrt(nsq), np.float32(1e-10))
    met = (rows * inv[..., None]).astype(np.float32).ravel()
    for m in mids:
        assert {-1, 0, 1} <= set((step_of(met[np.abs(met - m) < 1e-6]) - step_of(m)).tolist()), m
    n = len(rows)
    A, B = (new_layer(lib, D, H, 0, 0, n_ubatch=256) for _ in range(2))
    va, vb = lib.sjk_layer_view(C.byref(A)), lib.sjk_layer_view(C.byref(B))
    try:
        assert n <= va.cap
        p = Proj(dev, rng, n, 0, H, D, sjk.F32, False, 0, 0, rotate_v=0)
        p.m.rotate_qk = 0
        p.x.host[p.x.index()] = rows.view(np.uint32)
        dev.upload(p.x.d, p.x.host)
        _, k, v = p.ptrs()
        sjk.check(lib.sjk_hip_store_qkv(C.byref(va), 200, n, C.byref(p.m), None, None, k, v, None, None), "store_qkv")
        dk, dv = (dev.put(np.ascontiguousarray(rows[:, a:a + H])) for a in (0, H))
        sjk.check(lib.sjk_hip_layer_store(C.byref(vb), 200, n, dk, dv, 0, None), "layer_store")
        dev.sync()
        for got, want in zip(cache_bytes(dev, va), cache_bytes(dev, vb)):
            assert np.array_equal(got, want)
    finally:
        lib.sj_kvarn_layer_free(C.byref(A))
        lib.sj_kvarn_layer_free(C.byref(B))
