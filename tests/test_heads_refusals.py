"""What the calls between projections and cache, and those that move pages, decide on the host (no GPU): the frequency
tables of rotary positions against the same formulas in extended precision, and the calls that are refused before anything
is launched (every pointer in them is fake)."""
import ctypes as C
import sys

import numpy as np
import pytest

import cabi

sys.path.insert(0, cabi.PKG)
import sjk  # noqa: E402

ARG, CAPACITY, UNSUPPORTED = -100, -109, -141
FAKE = 0x10000
L = np.longdouble
TWO_PI = L("6.28318530717958647692528676655900577")


@pytest.fixture(scope="module")
def lib():
    return sjk.load()


def config(n_rot, scaling=0, base=1e4, factor=1.0, n_orig=0.0, low=0.0, high=0.0, divisors=None):
    c = sjk.RopeConfig(n_rot, scaling, base, factor, n_orig, low, high, None)
    if divisors is not None:
        c.divisors = (C.c_double * len(divisors))(*divisors)
    return c


def turns(lib, c):
    out, m = np.full(max(1, c.n_rot // 2), -1.0), C.c_float(-1)
    rc = lib.sjk_rope_turns(C.byref(c), out.ctypes.data_as(C.POINTER(C.c_double)), C.byref(m))
    return rc, out[:c.n_rot // 2], m.value


def want(n, scaling, base, factor, n_orig, low, high, divisors):
    i = np.arange(n // 2).astype(L)
    base, factor = L(base), L(factor)
    if scaling == sjk.ROPE_NTK and n > 2:
        base = base * factor ** (L(n) / (n - 2))
    f = base ** (-2 * i / n)
    if divisors is not None:
        f = f / np.asarray(divisors, L)
    if scaling == sjk.ROPE_LINEAR or (scaling == sjk.ROPE_NTK and n == 2):
        f = f / factor
    if scaling == sjk.ROPE_RAMP:
        lo = max(np.floor(n * np.log(L(n_orig) / (high * TWO_PI)) / (2 * np.log(base))), L(0))
        hi = min(np.ceil(n * np.log(L(n_orig) / (low * TWO_PI)) / (2 * np.log(base))), L(n - 1))
        r = np.clip((i - lo) / max(hi - lo, L(0.001)), 0, 1)
        f = f / factor * r + f * (1 - r)
    if scaling == sjk.ROPE_BANDS:
        s = np.clip((L(n_orig) * f / TWO_PI - low) / (L(high) - low), 0, 1)
        f = f / factor * (1 - s) + f * s
    return f / TWO_PI


@pytest.mark.parametrize("n", [2, 4, 50, 64, 128, 256])
@pytest.mark.parametrize("scaling,factor,n_orig,low,high", [(0, 1, 0, 0, 0), (1, 4, 0, 0, 0), (2, 8, 0, 0, 0), (3, 16, 4096, 1, 32),
                                                            (3, 1, 4096, 1, 32), (3, 40, 32, 0.25, 64), (4, 8, 8192, 1, 4)])
def test_turns_of_every_scaling(lib, n, scaling, factor, n_orig, low, high):
    for base in (1e4, 5e5):
        for div in (None, np.linspace(1.0, 40.0, n // 2)):
            rc, got, m = turns(lib, config(n, scaling, base, factor, n_orig, low, high, div))
            assert rc == 0
            ref = want(n, scaling, base, factor, n_orig, low, high, div)
            # a power (an ulp or two, and the exponent's rounding times its logarithm, at most 13), a handful of products
            assert np.all(np.abs(got - ref) <= 40 * 2.0 ** -53 * ref)
            assert m == np.float32(0.1 * np.log(factor) + 1 if scaling == 3 else 1.0)


def test_turns_refuses_what_has_no_meaning(lib):
    good = dict(n_rot=64, scaling=4, base=1e4, factor=8.0, n_orig=8192.0, low=1.0, high=4.0)
    assert turns(lib, config(**good))[0] == 0
    for k, v in (("n_rot", 63), ("n_rot", -2), ("scaling", 5), ("scaling", -1), ("base", 1.0), ("base", np.nan), ("factor", 0.0),
                 ("factor", np.inf), ("n_orig", 0.0), ("low", 0.0), ("low", 4.0), ("high", np.nan)):
        rc, out, m = turns(lib, config(**dict(good, **{k: v})))
        assert rc == ARG and m == -1 and np.all(out == -1), (k, v)
    assert turns(lib, config(64, 3, factor=0.5, n_orig=10.0, low=1.0, high=2.0))[0] == ARG
    assert turns(lib, config(4, divisors=[1.0, 0.0]))[0] == ARG
    assert turns(lib, config(0))[0] == 0


def job(**kw):
    j = sjk.HeadJob(FAKE, FAKE, 512, 128, 512, 128, sjk.F32, sjk.F32, 4, 0, 0, 0.0, None, 0)
    for k, v in kw.items():
        setattr(j, k, v)
    return j


def rope(**kw):
    r = sjk.Rope(sjk.ROPE_HALVES, 128, 0, 1.0, FAKE)
    for k, v in kw.items():
        setattr(r, k, v)
    return r


def test_head_rows_refusals(lib):
    def call(j, D=128, n=4, r=None, n_jobs=1, d_pos=None):
        return lib.sjk_hip_head_rows(C.byref(j) if j is not None else None, n_jobs, n, D, C.byref(r) if r is not None else None, 0,
                                     d_pos, None)

    assert call(None) == ARG and call(job(), n_jobs=-1) == ARG
    assert call(None, n_jobs=0) == 0 and call(job(), n=0) == 0 and call(job(n_heads=0)) == 0
    for bad in (dict(d_x=None), dict(d_out=None), dict(n_heads=-1), dict(x_type=3), dict(out_type=-1), dict(d_x=FAKE + 2),
                dict(x_type=1, d_x=FAKE + 1), dict(out_type=2, d_out=FAKE + 1)):
        assert call(job(**bad)) == ARG, bad
    for D in (0, -1, 513):
        assert call(job(), D=D) == ARG
    for eps in (0.0, -1e-6, 1e-40, np.nan, np.inf):
        assert call(job(d_norm=FAKE, eps=eps)) == ARG
    assert call(job(d_norm=FAKE + 2, eps=1e-6)) == ARG
    assert call(job(rope=1)) == ARG                                   # no rope given
    for bad in (dict(layout=2), dict(n_rot=63), dict(n_rot=-2), dict(n_rot=130), dict(d_turns=None), dict(d_turns=FAKE + 4),
                dict(mscale=np.nan), dict(mscale=np.inf)):
        assert call(job(rope=1), r=rope(**bad)) == ARG, bad
    for D in (1, 32, 80, 96, 192, 384):
        assert call(job(rotate=1), D=D) == UNSUPPORTED
    assert b"64, 128, 256 or 512" in lib.sjk_last_error()
    assert call(job(n_heads=1 << 20), n=1 << 12) == ARG               # 2^32 rows
    assert call(job(), d_pos=FAKE + 2) == ARG
    two = (sjk.HeadJob * 2)(job(), job(out_type=9))                   # the second of two jobs
    assert lib.sjk_hip_head_rows(two, 2, 4, 128, None, 0, None, None) == ARG


def view(lib, D=128, H=2, staging=0, sink_type=0, cap=256, **kw):
    v = sjk.View()
    assert lib.sj_kvarn_layout_init(C.byref(v.lay), D, 128, 4, 4, 0) == 0
    v.n_head_kv, v.staging, v.sink_type, v.S, v.cap = H, staging, sink_type, 128, cap
    v.stage_bytes = lib.sj_kvarn_stage_row_bytes(staging, D)
    v.sink, v.ring, v.body = FAKE, FAKE * 2, FAKE * 3
    for k, x in kw.items():
        setattr(v, k, x)
    return v


def qkv(**kw):
    m = sjk.Qkv()
    m.type, m.n_head, m.rotate_qk, m.rotate_v, m.eps = sjk.F32, 4, 1, 1, 1e-6
    m.q_pos = m.k_pos = m.v_pos = 1024
    m.q_head = m.k_head = m.v_head = 128
    for k, x in kw.items():
        setattr(m, k, x)
    return m


def test_store_qkv_refusals(lib):
    def calls(v, m, n=1, pos0=0, d_pos=None, q=FAKE, k=FAKE, x=FAKE, out=FAKE, dyn=True):
        pm = C.byref(m) if m is not None else None
        pv = C.byref(v) if v is not None else None
        got = {lib.sjk_hip_store_qkv(pv, pos0, n, pm, d_pos, q, k, x, out, None)}
        if dyn:
            got.add(lib.sjk_hip_store_qkv_dyn(pv, FAKE, n, pm, d_pos, q, k, x, out, None))
        if v is not None:
            j = sjk.QkvJob(v, pos0, d_pos, q, k, x, out)
            got.add(lib.sjk_hip_store_qkv_batch(C.byref(j), 1, n, pm, None))
        assert len(got) == 1, got
        return got.pop()

    assert calls(view(lib), qkv(), n=0) == 0
    assert calls(None, qkv()) == ARG and calls(view(lib), None) == ARG
    assert lib.sjk_hip_store_qkv_dyn(C.byref(view(lib)), None, 1, C.byref(qkv()), None, FAKE, FAKE, FAKE, FAKE, None) == ARG
    for kw in (dict(q=None), dict(k=None), dict(x=None), dict(out=None), dict(out=FAKE + 2), dict(q=FAKE + 2), dict(d_pos=FAKE + 1)):
        assert calls(view(lib), qkv(), **kw) == ARG, kw
    for bad in (dict(sink=None), dict(ring=None), dict(cap=0), dict(n_head_kv=0), dict(staging=2), dict(sink_type=2),
                dict(stage_bytes=100), dict(ring=FAKE + 1)):
        assert calls(view(lib, **bad), qkv()) == ARG, bad
    for bad in (dict(type=3), dict(n_head=-1), dict(d_q_norm=FAKE, eps=0.0), dict(d_k_norm=FAKE, eps=np.nan),
                dict(rope=rope(n_rot=130)), dict(rope=rope(layout=2)), dict(rope=rope(d_turns=None))):
        assert calls(view(lib), qkv(**bad)) == ARG, bad
    assert calls(view(lib, D=512), qkv()) == UNSUPPORTED
    assert calls(view(lib), qkv(), n=257, pos0=128) == CAPACITY       # two positions a slot
    assert calls(view(lib), qkv(), n=257, pos0=5000) == CAPACITY
    assert calls(view(lib), qkv(), n=385, pos0=0, dyn=False) == CAPACITY
    assert calls(view(lib), qkv(), n=200, pos0=0xFFFFFF80, dyn=False) == ARG
    two = (sjk.QkvJob * 2)(*[sjk.QkvJob(view(lib), p, None, FAKE, FAKE, FAKE, FAKE) for p in (0, 5)])
    assert lib.sjk_hip_store_qkv_batch(two, 2, 1, C.byref(qkv()), None) == ARG        # one ring twice
    two[1].v = view(lib, D=256, ring=FAKE * 5)
    assert lib.sjk_hip_store_qkv_batch(two, 2, 1, C.byref(qkv()), None) == ARG        # another head width
    assert lib.sjk_hip_store_qkv_batch(None, 1, 1, C.byref(qkv()), None) == ARG
    assert lib.sjk_hip_store_qkv_batch(two, -1, 1, C.byref(qkv()), None) == ARG
    assert lib.sjk_hip_seq_store_qkv_batch(None, 1, 0, 1, C.byref(qkv()), None) == ARG
    nobody = sjk.SeqQkvJob()
    assert lib.sjk_hip_seq_store_qkv_batch(C.byref(nobody), 1, 0, 1, C.byref(qkv()), None) == ARG


def test_fork_refusals(lib):
    def call(d, s, B=128, N=200, n=1):
        return lib.sjk_hip_fork(C.byref(d), C.byref(s), n, B, N, None)

    far = dict(sink=FAKE * 16, ring=FAKE * 32)
    s = view(lib)
    assert lib.sjk_hip_fork(None, None, 0, 128, 0, None) == 0
    assert lib.sjk_hip_fork(None, C.byref(s), 1, 128, 0, None) == ARG and call(view(lib, **far), s, n=-1) == ARG
    assert call(view(lib, **far), s, N=0) == 0                         # nothing to copy
    assert call(s, s) == ARG
    for kw in (dict(B=0), dict(B=127), dict(B=129), dict(B=256, N=255)):
        assert call(view(lib, **far), s, **kw) == ARG, kw
    for bad in (dict(D=256), dict(H=4), dict(staging=1), dict(sink_type=1), dict(S=192), dict(cap=0), dict(sink=None, ring=FAKE),
                dict(ring=FAKE * 32 + 2, sink=FAKE * 16), dict(stage_bytes=0), dict(sink=FAKE, ring=FAKE * 32), dict(sink=FAKE * 16, ring=FAKE * 2)):
        assert call(view(lib, **dict(far, **bad)), s) == ARG, bad
    assert call(view(lib, **far), s, N=128 + 257) == CAPACITY
    assert call(view(lib, cap=128, **far), s, N=128 + 129) == CAPACITY
    ds = (sjk.View * 2)(view(lib, **far), view(lib, cap=384, **far))
    ss = (sjk.View * 2)(s, s)
    assert lib.sjk_hip_fork(ds, ss, 2, 128, 200, None) == ARG          # capacities differ from layer to layer
    ss[1] = view(lib, sink=FAKE * 64, ring=FAKE * 80)
    for bad in (dict(sink=FAKE * 16, ring=FAKE * 48), dict(sink=FAKE * 48, ring=FAKE * 32), dict(sink=FAKE, ring=FAKE * 48),
                dict(sink=FAKE * 48, ring=FAKE * 2)):                  # one buffer twice, or another layer's source
        ds[1] = view(lib, **bad)
        assert lib.sjk_hip_fork(ds, ss, 2, 128, 200, None) == ARG, bad


def test_copy_blocks_refusals(lib):
    ids = lambda *x: (C.c_uint32 * len(x))(*x)  # noqa: E731

    def call(src, dst, d=FAKE, s=FAKE, nd=8, ns=8, layers=2, dl=8 * 64, sl=8 * 64, block=64, n=None):
        return lib.sjk_hip_copy_blocks(d, dl, nd, s, sl, ns, layers, block, src, dst, len(src) if n is None else n, None)

    assert call(ids(0), ids(1), n=0) == 0 and call(ids(0), ids(1), layers=0) == 0
    assert call(ids(0), ids(8)) == ARG and call(ids(8), ids(0)) == ARG and call(ids(0), ids(0xFFFFFFFF)) == ARG
    assert call(ids(0, 1), ids(2, 2)) == ARG                           # a destination twice
    assert call(ids(0), ids(0)) == ARG and call(ids(0, 1), ids(1, 2)) == ARG   # a destination that is a source
    assert call(ids(0), ids(1), d=None) == ARG and call(ids(0), ids(1), s=None) == ARG
    assert call(None, ids(1), n=1) == ARG and call(ids(1), None, n=1) == ARG
    assert call(ids(0), ids(1), layers=-1) == ARG and call(ids(0), ids(1), block=0) == ARG
    for bad in (dict(d=FAKE + 2, s=FAKE + 2), dict(block=62), dict(dl=513, sl=513)):
        assert call(ids(0), ids(1), **bad) == ARG, bad
    assert call(ids(0), ids(1), dl=7 * 64, sl=7 * 64) == ARG           # layers that overlap
    assert call(ids(0), ids(1), s=FAKE + 64) == ARG                    # slabs that overlap without being one
    assert call(ids(0), ids(1), sl=9 * 64) == ARG


def test_sequence_calls_refuse_nothing_at_all(lib):
    s = sjk.Seq()
    assert lib.sjk_hip_seq_fork(None, None, 0, None, None) == ARG
    assert lib.sjk_hip_seq_fork(C.byref(s), C.byref(s), 0, None, None) == ARG
    assert lib.sjk_hip_pool_compact(None, None, 0, None, None) == ARG
    p = sjk.Pool()
    assert lib.sjk_hip_pool_compact(C.byref(p), None, 0, None, None) == ARG
    assert lib.sjk_hip_pool_refs(None, 0) == 0 and lib.sjk_hip_pool_refs(C.byref(p), 0) == 0
