"""Selection of sealed groups and attention over them (sjk_hip_select_groups, sjk_hip_attend_groups; their batch, descriptor and
sequence forms) on the GPU: lists against the same bounds in extended precision, outputs against attention in 64 bits over the
device's own rows (sjk_hip_kv_rows)."""
import ctypes as C
import sys

import numpy as np
import pytest

import cabi
import parts
from parts import G, S, Ctx, Graph, Out, attention, check, check_norm, descriptor

sys.path.insert(0, cabi.PKG)
import sjk  # noqa: E402

pytestmark = pytest.mark.gpu
LD = np.longdouble
BODIES = [(4, 4, 0), (3, 3, 0), (4, 2, 0), (2, 3, 0), (3, 3, 1), (3, 2, 1), (2, 2, 1)]
IDS = ["%d/%d%s" % (a, b, "t" if c else "s") for a, b, c in BODIES]


@pytest.fixture(scope="module")
def lib():
    return sjk.load()


@pytest.fixture
def dev():
    d = sjk.Device()
    yield d
    d.sync()
    d.free_all()


def code_range(bits, body):
    if not body:
        return 0.0, float(2 ** bits - 1)
    text = open(cabi.ROOT + "/include/sjk_tables.h").read()
    part = text.split("#define SJK_CB%d_K_INIT {" % bits)[1].split("}")[0]
    cb = np.array([int(x, 16) for x in part.replace("\\", " ").replace(",", " ").split()], np.uint16).view(np.float16).astype(float)
    return cb.min(), cb.max()


def scores(lay, recs, q, H):
    """bounds [n_q][H][n] of records [n][H][bytes] in extended precision, and how far a sum in 64 bits may be off"""
    n, D = recs.shape[0], lay.D
    half = lambda at, m: recs[:, :, at:at + 2 * m].copy().view(np.float16).astype(LD)  # noqa: E731
    ks, kz, kt = half(lay.k_scale, D), half(lay.k_zero, D), half(lay.k_tok, G)
    lib = sjk.load()
    idx = np.array([lib.sj_kvarn_k_ch_idx(C.byref(lay), d) for d in range(D)])
    ks, kz = ks[:, :, idx], kz[:, :, idx]
    c0, c1 = code_range(lay.bits_k, lay.body)
    per = q.shape[1] // H
    out, err = np.empty((q.shape[0], H, n), LD), np.empty((q.shape[0], H, n))
    for i in range(q.shape[0]):
        for h in range(H):
            best = np.full(n, -np.inf, LD)
            e = np.zeros(n)
            for j in range(per):
                x = q[i, h * per + j].astype(LD)
                w = np.where(x > 0, x * LD(c1), x * LD(c0))
                a, b = kz[:, h] * x, ks[:, h] * w
                u = a.sum(-1) + b.sum(-1)
                hi, lo = kt[:, h].max(-1), kt[:, h].min(-1)
                s = np.where(np.isnan(u) | np.isnan(kt[:, h]).any(-1), LD("nan"), np.where(u >= 0, u * hi, u * lo))
                best = np.where(np.isnan(s) | np.isnan(best), LD("nan"), np.maximum(best, s))
                e = np.maximum(e, ((np.abs(a).sum(-1) + np.abs(b).sum(-1)) * np.abs(hi) * (2 * D + 8)).astype(float) * 2.0 ** -53)
            out[i, h], err[i, h] = best, e
    return out, err


def check_list(got, s, err, top, what=""):
    """the `top` largest scores, of equal ones the lower group, ascending; scores that 64-bit sums cannot tell apart may change places"""
    n = len(s)
    k = min(top, n)
    assert (got[k:] == -1).all() and (np.diff(got[:k]) > 0).all() and (k == 0 or (got[0] >= 0 and got[k - 1] < n)), (what, got)
    key = np.where(np.isnan(s), LD(np.inf), s)
    want = np.sort(np.lexsort((np.arange(n), -key))[:k])
    if np.array_equal(got[:k], want):
        return
    inside = np.zeros(n, bool)
    inside[got[:k]] = True
    worst, best = np.where(inside)[0][np.argmin(key[inside])], np.where(~inside)[0][np.argmax(key[~inside])]
    gap = key[best] - key[worst]
    assert 0 < gap <= err[best] + err[worst] and np.setxor1d(got[:k], want).size <= 2, (what, gap, got, want)


def record_bytes(ctx, view, ids):
    b = ctx.dev.get(C.c_void_p(view.body), (max(ids) + 1) * ctx.H * view.lay.bytes, np.uint8)
    return b.reshape(-1, ctx.H, view.lay.bytes)[ids]


def select(lib, dev, view, B, N, qpos0, q, top, H, n_q=None):
    n_q, n_head = q.shape[0], q.shape[1]
    dq, sel = dev.put(q), dev.put(np.full(n_q * H * top + 2, 77, np.int32))
    sjk.check(lib.sjk_hip_select_groups(C.byref(view), B, N, qpos0, n_q, n_head, dq, top, C.c_void_p(sel.value + 4), None), "select")
    dev.sync()
    x = dev.get(sel, 4 * (n_q * H * top + 2), np.int32)
    assert x[0] == 77 and x[-1] == 77
    return x[1:-1].reshape(n_q, H, top)


def queries(rng, n_q, n_head, D):
    return (rng.standard_normal((n_q, n_head, D)) * rng.lognormal(0, 0.4, (1, n_head, 1))).astype(np.float32)


@pytest.mark.parametrize("D", [128, 256])
@pytest.mark.parametrize("bits", BODIES, ids=IDS)
def test_lists_of_every_body(lib, dev, D, bits):
    """real records, query heads per KV head from 1 to past a tile, lists from one group to more than there are; a bound is one"""
    rng = np.random.default_rng(D + 10 * bits[0] + bits[1])
    ctx = Ctx(lib, dev, D, 2, bits, n_groups=9, tail=17, seed=3)
    recs = record_bytes(ctx, ctx.view, list(range(9)))
    K, _ = ctx.rows(ctx.B)
    for n_q, per, top in ((1, 1, 1), (1, 4, 4), (3, 5, 8), (2, 17, 3), (5, 2, 9), (1, 16, 40), (1, 40, 2)):
        q = queries(rng, n_q, 2 * per, D)
        s, err = scores(ctx.view.lay, recs, q, 2)
        got = select(lib, dev, ctx.view, ctx.B, ctx.N, ctx.N - n_q, q, top, 2)
        for i in range(n_q):
            for h in range(2):
                check_list(got[i, h], s[i, h], err[i, h], top, (n_q, per, top, i, h))
                real = (q[i, h * per:(h + 1) * per].astype(float) @ K[h][S:].T).reshape(per, 9, G).max((0, 2))
                # (decoded keys have two roundings to fp32)
                assert (real <= s[i, h].astype(float) + 4 * parts.U * np.abs(q[i, h * per:(h + 1) * per]).sum() * np.abs(K[h]).max()).all()
    ctx.close()


def fake_view(lib, dev, D, H, bits, recs, blocks, work=True):
    """a view over given record bytes [n][H][bytes] and a block table"""
    v = sjk.View()
    v.lay = sjk.layout(D, G, *bits)
    v.n_head_kv, v.staging, v.sink_type, v.S, v.cap = H, 1, 0, S, 256
    v.stage_bytes = 2 * D
    rng = np.random.default_rng(5)
    v.sink = dev.put(rng.standard_normal((S, H, 2, D)).astype(np.float16)).value
    v.ring = dev.put(rng.standard_normal((256, H, 2, D)).astype(np.float16)).value
    v.body, v.blocks = dev.put(recs).value, dev.put(np.asarray(blocks, np.uint32)).value
    if work:
        v.work_bytes = lib.sjk_hip_workspace_bytes(C.byref(v.lay), H)
        v.work = dev.alloc(v.work_bytes).value
    return v


def records(rng, lay, n, H):
    """random codes, scales as a seal makes them"""
    r = rng.integers(0, 256, (n, H, lay.bytes), dtype=np.uint8)
    put = lambda at, x: r[:, :, at:at + 2 * x.shape[-1]].__setitem__(Ellipsis, x.astype(np.float16).view(np.uint8))  # noqa: E731
    top = 2.0 ** lay.bits_k
    ks = 4 / top * rng.lognormal(0, 0.3, (n, H, lay.D))
    put(lay.k_scale, ks)
    put(lay.k_zero, rng.standard_normal((n, H, lay.D)) - 0.5 * top * ks)
    put(lay.k_tok, rng.lognormal(0, 0.1, (n, H, G)))
    put(lay.v_ch, rng.lognormal(0, 0.2, (n, H, lay.D)))
    vs = 4 / 2.0 ** lay.bits_v * rng.lognormal(0, 0.2, (n, H, G))
    put(lay.v_scale, vs)
    put(lay.v_zero, -0.5 * 2.0 ** lay.bits_v * vs)
    return r


@pytest.mark.parametrize("n", [1, 15, 16, 17, 1023, 1024, 1025, 9001])
def test_lists_of_many_groups(lib, dev, n):
    """paged, with blocks that several groups share (equal scores: the lower group), across the pass sizes of the list's kernel"""
    rng = np.random.default_rng(n)
    D, H = 128, 2
    lay = sjk.layout(D, G, 3, 3, 0)
    phys = min(n, 700)
    recs = records(rng, lay, phys, H)
    blocks = rng.integers(0, phys, n)
    v = fake_view(lib, dev, D, H, (3, 3, 0), recs, blocks)
    q = queries(rng, 2, 6, D)
    s, err = scores(lay, recs, q, H)
    s, err = s[:, :, blocks], err[:, :, blocks]
    for top in sorted({1, 2, min(64, n), max(1, n - 1), n, n + 3}):
        got = select(lib, dev, v, S + G * n, S + G * n + 40, S + G * n + 38, q, top, H)
        for i in range(2):
            for h in range(H):
                check_list(got[i, h], s[i, h], err[i, h], top, (top, i, h))


def test_lists_of_equal_and_strange_scores(lib, dev):
    """all scores equal; zero queries (both zeros); scores that are not numbers first; infinities; negative token scales"""
    rng = np.random.default_rng(9)
    D, H, n = 256, 1, 40
    lay = sjk.layout(D, G, 4, 4, 0)
    one = records(rng, lay, 1, H)
    v = fake_view(lib, dev, D, H, (4, 4, 0), one, np.zeros(n, int))
    B = S + G * n
    q = queries(rng, 1, 4, D)
    assert np.array_equal(select(lib, dev, v, B, B + 1, B, q, 7, H)[0, 0], np.arange(7))
    recs = records(rng, lay, n, H)
    v = fake_view(lib, dev, D, H, (4, 4, 0), recs, rng.permutation(n))
    z = np.zeros_like(q)
    z[0, 1::2] = -0.0
    assert np.array_equal(select(lib, dev, v, B, B + 1, B, z, 5, H)[0, 0], np.arange(5))
    half = lambda g, at, i, x: recs[g, 0, at + 2 * i:at + 2 * i + 2].__setitem__(Ellipsis, np.array([x], np.float16).view(np.uint8))  # noqa: E731
    half(31, lay.k_tok, 100, np.nan)
    half(7, lay.k_zero, 3, np.nan)
    half(20, lay.k_scale, 9, np.inf)
    half(12, lay.k_zero, 200, -np.inf)
    half(15, lay.k_tok, 0, -3.0)
    v = fake_view(lib, dev, D, H, (4, 4, 0), recs, np.arange(n))
    q = np.abs(q) * np.float32(0.1)
    with np.errstate(invalid="ignore"):
        s, err = scores(lay, recs, q, H)
    got = select(lib, dev, v, B, B + 1, B, q, 9, H)[0, 0]
    assert {31, 7, 20} <= set(got.tolist()) and 12 not in got
    err = np.where(np.isfinite(err), err, 0)
    check_list(got, s[0, 0], err[0, 0], 9)


def test_lists_in_pieces_of_the_workspace(lib, dev):
    """more positions than the workspace holds scores of, and one position too many groups"""
    rng = np.random.default_rng(4)
    D, H, n = 128, 1, 3000
    lay = sjk.layout(D, G, 3, 3, 0)
    recs = records(rng, lay, 300, H)
    blocks = rng.integers(0, 300, n)
    v = fake_view(lib, dev, D, H, (3, 3, 0), recs, blocks)
    B = S + G * n
    q = queries(rng, 70, 2, D)
    whole = select(lib, dev, v, B, B + 70, B, q, 33, H)
    head = 4096 + ((H * D * 8 + 255) & ~255)
    slot = 16 * (D + 2) * 4
    v.work_bytes = head + -(-(20 * n * 8) // slot) * slot
    assert np.array_equal(select(lib, dev, v, B, B + 70, B, q, 33, H), whole)
    v.work_bytes = head + (n * 8 // slot) * slot
    dq, sel = dev.put(q), dev.alloc(70 * 33 * 4)
    assert lib.sjk_hip_select_groups(C.byref(v), B, B + 70, B, 70, 2, dq, 33, sel, None) == -109
    s, err = scores(lay, recs, q, H)
    for i in (0, 19, 20, 69):
        check_list(whole[i, 0], s[i, 0][blocks], err[i, 0][blocks], 33)


def seen_of(ctx, lists, n_q, qpos0):
    seen = np.zeros((n_q, ctx.H, ctx.N), bool)
    for i in range(n_q):
        for h in range(ctx.H):
            seen[i, h, :min(S, qpos0 + i + 1)] = True
            if ctx.N > ctx.B:
                seen[i, h, ctx.B:qpos0 + i + 1] = True
            for g in lists[i][h]:
                seen[i, h, S + G * g:S + G * (g + 1)] = True
    return seen


def attend(lib, dev, view, B, N, qpos0, q, sel, t=sjk.F32, scale=None, stream=None):
    n_q, n_head, D = q.shape
    out = Out(dev, q.size, t)
    sel = np.ascontiguousarray(sel, np.int32)
    sjk.check(lib.sjk_hip_attend_groups(C.byref(view), B, N, qpos0, n_q, n_head, dev.put(q), scale or D ** -0.5, dev.put(sel), sel.shape[-1], t,
                                        out.at, stream), "attend_groups")
    return out


@pytest.mark.parametrize("D,H,per", [(128, 2, 4), (256, 1, 5)])
@pytest.mark.parametrize("bits,staging,sink_type", [(b, 0, 0) for b in BODIES] + [(b, s, k) for b in BODIES[::4] for s, k in ((1, 0), (0, 1))])
def test_attention_over_lists(lib, dev, D, H, per, bits, staging, sink_type):
    """lists of every kind: some, one, all, none, shorter than top, and entries that name no group or come twice"""
    rng = np.random.default_rng(D + bits[0] * 7 + bits[1])
    ctx = Ctx(lib, dev, D, H, bits, staging, sink_type, n_groups=6, tail=41, seed=2)
    K, V = ctx.rows(ctx.N)
    n_q = 3
    q = queries(rng, n_q, H * per, D)
    qpos0 = ctx.N - n_q
    rows = [([1, 4, 5, -1], [1, 4, 5]), ([0, 1, 2, 3, 4, 5], [0, 1, 2, 3, 4, 5]), ([-1, -1], []), ([3], [3]), ([2, 2, 6, 4, 3, 5], [2, 4, 5]),
            ([7, 1 << 30, -5, 0, 0, 5], [0, 5])]
    for k in range(len(rows)):
        # every position and head a list of its own, of one length
        pick = [[rows[(k + i + h) % len(rows)] for h in range(H)] for i in range(n_q)]
        top = max(len(x[0]) for r in pick for x in r)
        sel = np.array([[x[0] + [-1] * (top - len(x[0])) for x in r] for r in pick], np.int32)
        # an entry that is no group: the one behind it has to be above it all the same
        lists = [[[g for j, g in enumerate(x[0]) if 0 <= g < 6 and (j == 0 or g > x[0][j - 1])] for x in r] for r in pick]
        want, tol = attention(q, K, V, seen_of(ctx, lists, n_q, qpos0), D ** -0.5)
        for t in (sjk.F32, sjk.F16, sjk.BF16):
            got = attend(lib, dev, ctx.view, ctx.B, ctx.N, qpos0, q, sel, t).get().reshape(q.shape)
            check(got, want, tol, t, (k, t))
            if t == sjk.F32:
                # independent roundings: 2 D of a score's partial sums, U of about twice a score's size each, make 2e-6 of a weight
                check_norm(got, want, 1e-5 if not bits[2] else 3e-4, k)
    ctx.close()


@pytest.mark.parametrize("D", [128, 256])
@pytest.mark.parametrize("bits", [(4, 4, 0), (3, 3, 0), (3, 3, 1)])
def test_unlisted_groups_stay_out(lib, dev, D, bits):
    """records that are not listed hold infinities and NaNs, the first group's among them; entries that name no group beside them"""
    rng = np.random.default_rng(D + bits[0])
    H, per, n = 2, 4, 9
    ctx = Ctx(lib, dev, D, H, bits, n_groups=n, tail=30, seed=31)
    lay = ctx.view.lay
    q = queries(rng, 2, H * per, D)
    sel = np.array([[[-1, 2, 3, 40, 7, -1], [-1, -1, -1, -1, -1, -1]], [[-3, -1, 5, 5, -1, 8], [1, 0, 2, 1, -1, 3]]], np.int32)
    clean = [attend(lib, dev, ctx.view, ctx.B, ctx.N, ctx.N - 2, q, sel, t).bits() for t in (sjk.F32, sjk.F16, sjk.BF16)]
    raw = dev.get(C.c_void_p(ctx.view.body), n * H * lay.bytes, np.uint8).reshape(n, H, lay.bytes)
    bad = raw.copy()
    for g in (0, 4, 6):
        for h in range(H):
            if (g, h) in ((0, 1),):
                continue
            for at, x in ((lay.k_scale, 0x7C00), (lay.k_zero, 0x7E00), (lay.k_tok, 0xFC00), (lay.v_ch, 0x7E00), (lay.v_scale, 0x7C00), (lay.v_zero, 0xFE00)):
                bad[g, h, at + 10:at + 12] = np.array([x], np.uint16).view(np.uint8)
    dev.upload(C.c_void_p(ctx.view.body), bad)
    for t, want in zip((sjk.F32, sjk.F16, sjk.BF16), clean):
        assert np.array_equal(attend(lib, dev, ctx.view, ctx.B, ctx.N, ctx.N - 2, q, sel, t).bits(), want), t
    # the first group where it is an entry's own
    sel[0, 0] = [0, 2, 3, 4, 7, 8]
    got = parts.values(attend(lib, dev, ctx.view, ctx.B, ctx.N, ctx.N - 2, q, sel).bits(), sjk.F32).reshape(2, H, per, D)
    assert not np.isfinite(got[0, 0]).any() and np.isfinite(got[0, 1]).all() and np.isfinite(got[1]).all()
    dev.upload(C.c_void_p(ctx.view.body), raw)
    ctx.close()


def test_all_groups_listed_is_the_whole_context(lib, dev):
    """against sjk_hip_attend (its own tolerance), at a length where every workgroup has several records; and no groups at all"""
    rng = np.random.default_rng(3)
    D, H = 128, 2
    lay = sjk.layout(D, G, 4, 4, 0)
    recs = records(rng, lay, 200, H)
    n = 2500
    v = fake_view(lib, dev, D, H, (4, 4, 0), recs, rng.integers(0, 200, n))
    B, N = S + G * n, S + G * n + 200
    q = queries(rng, 2, 8, D)
    sel = np.broadcast_to(np.arange(n, dtype=np.int32), (2, H, n))
    got = attend(lib, dev, v, B, N, N - 2, q, sel).get()
    out = dev.alloc(q.nbytes)
    sjk.check(lib.sjk_hip_attend(C.byref(v), B, N, N - 2, 2, 8, dev.put(q), D ** -0.5, out, None), "attend")
    dev.sync()
    dense = dev.get(out, q.nbytes, np.float32)
    assert np.abs(got - dense).max() <= 1e-3 + 1e-3 * np.abs(dense).max()
    for B2, N2 in ((0, 5), (S, 77), (S, S + 100)):      # nothing sealed: the list adds nothing
        got = attend(lib, dev, v, B2, N2, N2 - 2, q, sel[:, :, :3]).get()
        sjk.check(lib.sjk_hip_attend(C.byref(v), B2, N2, N2 - 2, 2, 8, dev.put(q), D ** -0.5, out, None), "attend")
        dev.sync()
        assert np.abs(got - dev.get(out, q.nbytes, np.float32)).max() <= 1e-5


def test_batch_and_descriptor_forms(lib, dev):
    """a batch of different contexts is its single calls bit for bit, and so is a captured graph of selection and attention,
    replayed over several contexts with eager work between; descriptors that do not hold give lists of -1 and NaN rows"""
    rng = np.random.default_rng(12)
    D, H, per, top = 256, 2, 4, 3
    scale = D ** -0.5
    ctxs = [Ctx(lib, dev, D, H, (4, 4, 0), n_groups=n, tail=t, seed=20 + n) for n, t in ((7, 30), (2, 90), (0, 60), (5, 1))]
    qs = [queries(rng, 1, H * per, D) for _ in ctxs]
    single = []
    for c, q in zip(ctxs, qs):
        B = c.B if c.n_groups else S
        sel = select(lib, dev, c.view, B, c.N, c.N - 1, q, top, H)
        single.append((sel, attend(lib, dev, c.view, B, c.N, c.N - 1, q, sel, sjk.BF16).bits()))
    jobs = (sjk.GroupsJob * len(ctxs))()
    outs, sels = [], []
    for j, c, q in zip(jobs, ctxs, qs):
        sels.append(dev.alloc(H * top * 4))
        outs.append(Out(dev, q.size, sjk.BF16))
        j.v, j.B, j.N, j.qpos0 = c.view, (c.B if c.n_groups else S), c.N, c.N - 1
        j.d_q, j.d_sel, j.d_out = dev.put(q), sels[-1], outs[-1].at
    sjk.check(lib.sjk_hip_select_groups_batch(jobs, len(jobs), 1, H * per, top, None), "select batch")
    sjk.check(lib.sjk_hip_attend_groups_batch(jobs, len(jobs), 1, H * per, scale, top, sjk.BF16, None), "attend batch")
    dev.sync()
    for k in range(len(ctxs)):
        assert np.array_equal(dev.get(sels[k], H * top * 4, np.int32).reshape(1, H, top), single[k][0])
        assert np.abs(outs[k].get() - parts.values(single[k][1], sjk.BF16)).max() <= 2 ** -7 * np.abs(outs[k].get()).max()
    # one graph over one layer's buffers, its context growing
    c = ctxs[0]
    q = qs[0]
    st = dev.stream()
    desc, dq, sel, out = dev.put(descriptor(0, 0, 0)), dev.put(q), dev.alloc(H * top * 4), Out(dev, q.size, sjk.F32)
    n_max = c.B + c.L.cap
    g = Graph(dev, st, [lambda: lib.sjk_hip_select_groups_dyn(C.byref(c.view), desc, n_max, 1, H * per, dq, top, sel, st),
                        lambda: lib.sjk_hip_attend_groups_dyn(C.byref(c.view), desc, n_max, 1, H * per, dq, scale, sel, top, sjk.F32, out.at, st)])
    for B, N in ((c.B, c.N), (c.B, c.B), (c.B, c.B + 3), (S, 40), (c.B, c.N), (S + G * 2, S + G * 2)):
        dev.upload(desc, descriptor(B, N, N - 1))
        dev.sync()
        g.replay()
        got, lst = out.bits(), dev.get(sel, H * top * 4, np.int32).reshape(1, H, top)
        e_sel = select(lib, dev, c.view, B, N, N - 1, q, top, H)
        assert np.array_equal(lst, e_sel)
        assert np.array_equal(got, attend(lib, dev, c.view, B, N, N - 1, q, e_sel).bits()), (B, N)
    for bad in ((c.B + 1, c.N, c.N - 1), (c.B, c.B - 1, c.B - 2), (c.B, c.N, c.B - 3), (-1, 5, 4), (c.B, n_max + 1, n_max), (S, S + c.L.cap + 1, S)):
        dev.upload(desc, descriptor(*bad))
        dev.sync()
        g.replay()
        if bad[:2] != (S, S + c.L.cap + 1):
            assert (dev.get(sel, H * top * 4, np.int32) == -1).all(), bad
            assert np.isnan(out.get()).all(), bad
    dev.upload(desc, descriptor(c.B, c.N, c.N - 1))
    dev.sync()
    g.replay()
    assert np.array_equal(out.bits(), attend(lib, dev, c.view, c.B, c.N, c.N - 1, q, single[0][0]).bits())
    g.close()
    for x in ctxs:
        x.close()


def test_lists_of_a_batch_of_many_lengths(lib, dev):
    """jobs whose groups are all listed need no scores, nor a workspace; the others share theirs"""
    rng = np.random.default_rng(14)
    D, H, top = 128, 2, 20
    lay = sjk.layout(D, G, 3, 3, 0)
    recs = records(rng, lay, 300, H)
    lengths = (300, 5, 0, 77, 20, 21, 150)
    jobs = (sjk.GroupsJob * len(lengths))()
    views = [fake_view(lib, dev, D, H, (3, 3, 0), recs, rng.permutation(300), work=n > top) for n in lengths]
    views[3].work, views[6].work_bytes = views[0].work, views[6].work_bytes
    views[1].work, views[1].work_bytes = dev.alloc(256).value, 256
    q = [queries(rng, 3, 8, D) for _ in lengths]
    sel = dev.put(np.full((len(lengths), 3, H, top), 77, np.int32))
    for k, n in enumerate(lengths):
        B = S + G * n
        jobs[k] = sjk.GroupsJob(views[k], B, B + 3, B, dev.put(q[k]), C.c_void_p(sel.value + 4 * k * 3 * H * top), None)
    sjk.check(lib.sjk_hip_select_groups_batch(jobs, len(lengths), 3, 8, top, None), "batch")
    dev.sync()
    got = dev.get(sel, 4 * len(lengths) * 3 * H * top, np.int32).reshape(len(lengths), 3, H, top)
    for k, n in enumerate(lengths):
        if n <= top:
            assert (got[k] == np.concatenate([np.arange(n), np.full(top - n, -1)])).all(), n
        else:
            B = S + G * n
            assert np.array_equal(got[k], select(lib, dev, views[k], B, B + 3, B, q[k], top, H)), n


@pytest.mark.parametrize("bits", [(3, 3, 0), (4, 4, 0), (3, 3, 1)])
def test_many_short_jobs_beside_a_long_one(lib, dev, bits):
    """jobs on one workspace and on another's: a launch's partials fit each"""
    rng = np.random.default_rng(15)
    D, H, per, top = 128, 8, 2, 30
    long, own = Ctx(lib, dev, D, H, bits, n_groups=30, tail=300, seed=70), Ctx(lib, dev, D, H, bits, tail=40, seed=71)
    short = Ctx(lib, dev, D, H, bits, tail=25, seed=72)
    ctxs = [long] + [short] * 11 + [own]
    jobs, outs, qs = (sjk.GroupsJob * 13)(), [], []
    for k, c in enumerate(ctxs):
        v = sjk.View.from_buffer_copy(c.view)
        if c is short:
            v.work, v.work_bytes = long.view.work, long.view.work_bytes
        q = queries(rng, 1, H * per, D)
        sel = dev.put(np.broadcast_to(np.arange(30, dtype=np.int32), (H, top)).copy())
        outs.append(Out(dev, q.size, sjk.F32))
        qs.append(q)
        jobs[k] = sjk.GroupsJob(v, c.B if c.n_groups else 0, c.N, c.N - 1, dev.put(q), sel, outs[-1].at)
    sjk.check(lib.sjk_hip_attend_groups_batch(jobs, 13, 1, H * per, D ** -0.5, top, sjk.F32, None), "batch")
    for k, c in enumerate(ctxs):
        K, V = c.rows(c.N, B=max(jobs[k].B, S))
        seen = np.ones((1, H, c.N), bool)
        want, tol = attention(qs[k], K, V, seen, D ** -0.5)
        check(outs[k].get().reshape(want.shape), want, tol, sjk.F32, k)
    for c in (long, own, short):
        c.close()


def test_sequences(lib, dev):
    """a decode batch of sequences of one pool: selection and attention of a layer, against the views' calls"""
    rng = np.random.default_rng(30)
    D, H, NL, top = 128, 2, 2, 2
    cfg = lib.sj_kvarn_config_default(D, H, 2048, 64)
    cfg.bits_k, cfg.bits_v, cfg.body, cfg.tail, cfg.tail_max = 3, 3, 1, 128, 256
    pool = sjk.Pool()
    sjk.check(lib.sj_kvarn_pool_init(C.byref(pool), C.byref(cfg), NL, 24), "pool")
    seqs = [sjk.Seq() for _ in range(3)]
    for s, n in zip(seqs, (900, 500, 100)):
        sjk.check(lib.sj_kvarn_seq_init(C.byref(s), C.byref(cfg), NL, C.byref(pool)), "seq")
        for p in range(0, n, 50):
            m = min(50, n - p)
            sjk.check(lib.sjk_hip_seq_begin_ubatch(C.byref(s), p, m, None), "begin")
            for il in range(NL):
                k, v = rng.standard_normal((2, m, H, D)).astype(np.float32)
                sjk.check(lib.sjk_hip_seq_store(C.byref(s), il, p, m, dev.put(k), dev.put(v), 1, None), "store")
    dev.sync()
    q = queries(rng, 1, 4 * H, D)
    jobs = (sjk.SeqGroupsJob * 3)()
    sels, outs = [dev.alloc(H * top * 4) for _ in seqs], [Out(dev, q.size, sjk.F32) for _ in seqs]
    for j, s, a, o in zip(jobs, seqs, sels, outs):
        j.seq, j.pos0, j.d_q, j.d_sel, j.d_out = C.pointer(s), s.n - 1, dev.put(q), a, o.at
    for il in range(NL):
        sjk.check(lib.sjk_hip_seq_select_groups_batch(jobs, 3, il, 1, 4 * H, top, None), "seq select")
        sjk.check(lib.sjk_hip_seq_attend_groups_batch(jobs, 3, il, 1, 4 * H, D ** -0.5, top, sjk.F32, None), "seq attend")
        dev.sync()
        for s, a, o in zip(seqs, sels, outs):
            v = lib.sjk_layer_view(C.byref(s.layers[il]))
            want = select(lib, dev, v, s.pol.B, s.n, s.n - 1, q, top, H)
            assert np.array_equal(dev.get(a, H * top * 4, np.int32).reshape(1, H, top), want)
            ref = attend(lib, dev, v, s.pol.B, s.n, s.n - 1, q, want).get()
            assert np.abs(o.get() - ref).max() <= 1e-5 * np.abs(ref).max()      # another split of the same sums
    assert seqs[0].pol.B > S + 3 * G and seqs[2].pol.B == S
    for s in seqs:
        lib.sj_kvarn_seq_free(C.byref(s))
    lib.sj_kvarn_pool_free(C.byref(pool))
