"""Attention of drafted nodes and the acceptance of a path (sjk_hip_attend_tree, sjk_hip_accept; their batch, descriptor and sequence
forms) on the GPU: outputs against attention in 64 bits over the device's own rows, moved rows byte for byte."""
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


@pytest.fixture(scope="module")
def lib():
    return sjk.load()


@pytest.fixture
def dev():
    d = sjk.Device()
    yield d
    d.sync()
    d.free_all()


def queries(rng, n_q, n_head, D):
    return (rng.standard_normal((n_q, n_head, D)) * rng.lognormal(0, 0.4, (1, n_head, 1))).astype(np.float32)


def tree(rng, n, width=6):
    """[n][n] ancestors and self of a random tree"""
    a = np.eye(n, dtype=bool)
    for i in range(n):
        p = i - 1 - int(rng.integers(0, width))
        if p >= 0:
            a[i] |= a[p]
    return a


def words(mask, junk=None):
    """the bit words of mask [n_q][n]; junk fills the bits past the nodes"""
    n_q, n = mask.shape
    w = -(-n // 64)
    b = np.zeros((n_q, w * 64), bool)
    if junk is not None:
        b[:] = junk.integers(0, 2, b.shape).astype(bool)
    b[:, :n] = mask
    return np.packbits(b.reshape(n_q, w, 64), axis=-1, bitorder="little").view(np.uint64).reshape(n_q, w)


def run(lib, dev, view, B, base, mask, q, t=sjk.F32, scale=None, junk=None):
    n_q, n_head, D = q.shape
    out = Out(dev, q.size, t)
    sjk.check(lib.sjk_hip_attend_tree(C.byref(view), B, base, mask.shape[1], n_q, n_head, dev.put(q), scale or D ** -0.5,
                                      dev.put(words(mask, junk)), t, out.at, None), "attend_tree")
    return out


def seen_of(mask, base, H):
    n_q, n = mask.shape
    s = np.concatenate([np.ones((n_q, base), bool), mask], 1)
    return np.broadcast_to(s[:, None], (n_q, H, base + n))


BODIES = [(4, 4, 0), (3, 3, 0), (2, 4, 0), (3, 3, 1), (2, 2, 1)]


@pytest.mark.parametrize("D,H,per", [(128, 2, 5), (256, 1, 4)])
@pytest.mark.parametrize("bits,staging,sink_type", [(b, s, 0) for b in BODIES for s in (0, 1)] + [(BODIES[0], 0, 1)])
def test_trees(lib, dev, D, H, per, bits, staging, sink_type):
    """trees from one node to several words and tiles, rows that see no node, the last level asking alone, bits past the nodes"""
    rng = np.random.default_rng(bits[0] + 3 * bits[1] + D)
    ctx = Ctx(lib, dev, D, H, bits, staging, sink_type, n_groups=3, tail=170, seed=4)
    for base, n, n_q in ((ctx.B, 1, 1), (ctx.B + 1, 7, 7), (ctx.B + 16, 16, 3), (ctx.B + 37, 67, 67), (ctx.B + 30, 130, 9), (ctx.B, 64, 20)):
        K, V = ctx.rows(base + n)
        mask = tree(rng, n)[n - n_q:]
        if n_q > 2:
            mask[1] = False
        q = queries(rng, n_q, H * per, D)
        want, tol = attention(q, K, V, seen_of(mask, base, H), D ** -0.5)
        for t in (sjk.F32, sjk.F16, sjk.BF16):
            got = run(lib, dev, ctx.view, ctx.B, base, mask, q, t, junk=rng).get().reshape(q.shape)
            check(got, want, tol, t, (base, n, n_q, t))
            if t == sjk.F32:
                check_norm(got, want, 1e-5 if not bits[2] else 3e-4, (base, n, n_q))
    ctx.close()


@pytest.mark.parametrize("staging,sink_type", [(0, 0), (1, 0), (0, 1)])
@pytest.mark.parametrize("D", [128, 256])
def test_short_contexts(lib, dev, D, staging, sink_type):
    """no context at all (a row without nodes is zero), nodes inside the sink, across its end, and across the end of the ring"""
    rng = np.random.default_rng(D)
    H, per = 1, 3
    ctx = Ctx(lib, dev, D, H, (4, 4, 0), staging, sink_type, tail=380, seed=6)
    for base, n in ((0, 1), (0, 20), (5, 30), (100, 28), (100, 29), (120, 60), (128, 17), (301, 40)):
        K, V = ctx.rows(base + n, B=S)
        mask = tree(rng, n, 3)
        mask[0] = False
        q = queries(rng, n, H * per, D)
        want, tol = attention(q, K, V, seen_of(mask, base, H), D ** -0.5)
        got = run(lib, dev, ctx.view, 0 if base < S else S, base, mask, q).get().reshape(q.shape)
        check(got, want, tol, sjk.F32, (base, n))
        if base == 0:
            assert (got[0] == 0).all()
    ctx.close()
    ctx = Ctx(lib, dev, D, H, (4, 4, 0), staging, sink_type, n_groups=9, tail=200, seed=6)       # the ring has wrapped
    assert (ctx.B - S) % ctx.L.cap + 200 > ctx.L.cap or (ctx.B - S) // ctx.L.cap != (ctx.N - S) // ctx.L.cap or ctx.B - S > ctx.L.cap
    K, V = ctx.rows(ctx.N)
    mask = tree(rng, 180)
    q = queries(rng, 180, H * per, D)
    want, tol = attention(q, K, V, seen_of(mask, ctx.N - 180, H), D ** -0.5)
    check(run(lib, dev, ctx.view, ctx.B, ctx.N - 180, mask, q).get().reshape(q.shape), want, tol, sjk.F32)
    ctx.close()


@pytest.mark.parametrize("n_q,per,H", [(40, 8, 2), (64, 4, 4), (33, 16, 1)])
def test_many_rows(lib, dev, n_q, per, H):
    """more rows than a launch takes, and than the kernels for few rows take"""
    rng = np.random.default_rng(n_q)
    D = 128
    ctx = Ctx(lib, dev, D, H, (4, 4, 0), n_groups=4, tail=150, seed=8)
    K, V = ctx.rows(ctx.N)
    base = ctx.N - n_q
    mask = tree(rng, n_q)
    mask[5] = False
    q = queries(rng, n_q, H * per, D)
    want, tol = attention(q, K, V, seen_of(mask, base, H), D ** -0.5)
    for t in (sjk.F32, sjk.F16, sjk.BF16):
        got = run(lib, dev, ctx.view, ctx.B, base, mask, q, t).get().reshape(q.shape)
        # weights of 16-bit outputs may be rounded to fp16 once (2^-12 of each weight)
        check(got, want, tol + (0 if t == sjk.F32 else 2.0 ** -11 * np.abs(V).max()), t, t)
    ctx.close()


@pytest.mark.parametrize("D,H,per,staging,sink_type,n_groups,tail,base,n,n_q", [
    (128, 1, 4, 0, 0, 0, 70, 0, 70, 70),             # no context: rows without nodes are zero
    (256, 1, 8, 1, 0, 0, 150, 100, 50, 33),          # nodes across the sink's end
    (128, 2, 3, 0, 1, 0, 300, 125, 175, 90),
    (256, 2, 2, 0, 0, 3, 170, 0, 131, 131),          # several words a row
    (128, 1, 16, 1, 0, 9, 200, 61, 129, 16),         # the ring has wrapped
    (128, 8, 4, 0, 0, 2, 140, 5, 97, 64),
])
def test_rows_of_a_ubatch(lib, dev, D, H, per, staging, sink_type, n_groups, tail, base, n, n_q):
    """256 rows per head and more (BF16 outputs: the 32-row kernel), eager and captured"""
    rng = np.random.default_rng(n * n_q)
    ctx = Ctx(lib, dev, D, H, (4, 4, 0), staging, sink_type, n_groups=n_groups, tail=tail, seed=12)
    base += ctx.B if n_groups else 0
    B = ctx.B if n_groups else 0 if base < S else S
    K, V = ctx.rows(base + n, B=max(B, S))
    mask = tree(rng, n)[n - n_q:]
    mask[[0, 7, n_q - 1]] = False
    q = queries(rng, n_q, H * per, D)
    want, tol = attention(q, K, V, seen_of(mask, base, H), D ** -0.5)
    bits = {}
    for t in (sjk.F16, sjk.BF16):
        bits[t] = run(lib, dev, ctx.view, B, base, mask, q, t, junk=rng).bits()
        # weights of 16-bit outputs may be rounded to fp16 once (half a step of each), times values up to twice the largest off the zero point
        got = parts.values(bits[t], t).reshape(q.shape)
        check(got, want, tol + 2.0 ** -10 * np.abs(V).max(), t, t)
        if base == 0:
            assert (got[[0, 7, n_q - 1]] == 0).all()
    st, desc = dev.stream(), dev.put(descriptor(0, 0, 0))
    dq, dm = dev.put(q), dev.put(words(mask))
    out = Out(dev, q.size, sjk.BF16)
    n_max = base + n + 5
    if B == 0 and n_max > S + ctx.L.cap:
        n_max = S + ctx.L.cap
    g = Graph(dev, st, [lambda: lib.sjk_hip_attend_tree_dyn(C.byref(ctx.view), desc, n_max, n, n_q, H * per, dq, D ** -0.5, dm, sjk.BF16, out.at, st)])
    for d, ok in (((B, 0, base), 1), ((B, 0, -1), 0), ((B, 9, base), 1), ((B, 0, n_max - n + 1), 0), ((S + 64, 0, base), 0), ((B, 0, base), 1)):
        dev.upload(desc, descriptor(*d))
        run(lib, dev, ctx.view, B, base, mask, q, sjk.BF16).bits()         # eager work on the same workspace between the replays
        g.replay()
        if ok:
            assert np.array_equal(out.bits(), bits[sjk.BF16]), d
        else:
            assert np.isnan(out.get()).all(), d
    g.close()
    ctx.close()


@pytest.mark.parametrize("D,H,n_q,per,n_groups", [(128, 4, 64, 3, 260), (256, 8, 40, 2, 310)])
def test_long_contexts_of_some_rows(lib, dev, D, H, n_q, per, n_groups):
    """64 rows and more on contexts that are long enough for the 32-row kernel, against the FP32 output"""
    rng = np.random.default_rng(n_q)
    ctx = Ctx(lib, dev, D, H, (4, 4, 0), n_groups=n_groups, tail=150, seed=14)
    assert n_q * per * H * ctx.N >= 24 << 20
    most = max(np.abs(ctx.rows(ctx.N)[1]).max(), 1)
    base = ctx.N - n_q
    mask = tree(rng, n_q)
    mask[9] = False
    q = queries(rng, n_q, H * per, D)
    want = run(lib, dev, ctx.view, ctx.B, base, mask, q).get()
    for t in (sjk.F16, sjk.BF16):
        check(run(lib, dev, ctx.view, ctx.B, base, mask, q, t).get(), want, 2.0 ** -10 * most, t, t)
    ctx.close()


def test_a_chain_is_causal_attention(lib, dev):
    rng = np.random.default_rng(2)
    D, H = 256, 2
    ctx = Ctx(lib, dev, D, H, (4, 4, 0), n_groups=5, tail=77, seed=9)
    q = queries(rng, 4, 8, D)
    got = run(lib, dev, ctx.view, ctx.B, ctx.N - 4, np.tril(np.ones((4, 4), bool)), q).get()
    out = dev.alloc(q.nbytes)
    sjk.check(lib.sjk_hip_attend(C.byref(ctx.view), ctx.B, ctx.N, ctx.N - 4, 4, 8, dev.put(q), D ** -0.5, out, None), "attend")
    dev.sync()
    want = dev.get(out, q.nbytes, np.float32)
    assert np.abs(got - want).max() <= 1e-3 + 1e-3 * np.abs(want).max()
    ctx.close()


@pytest.mark.parametrize("staging,sink_type,base", [(0, 0, 400), (1, 0, 400), (0, 0, 60), (0, 1, 60), (1, 0, 118)])
@pytest.mark.parametrize("n_q", [12, 48])
def test_unseen_nodes_stay_out(lib, dev, staging, sink_type, base, n_q):
    """infinities and NaNs in the rows of some nodes: rows that do not see them keep their bits, those that do are not finite"""
    rng = np.random.default_rng(base + staging)
    D, H, per = 128, 1, 6
    ctx = Ctx(lib, dev, D, H, (4, 4, 0), staging, sink_type, tail=base + 60, seed=10)
    v, B = ctx.view, S if base >= S else 0
    mask = tree(rng, n_q, 4)
    q = queries(rng, n_q, H * per, D)
    for t in (sjk.F32, sjk.BF16):
        clean = run(lib, dev, v, B, base, mask, q, t).bits().reshape(n_q, -1)
        bad_nodes = [1, 5, n_q - 2]
        saved = []
        for node, x in zip(bad_nodes, (0x7C00, 0x7E00, 0xFC00)):
            p = base + node
            f16 = p < S and sink_type == 0 or staging == 1
            size = 4 * D if (p < S and sink_type == 0) else 2 * v.stage_bytes
            at = v.sink + p * H * size if p < S else v.ring + ((p - S) % v.cap) * H * size
            old = dev.get(C.c_void_p(at), size, np.uint8)
            saved.append((at, old))
            new = old.copy().view(np.uint16)
            if f16:
                new[[3, D + 70]] = x                 # a key's channel and a value's
            else:
                new[[0, size // 4]] = x              # the key's block norm and the value's
            dev.upload(C.c_void_p(at), new)
        got = run(lib, dev, v, B, base, mask, q, t).bits().reshape(n_q, -1)
        hit = mask[:, bad_nodes].any(1)
        assert hit.any() and not hit.all()
        assert np.array_equal(got[~hit], clean[~hit])
        assert not np.isfinite(parts.values(got[hit].ravel(), t).reshape(hit.sum(), -1)).all(1).any()
        for at, old in saved:
            dev.upload(C.c_void_p(at), old)
        dev.sync()
    ctx.close()


def test_batch_and_descriptor_forms(lib, dev):
    """a batch against its single calls, a captured graph replayed over several bases with eager work between, refused descriptors"""
    rng = np.random.default_rng(40)
    D, H, per, n, n_q = 128, 2, 4, 21, 9
    ctxs = [Ctx(lib, dev, D, H, (3, 3, 1), n_groups=k, tail=t, seed=50 + k) for k, t in ((4, 60), (0, 90), (1, 100))]
    mask = tree(rng, n)[n - n_q:]
    q = queries(rng, n_q, H * per, D)
    dq, dm = dev.put(q), dev.put(words(mask))
    jobs = (sjk.TreeJob * 3)()
    outs = [Out(dev, q.size, sjk.F32) for _ in ctxs]
    for j, c, o in zip(jobs, ctxs, outs):
        j.v, j.B, j.base, j.d_seen, j.d_q, j.d_out = c.view, (c.B if c.n_groups else 0), c.N - n, dm, dq, o.at
    sjk.check(lib.sjk_hip_attend_tree_batch(jobs, 3, n, n_q, H * per, D ** -0.5, sjk.F32, None), "batch")
    for j, c, o in zip(jobs, ctxs, outs):
        one = run(lib, dev, c.view, j.B, j.base, mask, q).get()
        assert np.abs(o.get() - one).max() <= 3e-5 * np.abs(one).max()          # another split of the same sums
    for c in ctxs[:2]:
        st = dev.stream()
        desc, out = dev.put(descriptor(0, 0, 0)), Out(dev, q.size, sjk.F16)
        B = c.B if c.n_groups else 0
        n_max = (c.B if c.n_groups else S) + c.L.cap
        g = Graph(dev, st, [lambda: lib.sjk_hip_attend_tree_dyn(C.byref(c.view), desc, n_max, n, n_q, H * per, dq, D ** -0.5, dm, sjk.F16, out.at, st)])
        for base in (c.N - n, c.N - n - 1, c.N - n - 17, c.N - n):
            dev.upload(desc, descriptor(B, -7, base))                          # N is not read
            if c.n_groups == 0:
                dev.upload(desc, descriptor(B, 0, base))
            d = descriptor(B, 0, base)
            dev.upload(desc, d)
            dev.sync()
            g.replay()
            assert np.array_equal(out.bits(), run(lib, dev, c.view, B, base, mask, q, sjk.F16).bits()), base
        for bad in ((B, 0, -1), (-1, 0, c.N - n), (S + 64, 0, c.N - n), (S + G * 40, 0, c.N - n), (B, 0, n_max - n + 1)):
            dev.upload(desc, descriptor(*bad))
            dev.sync()
            g.replay()
            assert np.isnan(out.get()).all(), bad
        g.close()
    for x in ctxs:
        x.close()


# ---- accept ----

def accept_ref(sink, ring, S_, cap, base, path, to_half):
    """rows moved one after the other; to_half(ring row): its values as an fp16 sink row, or None where the formats agree"""
    for i, p in enumerate(path):
        a, b = base + p, base + i
        row = sink[a] if a < S_ else ring[(a - S_) % cap]
        if a >= S_ > b and to_half is not None:
            row = to_half(row)
        if b < S_:
            sink[b] = row
        else:
            ring[(b - S_) % cap] = row


@pytest.mark.parametrize("D,H,staging,sink_type", [(128, 1, 0, 0), (128, 3, 0, 0), (256, 2, 0, 0), (128, 2, 1, 0), (256, 1, 0, 1)])
def test_accepted_rows(lib, dev, D, H, staging, sink_type):
    """every place of a tree (sink, across its end, ring, across the ring's end), paths from none to longer than a turn of the kernel's,
    paths that end early, several layers; every other byte as it was"""
    rng = np.random.default_rng(D + H + staging)
    cap, NL = 256, 3
    sb = 2 * D if staging else D // 128 * 98
    ring_row = H * 2 * sb
    sink_row = H * 4 * D if sink_type == 0 else ring_row

    def to_half(row):
        blocks = row.reshape(H, 2, D // 128, 98)
        x = np.empty((H, 2, D), np.float32)
        dp, fp = dev.put(np.ascontiguousarray(row)), dev.alloc(2 * H * D * 4)
        sjk.check(lib.sjk_hip_unstage(0, dp, sb, fp, D, 2 * H, None), "unstage")
        dev.sync()
        x = dev.get(fp, 2 * H * D * 4, np.float32)
        dev.free(dp)
        dev.free(fp)
        assert blocks.shape[0] == H
        return x.astype(np.float16).view(np.uint8)

    mixed = sink_row != ring_row
    desc = dev.put(descriptor(0, 0, 0))
    for base, n, path in ((500, 16, [0, 2, 3, 9, 15]), (500, 16, []), (500, 1, [0]), (S + 5 * cap - 9, 40, [1, 5, 8, 9, 20, 38, 39]), (3, 60, [2, 3, 50]),
                          (70, 120, [0, 4, 57, 58, 70, 71, 100, 119]), (S - 1, 9, [1, 2, 8]), (S - 30, 200, list(range(3, 200, 2))),
                          (9000, 220, list(range(1, 220, 1))), (9000, 220, sorted(rng.choice(220, 150, replace=False).tolist())), (S, 30, [29])):
        sinks = rng.integers(0, 256, (NL, S, sink_row), dtype=np.uint8)
        rings = rng.integers(0, 256, (NL, cap, ring_row), dtype=np.uint8)
        if not staging:                                              # block norms that are numbers
            rings.reshape(NL, cap, H * 2 * (D // 128), 98)[..., 1] &= 0x3F
        views = (sjk.View * NL)()
        for il in range(NL):
            v = views[il]
            v.lay = sjk.layout(D, G, 4, 4, 0)
            v.n_head_kv, v.staging, v.sink_type, v.S, v.cap, v.stage_bytes = H, staging, sink_type, S, cap, sb
            v.sink, v.ring = dev.put(sinks[il]).value, dev.put(rings[il]).value
        for il in range(NL):
            accept_ref(sinks[il], rings[il], S, cap, base, path, to_half if mixed and not staging else None)
        for form in (0, 1):
            # entries behind the path's end do not count
            d_path = dev.put(np.array(path + [-1, n, 0], np.int32))
            k = len(path) + 3
            if form == 0:
                rc = lib.sjk_hip_accept(views, NL, base, n, d_path, k, None)
                got = [(dev.get(C.c_void_p(v.sink), S * sink_row, np.uint8), dev.get(C.c_void_p(v.ring), cap * ring_row, np.uint8)) for v in views]
            else:
                # again, from the descriptor: what it makes of the rows now there
                for il in range(NL):
                    accept_ref(sinks[il], rings[il], S, cap, base, path, to_half if mixed and not staging else None)
                dev.upload(desc, descriptor(0, 0, base))
                rc = lib.sjk_hip_accept_dyn(views, NL, desc, n, d_path, k, None)
                dev.sync()
                got = [(dev.get(C.c_void_p(v.sink), S * sink_row, np.uint8), dev.get(C.c_void_p(v.ring), cap * ring_row, np.uint8)) for v in views]
            assert rc == 0
            for il in range(NL):
                assert np.array_equal(got[il][0], sinks[il].ravel()), (base, n, form, il)
                assert np.array_equal(got[il][1], rings[il].ravel()), (base, n, form, il)
        dev.upload(desc, descriptor(0, 0, -1))
        sjk.check(lib.sjk_hip_accept_dyn(views, NL, desc, n, d_path, k, None), "accept")
        dev.sync()
        assert np.array_equal(dev.get(C.c_void_p(views[0].ring), cap * ring_row, np.uint8), rings[0].ravel())


def test_accept_in_many_layers(lib, dev):
    """more layers than a launch takes, rows past 4 GiB of a ring"""
    rng = np.random.default_rng(1)
    D, H, cap, NL = 128, 2, 128, 131
    sb = 98
    rings = rng.integers(0, 256, (NL, cap, H * 2 * sb), dtype=np.uint8)
    buf = dev.put(rings)
    sink = dev.alloc(S * H * 4 * D)
    views = (sjk.View * NL)()
    for il in range(NL):
        v = views[il]
        v.lay = sjk.layout(D, G, 4, 4, 0)
        v.n_head_kv, v.S, v.cap, v.stage_bytes = H, S, cap, sb
        v.sink, v.ring = sink.value, buf.value + il * cap * H * 2 * sb
    path = [3, 4, 90]
    sjk.check(lib.sjk_hip_accept(views, NL, 1000, 100, dev.put(np.array(path, np.int32)), 3, None), "accept")
    dev.sync()
    for i, p in enumerate(path):
        rings[:, (1000 + i - S) % cap] = rings[:, (1000 + p - S) % cap]
    assert np.array_equal(dev.get(buf, rings.nbytes, np.uint8), rings.ravel())
    D, H = 256, 8
    entry = H * 2 * 2 * D
    cap = (5 << 30) // entry
    ring = dev.alloc(cap * entry, zero=False)
    v = views[0]
    v.lay = sjk.layout(D, G, 4, 4, 0)
    v.n_head_kv, v.staging, v.S, v.cap, v.stage_bytes, v.ring = H, 1, S, cap, 2 * D, ring.value
    base = S + cap - 30
    a, b = (rng.integers(0, 256, entry, dtype=np.uint8) for _ in range(2))
    dev.upload(ring, a, offset=(cap - 10) * entry)
    dev.upload(ring, b, offset=4 * entry)
    sjk.check(lib.sjk_hip_accept(views, 1, base, 64, dev.put(np.array([20, 34], np.int32)), 2, None), "accept")
    dev.sync()
    assert np.array_equal(dev.get(C.c_void_p(ring.value + (cap - 30) * entry), entry, np.uint8), a)
    assert np.array_equal(dev.get(C.c_void_p(ring.value + (cap - 29) * entry), entry, np.uint8), b)


def test_a_drafted_step_equals_plain_steps(lib, dev):
    """A sequence that drafts a tree, attends it, accepts a path and goes on holds the bytes of one that stored the accepted tokens
    one after the other, and each accepted node's attention is that of the plain step; twice, and then no node accepted."""
    rng = np.random.default_rng(77)
    D, H, NL, per = 128, 2, 2, 2
    heads = H * per
    cfg = lib.sj_kvarn_config_default(D, H, 1024, 64)
    cfg.tail, cfg.tail_max = 128, 256
    draft, plain = sjk.Seq(), sjk.Seq()
    for s in (draft, plain):
        sjk.check(lib.sj_kvarn_seq_init(C.byref(s), C.byref(cfg), NL, None), "seq")
    c = sjk.RopeConfig(D, 0, 1e4, 1.0, 0, 0, 0, None)
    turns, ms = np.zeros(D // 2), C.c_float()
    assert lib.sjk_rope_turns(C.byref(c), turns.ctypes.data_as(C.POINTER(C.c_double)), C.byref(ms)) == 0
    m = sjk.Qkv()
    row = (heads + 2 * H) * D
    m.type, m.n_head, m.rotate_qk, m.rotate_v, m.eps = sjk.F32, heads, 1, 1, 1e-6
    m.q_pos = m.k_pos = m.v_pos = row
    m.q_head = m.k_head = m.v_head = D
    m.rope = sjk.Rope(0, D, 0, 1.0, dev.put(turns).value)

    def store(s, pos0, x, pos):
        """x [NL][n][heads + 2 H][D] of tokens at turn positions pos; the queries of every layer"""
        n = x.shape[1]
        sjk.check(lib.sjk_hip_seq_begin_ubatch(C.byref(s), pos0, n, None), "begin")
        qs = []
        for il in range(NL):
            p, q = dev.put(x[il]), dev.alloc(n * heads * D * 4)
            job = sjk.SeqQkvJob(C.pointer(s), pos0, dev.put(np.asarray(pos, np.int32)), p, p.value + heads * D * 4, p.value + (heads + H) * D * 4, q)
            sjk.check(lib.sjk_hip_seq_store_qkv_batch(C.byref(job), 1, il, n, C.byref(m), None), "store_qkv")
            qs.append(q)
        return qs

    prompt = rng.standard_normal((NL, 500, heads + 2 * H, D)).astype(np.float32)
    for s in (draft, plain):
        for p in range(0, 500, 50):
            store(s, p, prompt[:, p:p + 50], np.arange(p, p + 50))
    n = 20
    for turn, path in enumerate(([0, 3, 4, 11], [2], [])):
        base = draft.n
        assert base == plain.n
        x = rng.standard_normal((NL, n, heads + 2 * H, D)).astype(np.float32)
        anc = np.eye(n, dtype=bool)
        depth = np.zeros(n, int)
        for i in range(n):                                           # the path is a branch of the tree
            par = path[path.index(i) - 1] if i in path and path.index(i) else -1 if i in path or i < 2 else int(rng.integers(0, i))
            if par >= 0:
                anc[i] |= anc[par]
                depth[i] = depth[par] + 1
        qs = store(draft, base, x, base + depth)
        outs = []
        for il in range(NL):
            o = Out(dev, n * heads * D, sjk.F32)
            job = sjk.SeqTreeJob(C.pointer(draft), base, dev.put(words(anc)), qs[il], o.at)
            sjk.check(lib.sjk_hip_seq_attend_tree_batch(C.byref(job), 1, il, n, n, heads, D ** -0.5, sjk.F32, None), "tree")
            outs.append(o.get().reshape(n, heads, D))
        sjk.check(lib.sjk_hip_seq_accept(C.byref(draft), base, (C.c_int32 * max(1, len(path)))(*path), len(path), None), "accept")
        assert draft.n == base + len(path)
        for i, node in enumerate(path):
            qp = store(plain, base + i, x[:, node:node + 1], [base + i])
            for il in range(NL):
                o = dev.alloc(heads * D * 4)
                sjk.check(lib.sjk_hip_seq_attend(C.byref(plain), il, base + i, 1, heads, qp[il], D ** -0.5, o, None), "attend")
                dev.sync()
                want = dev.get(o, heads * D * 4, np.float32).reshape(heads, D)
                assert np.abs(outs[il][node] - want).max() <= 1e-3 + 1e-3 * np.abs(want).max()
        dev.sync()
        assert draft.pol.B == plain.pol.B
        sizes = [lib.sj_kvarn_seq_state_size(C.byref(s)) for s in (draft, plain)]
        assert sizes[0] == sizes[1]
        states = []
        for s in (draft, plain):
            buf, w = np.zeros(sizes[0], np.uint8), C.c_size_t()
            sjk.check(lib.sj_kvarn_seq_state_write(C.byref(s), buf.ctypes.data, sizes[0], C.byref(w)), "state")
            states.append(buf)
        assert np.array_equal(*states), turn
    P = C.c_int32 * 3
    assert lib.sjk_hip_seq_accept(C.byref(draft), draft.n - 3, P(0, 0, 1), 2, None) == -100
    assert lib.sjk_hip_seq_accept(C.byref(draft), draft.n - 3, P(1, 0, 2), 2, None) == -100
    assert lib.sjk_hip_seq_accept(C.byref(draft), draft.n - 3, P(0, 1, 3), 3, None) == -100
    assert lib.sjk_hip_seq_accept(C.byref(draft), draft.n + 1, P(), 0, None) == -100
    assert lib.sjk_hip_seq_accept(C.byref(draft), draft.pol.B - 1, P(), 0, None) == (-100 if draft.pol.B > S else 0)
    for s in (draft, plain):
        lib.sj_kvarn_seq_free(C.byref(s))
