"""Listed groups and drafted nodes at their edges, on the GPU: lists longer than the sealed groups are many, descriptors that hold more
than the view or less than the call reads, selections whose jobs share a workspace, long paths and many layers of an acceptance."""
import ctypes as C
import sys

import numpy as np
import pytest

import cabi
import parts
import test_gpu_groups as groups
import test_gpu_tree as trees
from parts import G, S, Ctx, Graph, Out, attention, check, descriptor

sys.path.insert(0, cabi.PKG)
import sjk  # noqa: E402

pytestmark = pytest.mark.gpu
TYPES = (sjk.F32, sjk.F16, sjk.BF16)
CAPACITY = -109


@pytest.fixture(scope="module")
def lib():
    return sjk.load()


@pytest.fixture
def dev():
    d = sjk.Device()
    yield d
    d.sync()
    d.free_all()


# ---- lists ----

def named(entries, n):
    """the groups that a list names: entries of [0, n) that are above the entry before them"""
    return [g for j, g in enumerate(entries) if 0 <= g < n and (j == 0 or g > entries[j - 1])]


def spread(rng, n, top):
    """an ascending list of `top` entries whose groups stand anywhere among repeats, -1 before the first"""
    at = np.sort(rng.choice(top, min(n, top), replace=False))
    x = np.full(top, -1)
    for g, i in enumerate(at):
        x[i:] = g
    return x.tolist()


@pytest.mark.parametrize("D,H,per", [(128, 2, 4), (256, 1, 5)])
@pytest.mark.parametrize("bits", groups.BODIES, ids=groups.IDS)
def test_lists_longer_than_the_groups(lib, dev, D, H, per, bits):
    """every entry of a list counts, wherever it stands: -1 and repeats ahead of it, long runs of them, whole lists of them; eager, captured
    and in a batch"""
    rng = np.random.default_rng(D + 10 * bits[0] + bits[1])
    n_q = 2
    st = dev.stream()
    for n, tops in ((1, (2, 40)), (2, (3, 300)), (3, (5, 6, 700))):
        ctx = Ctx(lib, dev, D, H, bits, n_groups=n, tail=21, seed=40 + n)
        K, V = ctx.rows(ctx.N)
        qpos0 = ctx.N - n_q
        for top in tops:
            rows = [spread(rng, n, top) for _ in range(n_q * H)]
            if top == 6:
                rows[1] = [-1] * top
            rows[0] = [-1] * (top - n) + list(range(n))               # the groups behind everything else
            rows[-1] = [0] * (top - n + 1) + list(range(1, n))
            pick = [rows[i * H:(i + 1) * H] for i in range(n_q)]
            lists = [[named(x, n) for x in r] for r in pick]
            assert lists[0][0] == list(range(n)) and lists[-1][-1] == list(range(n))
            sel = np.array(pick, np.int32)
            q = groups.queries(rng, n_q, H * per, D)
            want, tol = attention(q, K, V, groups.seen_of(ctx, lists, n_q, qpos0), D ** -0.5)
            for t in TYPES:
                eager = groups.attend(lib, dev, ctx.view, ctx.B, ctx.N, qpos0, q, sel, t).bits()
                check(parts.values(eager, t).reshape(q.shape), want, tol, t, (n, top, t))
                out, desc = Out(dev, q.size, t), dev.put(descriptor(ctx.B, ctx.N, qpos0))
                dq, ds = dev.put(q), dev.put(sel)
                g = Graph(dev, st, [lambda: lib.sjk_hip_attend_groups_dyn(C.byref(ctx.view), desc, ctx.N + 9, n_q, H * per, dq, D ** -0.5, ds, top,
                                                                          t, out.at, st)])
                for _ in range(3):
                    g.replay()
                    assert np.array_equal(out.bits(), eager), (n, top, t)
                    groups.attend(lib, dev, ctx.view, ctx.B, ctx.N, qpos0, q, sel, t).bits()
                g.close()
                jobs = (sjk.GroupsJob * 3)()
                outs = [Out(dev, q.size, t) for _ in jobs]
                for j, o in zip(jobs, outs):
                    j.v, j.B, j.N, j.qpos0, j.d_q, j.d_sel, j.d_out = ctx.view, ctx.B, ctx.N, qpos0, dq, ds, o.at
                sjk.check(lib.sjk_hip_attend_groups_batch(jobs, 3, n_q, H * per, D ** -0.5, top, t, None), "batch")
                for o in outs:
                    check(o.get().reshape(q.shape), want, tol, t, (n, top, t))
        ctx.close()


@pytest.mark.parametrize("bits", [(4, 4, 0), (3, 3, 0), (3, 3, 1)])
@pytest.mark.parametrize("H,per,n_q", [(1, 17, 2), (2, 40, 1), (48, 1, 3), (1, 1, 1), (1, 128, 1)])
def test_head_layouts(lib, dev, H, per, n_q, bits):
    """more query heads per KV head than a tile has rows, many KV heads, and one; lists and trees of them"""
    rng = np.random.default_rng(H + per)
    D, n = 128, 5
    ctx = Ctx(lib, dev, D, H, bits, n_groups=n, tail=33, seed=60)
    K, V = ctx.rows(ctx.N)
    q = groups.queries(rng, n_q, H * per, D)
    pick = [[np.sort(rng.choice(n, 3, replace=False)).tolist() for _ in range(H)] for _ in range(n_q)]
    want, tol = attention(q, K, V, groups.seen_of(ctx, pick, n_q, ctx.N - n_q), D ** -0.5)
    mask = trees.tree(rng, n_q, 2)
    tree_want, tree_tol = attention(q, K, V, trees.seen_of(mask, ctx.N - n_q, H), D ** -0.5)
    for t in TYPES:
        got = groups.attend(lib, dev, ctx.view, ctx.B, ctx.N, ctx.N - n_q, q, np.array(pick, np.int32), t).get().reshape(q.shape)
        check(got, want, tol, t, t)
        tree_got = trees.run(lib, dev, ctx.view, ctx.B, ctx.N - n_q, mask, q, t).get().reshape(q.shape)
        check(tree_got, tree_want, tree_tol, t, t)
        if t == sjk.F32:
            parts.check_norm(got, want, 1e-5)
            parts.check_norm(tree_got, tree_want, 1e-5)
    ctx.close()


# ---- descriptors ----

@pytest.mark.parametrize("bits", [(4, 4, 0), (3, 3, 0), (2, 2, 1)])
def test_a_tree_does_not_read_the_descriptors_n(lib, dev, bits):
    """any N, below zero too, gives the same rows, those of the eager call, in every kernel behind the call"""
    rng = np.random.default_rng(bits[0])
    D, H, per = 128, 1, 8
    ctx = Ctx(lib, dev, D, H, bits, n_groups=3, tail=70, seed=90)
    st, desc = dev.stream(), dev.put(descriptor(0, 0, 0))
    n_max = ctx.B + ctx.L.cap
    for n in (9, 40):                                # 72 and 320 rows a head: the 32-row kernel takes the latter's BF16 output
        base = ctx.N - n
        mask, q = trees.tree(rng, n), groups.queries(rng, n, H * per, D)
        dq, dm = dev.put(q), dev.put(trees.words(mask))
        for t in TYPES:
            out = Out(dev, q.size, t)
            g = Graph(dev, st, [lambda: lib.sjk_hip_attend_tree_dyn(C.byref(ctx.view), desc, n_max, n, n, H * per, dq, D ** -0.5, dm, t, out.at, st)])
            first = None
            for N in (ctx.N, -7, 0, 2 ** 31 - 1, -2 ** 31, ctx.N):
                want = trees.run(lib, dev, ctx.view, ctx.B, base, mask, q, t).bits()
                dev.upload(desc, descriptor(ctx.B, N, base))
                dev.sync()
                g.replay()
                got = out.bits()
                first = got if first is None else first
                assert np.array_equal(got, first), (n, t, N)
                # an eager call of many tiles may cut them into other launches (other partial sums, within their roundings)
                if n == 9 or bits[2] or t == sjk.BF16:
                    assert np.array_equal(got, want), (n, t, N)
                else:
                    check(parts.values(got, t), parts.values(want, t), 2.0 ** -12 * np.abs(parts.values(want, t)).max(), t, (n, t, N))
            g.close()
    ctx.close()


def test_descriptors_past_the_ring(lib, dev):
    """more staged positions than the ring holds: lists of -1 where the attention gives NaN rows, and the last place that fits"""
    rng = np.random.default_rng(3)
    D, H, per, top, n = 128, 2, 3, 4, 9
    lay = sjk.layout(D, G, 3, 3, 0)
    v = groups.fake_view(lib, dev, D, H, (3, 3, 0), groups.records(rng, lay, n, H), np.arange(n))
    B, cap = S + G * n, 256
    q = groups.queries(rng, 3, H * per, D)
    st = dev.stream()
    desc, dq, sel, out = dev.put(descriptor(0, 0, 0)), dev.put(q), dev.alloc(3 * H * top * 4), Out(dev, q.size, sjk.F32)
    g = Graph(dev, st, [lambda: lib.sjk_hip_select_groups_dyn(C.byref(v), desc, 1 << 20, 3, H * per, dq, top, sel, st),
                        lambda: lib.sjk_hip_attend_groups_dyn(C.byref(v), desc, 1 << 20, 3, H * per, dq, D ** -0.5, sel, top, sjk.F32, out.at, st)])
    lists = lambda: dev.get(sel, 3 * H * top * 4, np.int32).reshape(3, H, top)  # noqa: E731
    for N, qpos0, ok in ((B + cap, B + cap - 3, 1), (B + cap + 1, B + cap - 2, 0), (1 << 20, B + 700, 0), (B + cap + 900, B + 5, 1),
                         (B + 20, B + 700, 1), ((1 << 20) + 1, B + 5, 0), (B + 3, 2 ** 31 - 1, 1), (B + cap + 1, B + cap - 2, 0)):
        dev.upload(desc, descriptor(B, N, qpos0))
        dev.sync()
        g.replay()
        if ok:
            want = groups.select(lib, dev, v, B, N, qpos0, q, top, H)
            assert (want >= 0).all() and np.array_equal(lists(), want), (N, qpos0)
            assert np.array_equal(out.bits(), groups.attend(lib, dev, v, B, N, qpos0, q, want).bits()), (N, qpos0)
        else:
            assert (lists() == -1).all() and np.isnan(out.get()).all(), (N, qpos0)
    # nothing sealed: the list is -1 in any case, and a tail past the ring gives NaN rows
    for N, qpos0, ok in ((S + cap, S + cap - 3, 1), (S + cap + 1, S + cap - 2, 0), (S + cap + 1, S, 1)):
        dev.upload(desc, descriptor(S, N, qpos0))
        dev.sync()
        g.replay()
        assert (lists() == -1).all()
        assert np.isfinite(out.get()).all() if ok else np.isnan(out.get()).all(), (N, qpos0)
    g.close()


# ---- selections ----

def test_selections_that_share_a_workspace(lib, dev):
    """jobs of one workspace whose scores do not fit it together, beside jobs of their own: every list as alone. A job that does not fit at
    all: no list of the batch is written."""
    rng = np.random.default_rng(8)
    D, H, n, top = 128, 2, 900, 20
    lay = sjk.layout(D, G, 3, 3, 0)
    recs = groups.records(rng, lay, 200, H)
    head, slot = 4096 + ((H * D * 8 + 255) & ~255), 16 * (D + 2) * 4
    shared = dev.alloc(head + 64 * slot)
    own = dev.alloc(head + 64 * slot)
    views, q, lengths = [], [], []
    for k in range(37):
        v = groups.fake_view(lib, dev, D, H, (3, 3, 0), recs, rng.integers(0, 200, n), work=False)
        # the shared one holds the scores of 2 positions of 900 groups and 2 heads, the other of many
        v.work, v.work_bytes = (own.value, head + 64 * slot) if k in (4, 20) else (shared.value, head + -(-(2 * H * n * 8) // slot) * slot)
        views.append(v)
        q.append(groups.queries(rng, 5, 8, D))
        lengths.append(15 if k in (3, 30) else n - 20 * (k % 5))
    dqs = [dev.put(x) for x in q]
    sel = dev.put(np.full((37, 5, H, top), 77, np.int32))
    size = 5 * H * top * 4
    jobs = (sjk.GroupsJob * 37)()
    for k in range(37):
        B = S + G * lengths[k]
        jobs[k] = sjk.GroupsJob(views[k], B, B + 5, B, dqs[k], C.c_void_p(sel.value + k * size), None)
    want = np.stack([groups.select(lib, dev, views[k], jobs[k].B, jobs[k].N, jobs[k].qpos0, q[k], top, H) for k in range(37)])
    sjk.check(lib.sjk_hip_select_groups_batch(jobs, 37, 5, 8, top, None), "batch")
    dev.sync()
    assert np.array_equal(dev.get(sel, 37 * size, np.int32).reshape(want.shape), want)
    dev.upload(sel, np.full((37, 5, H, top), 77, np.int32))
    jobs[36].v.work_bytes = head + slot
    assert lib.sjk_hip_select_groups_batch(jobs, 37, 5, 8, top, None) == CAPACITY
    dev.sync()
    assert (dev.get(sel, 37 * size, np.int32) == 77).all()


# ---- acceptance ----

def staged_views(dev, D, H, cap, NL, rings, sink):
    """views of layers whose rings stand one after the other at `rings`"""
    views = (sjk.View * NL)()
    for il, v in enumerate(views):
        v.lay = sjk.layout(D, G, 4, 4, 0)
        v.n_head_kv, v.S, v.cap, v.stage_bytes = H, S, cap, D // 128 * 98
        v.sink, v.ring = sink.value, rings.value + il * cap * H * 2 * v.stage_bytes
    return views


@pytest.mark.parametrize("NL", [160, 161, 321])
def test_accept_in_more_layers_than_a_launch_takes(lib, dev, NL):
    rng = np.random.default_rng(NL)
    D, H, cap = 128, 1, 128
    rings = rng.integers(0, 256, (NL, cap, H * 2 * 98), dtype=np.uint8)
    buf, sink = dev.put(rings), dev.alloc(S * H * 4 * D)
    views = staged_views(dev, D, H, cap, NL, buf, sink)
    path = [1, 7, 8, 60, 99]
    sjk.check(lib.sjk_hip_accept(views, NL, 1000, 100, dev.put(np.array(path, np.int32)), len(path), None), "accept")
    dev.sync()
    for i, p in enumerate(path):
        rings[:, (1000 + i - S) % cap] = rings[:, (1000 + p - S) % cap]
    assert np.array_equal(dev.get(buf, rings.nbytes, np.uint8), rings.ravel())


@pytest.mark.parametrize("base", [9000, S - 20])
@pytest.mark.parametrize("sink_type", [0, 1])
def test_accept_of_long_paths(lib, dev, base, sink_type):
    """a path on the device past what a workgroup holds of it, through the ring's end, and from the ring into the sink"""
    rng = np.random.default_rng(base + sink_type)
    D, H, cap, n, NL = 128, 2, 4096, 4000, 2
    row = H * 2 * 98
    rings = rng.integers(0, 256, (NL, cap, row), dtype=np.uint8)
    rings.reshape(NL, cap, H * 2, 98)[..., 1] &= 0x3F                       # block norms that are numbers
    sink_row = row if sink_type else H * 4 * D
    sinks = rng.integers(0, 256, (NL, S, sink_row), dtype=np.uint8)
    for path in (list(range(1, n)), np.sort(rng.choice(n, 2500, replace=False)).tolist()):
        buf, sink = dev.put(rings), dev.put(sinks)
        views = staged_views(dev, D, H, cap, NL, buf, sink)
        for il, v in enumerate(views):
            v.sink_type, v.sink = sink_type, sink.value + il * S * sink_row
        want_s, want_r = sinks.copy(), rings.copy()

        def to_half(x):
            dp, fp = dev.put(np.ascontiguousarray(x)), dev.alloc(2 * H * D * 4)
            sjk.check(lib.sjk_hip_unstage(0, dp, 98, fp, D, 2 * H, None), "unstage")
            dev.sync()
            return dev.get(fp, 2 * H * D * 4, np.float32).astype(np.float16).view(np.uint8)

        for il in range(NL):
            trees.accept_ref(want_s[il], want_r[il], S, cap, base, path, None if sink_type else to_half)
        sjk.check(lib.sjk_hip_accept(views, NL, base, n, dev.put(np.array(path + [3], np.int32)), len(path) + 1, None), "accept")
        dev.sync()
        assert np.array_equal(dev.get(sink, sinks.nbytes, np.uint8), want_s.ravel())
        assert np.array_equal(dev.get(buf, rings.nbytes, np.uint8), want_r.ravel())


def test_a_sequence_accepts_long_paths_of_many_nodes(lib, dev):
    """paths past what one launch's arguments hold, of nodes past 65,535"""
    rng = np.random.default_rng(6)
    D, H, n_pos = 128, 1, 66100
    cfg = lib.sj_kvarn_config_default(D, H, 70000, 256)
    cfg.tail, cfg.tail_max = 128, 128 * 520
    s = sjk.Seq()
    sjk.check(lib.sj_kvarn_seq_init(C.byref(s), C.byref(cfg), 1, None), "seq")
    v = lib.sjk_layer_view(C.byref(s.layers[0]))
    assert v.cap >= n_pos - S
    dk, dv = (dev.put(rng.standard_normal((n_pos, H, D)).astype(np.float32)) for _ in range(2))
    for p in range(0, n_pos, 4096):
        m = min(4096, n_pos - p)
        sjk.check(lib.sjk_hip_seq_store(C.byref(s), 0, p, m, dk.value + p * H * D * 4, dv.value + p * H * D * 4, 1, None), "store")
    dev.sync()
    row = H * 2 * 98
    for base, pick in ((200, np.r_[[0, 2], 65530 + np.arange(0, 300, 7)]), (150, np.sort(rng.choice(65600, 1500, replace=False))),
                       (400, np.arange(700) * 90 + 1)):
        s.n = n_pos
        path = pick.tolist()
        ring = dev.get(C.c_void_p(v.ring), v.cap * row, np.uint8).reshape(v.cap, row)
        for i, p in enumerate(path):
            ring[(base + i - S) % v.cap] = ring[(base + p - S) % v.cap]
        sjk.check(lib.sjk_hip_seq_accept(C.byref(s), base, (C.c_int32 * len(path))(*path), len(path), None), "accept")
        dev.sync()
        assert s.n == base + len(path)
        assert np.array_equal(dev.get(C.c_void_p(v.ring), v.cap * row, np.uint8), ring.ravel()), base
    lib.sj_kvarn_seq_free(C.byref(s))


# ---- precision ----

@pytest.mark.parametrize("D,seed,flat", [(128, 1, 1.0), (128, 2, 0.5), (128, 3, 0.25), (256, 4, 0.5), (256, 5, 0.25)])
def test_fp16_outputs_are_rounded_once(lib, dev, D, seed, flat):
    """4/4 records, 384 listed groups and a tree of 64 rows, weights from uneven to nearly equal: an error at most a tenth above that of
    the exact result rounded to fp16 (what is computed before the rounding is then within 0.46 of the rounding's error)"""
    rng = np.random.default_rng(seed)
    H, per, n = 2, 4, 400
    lay = sjk.layout(D, G, 4, 4, 0)
    recs = groups.records(rng, lay, n, H)
    # values around zero: a row over many of them is far smaller than they are
    vs = recs[:, :, lay.v_scale:lay.v_scale + 2 * G].copy().view(np.float16).astype(np.float64)
    recs[:, :, lay.v_zero:lay.v_zero + 2 * G] = (-7.5 * vs).astype(np.float16).view(np.uint8)
    v = groups.fake_view(lib, dev, D, H, (4, 4, 0), recs, rng.permutation(n))
    B, N = S + G * n, S + G * n + 200
    K, V = Ctx.rows(_Rows(lib, dev, D, H), N, view=v, B=B)
    q = groups.queries(rng, 2, H * per, D)
    sel = np.stack([np.sort(rng.choice(n, 384, replace=False)) for _ in range(2 * H)]).reshape(2, H, 384)
    seen = np.zeros((2, H, N), bool)
    for i in range(2):
        seen[i, :, :S] = seen[i, :, B:N - 1 + i] = True
        for h in range(H):
            for g in sel[i, h]:
                seen[i, h, S + G * g:S + G * (g + 1)] = True
    scale = D ** -0.5 * flat
    want, _ = attention(q, K, V, seen, scale)
    got = groups.attend(lib, dev, v, B, N, N - 2, q, sel, sjk.F16, scale).get().reshape(q.shape)
    plain = np.linalg.norm(want.astype(np.float16) - want)
    assert np.linalg.norm(got - want) <= 1.1 * plain, np.linalg.norm(got - want) / plain
    mask = np.eye(64, dtype=bool)
    q = groups.queries(rng, 64, H * per, D)
    seen = np.broadcast_to(np.concatenate([np.ones((64, N - 64), bool), mask], 1)[:, None], (64, H, N))[::9]
    want, _ = attention(q[::9], K, V, seen, scale)
    got = trees.run(lib, dev, v, B, N - 64, mask, q, sjk.F16, scale).get().reshape(q.shape)[::9]
    plain = np.linalg.norm(want.astype(np.float16) - want)
    assert np.linalg.norm(got - want) <= 1.1 * plain, np.linalg.norm(got - want) / plain


@pytest.mark.parametrize("D", [128, 256])
@pytest.mark.parametrize("bits", groups.BODIES, ids=groups.IDS)
def test_fp32_outputs_of_every_body(lib, dev, D, bits):
    """every body holds the same bound, the trellis bodies too: independent roundings, 2 D of a score's partial sums of U of about twice a
    score's size each, make 2e-6 of a weight and of a result"""
    rng = np.random.default_rng(D + bits[0])
    H, per, n, n_q = 2, 4, 24, 3
    ctx = Ctx(lib, dev, D, H, bits, n_groups=n, tail=300, seed=3)
    K, V = ctx.rows(ctx.N)
    q = groups.queries(rng, n_q, H * per, D)
    for listed in (range(n), range(1, n, 3)):
        sel = np.broadcast_to(np.array(listed, np.int32), (n_q, H, len(listed)))
        want, _ = attention(q, K, V, groups.seen_of(ctx, [[listed] * H] * n_q, n_q, ctx.N - n_q), D ** -0.5)
        got = groups.attend(lib, dev, ctx.view, ctx.B, ctx.N, ctx.N - n_q, q, sel).get().reshape(q.shape)
        parts.check_norm(got, want, 1e-5, len(listed))
    mask = trees.tree(rng, 20)
    q = groups.queries(rng, 20, H * per, D)
    want, _ = attention(q, K, V, trees.seen_of(mask, ctx.N - 20, H), D ** -0.5)
    parts.check_norm(trees.run(lib, dev, ctx.view, ctx.B, ctx.N - 20, mask, q).get().reshape(q.shape), want, 1e-5, "tree")
    ctx.close()


class _Rows:
    """what Ctx.rows asks of a context"""

    def __init__(self, lib, dev, D, H):
        self.lib, self.dev, self.D, self.H, self.view, self.B = lib, dev, D, H, None, 0
