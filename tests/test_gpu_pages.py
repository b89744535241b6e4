"""Forks, block moves and pool compaction on the GPU (sjk_hip_fork, sjk_hip_copy_blocks, sjk_hip_seq_fork, sjk_hip_pool_refs,
sjk_hip_pool_compact), and the calls that release blocks when some of them are shared.

Bytes against numpy's own slot arithmetic, state streams and attention bit for bit against sequences that were built alone
and truncated (sj_kvarn_seq_truncate, which the oracle's tests pin); what a call does not name stays as it was. The last test
runs everything together, from a projection's rows to the attention of forked sequences on a compacted pool."""
import ctypes as C
import sys

import numpy as np
import pytest

import cabi

sys.path.insert(0, cabi.PKG)
import sjk  # noqa: E402

from test_gpu_async import H, NL, N_HEAD, W, Rows, attend, config, grow, new_pool, new_seq, step, stream_bytes  # noqa: E402
from test_gpu_heads import Proj  # noqa: E402

pytestmark = pytest.mark.gpu
D, S, G = 128, 128, 128
NO = 0xFFFFFFFF


@pytest.fixture(scope="module")
def lib():
    return sjk.load()


@pytest.fixture
def dev():
    d = sjk.Device()
    yield d
    d.sync()
    d.free_all()


def raw_view(lib, dev, host, d, heads, staging, sink_type, cap):
    """a view over buffers of the given bytes"""
    v = sjk.View()
    assert lib.sj_kvarn_layout_init(C.byref(v.lay), d, 128, 4, 4, 0) == 0
    v.n_head_kv, v.staging, v.sink_type, v.S, v.cap = heads, staging, sink_type, S, cap
    v.stage_bytes = lib.sj_kvarn_stage_row_bytes(staging, d)
    v.sink, v.ring = dev.put(host[0]).value, dev.put(host[1]).value
    return v


@pytest.mark.parametrize("d,heads,staging,sink_type", [(128, 1, 0, 0), (256, 4, 0, 0), (128, 3, 1, 0), (128, 2, 0, 1), (256, 1, 1, 1)])
@pytest.mark.parametrize("cap_from,cap_to", [(256, 256), (256, 384), (640, 256)])
def test_fork_of_views(lib, dev, d, heads, staging, sink_type, cap_from, cap_to):
    """every region and wrap: nothing, a part of the sink, one staged position, rings that wrap in the source, in the
    destination and in both at different places, a full ring; 70 layers (two launches)"""
    rng = np.random.default_rng(d + heads + cap_to)
    sb = lib.sj_kvarn_stage_row_bytes(staging, d)
    entry = heads * 2 * sb
    sink_entry = heads * 4 * d if sink_type == 0 else entry
    most = min(cap_from, cap_to)
    for B, N, nl in ((128, 0, 2), (128, 1, 1), (128, 77, 3), (128, 128, 1), (128, 129, 2), (128, 128 + most, 1), (256, 256, 1),
                     (384, 500, 2), (1280, 1280 + most, 2), (128 * 41, 128 * 41 + 201, 70), (128 * 4000000, 128 * 4000000 + 255, 1)):
        hosts = [[(rng.integers(0, 256, S * sink_entry, dtype=np.uint8), rng.integers(0, 256, cap * entry, dtype=np.uint8))
                  for _ in range(nl)] for cap in (cap_from, cap_to)]
        src = (sjk.View * nl)(*[raw_view(lib, dev, h, d, heads, staging, sink_type, cap_from) for h in hosts[0]])
        dst = (sjk.View * nl)(*[raw_view(lib, dev, h, d, heads, staging, sink_type, cap_to) for h in hosts[1]])
        sjk.check(lib.sjk_hip_fork(dst, src, nl, B, N, None), "fork")
        dev.sync()
        pos = np.arange(B, max(N, B))
        for il in range(nl):
            sink, ring = hosts[1][il][0].copy(), hosts[1][il][1].copy().reshape(cap_to, entry)
            sink[:min(N, S) * sink_entry] = hosts[0][il][0][:min(N, S) * sink_entry]
            ring[(pos - S) % cap_to] = hosts[0][il][1].reshape(cap_from, entry)[(pos - S) % cap_from]
            assert np.array_equal(dev.get(C.c_void_p(dst[il].sink), sink.nbytes, np.uint8), sink), (B, N, il)
            assert np.array_equal(dev.get(C.c_void_p(dst[il].ring), ring.nbytes, np.uint8), ring.ravel()), (B, N, il)
            assert np.array_equal(dev.get(C.c_void_p(src[il].ring), cap_from * entry, np.uint8), hosts[0][il][1])
        dev.sync()
        dev.free_all()


@pytest.mark.parametrize("block", [4, 100, 16384, 16388, 17920, 70144])
def test_copy_blocks(lib, dev, block):
    """within a slab and between two of different sizes, one source to several destinations, sizes that end inside a tile,
    several layers with space between them; the rest of the slabs as it was"""
    rng = np.random.default_rng(block)
    nl, na, nb = 3, 23, 40
    la, lb = na * block + 64, nb * block
    a, b = (rng.integers(0, 256, nl * x, dtype=np.uint8) for x in (la, lb))
    da, db = dev.put(a), dev.put(b)

    def ids(x):
        return (C.c_uint32 * len(x))(*[int(i) for i in x])

    def expect(to, lt, frm, lf, src, dst):
        to = to.copy()
        for il in range(nl):
            for i, j in zip(src, dst):
                to[il * lt + j * block:il * lt + (j + 1) * block] = frm[il * lf + i * block:il * lf + (i + 1) * block]
        return to

    src, dst = [0, 22, 5, 5, 5], [39, 0, 7, 8, 20]
    sjk.check(lib.sjk_hip_copy_blocks(db, lb, nb, da, la, na, nl, block, ids(src), ids(dst), 5, None), "copy_blocks")
    dev.sync()
    b = expect(b, lb, a, la, src, dst)
    assert np.array_equal(dev.get(db, b.nbytes, np.uint8), b) and np.array_equal(dev.get(da, a.nbytes, np.uint8), a)
    perm = rng.permutation(na)
    src, dst = perm[:11], perm[11:22]
    sjk.check(lib.sjk_hip_copy_blocks(da, la, na, da, la, na, nl, block, ids(src), ids(dst), 11, None), "copy_blocks")
    dev.sync()
    a = expect(a, la, a, la, src, dst)
    assert np.array_equal(dev.get(da, a.nbytes, np.uint8), a)


def test_pages_past_32_bits(lib, dev):
    """blocks of a slab of 5 GiB and staged rows of a ring of 5 GiB"""
    rng = np.random.default_rng(8)
    block, n = 1 << 20, 5 << 10
    slab = dev.alloc(block * n, zero=False)
    far, near = rng.integers(0, 256, block, dtype=np.uint8), rng.integers(0, 256, block, dtype=np.uint8)
    dev.upload(slab, far, offset=(n - 1) * block)
    dev.upload(slab, near, offset=3 * block)
    src, dst = (C.c_uint32 * 2)(n - 1, 3), (C.c_uint32 * 2)(7, n - 2)
    sjk.check(lib.sjk_hip_copy_blocks(slab, block * n, n, slab, block * n, n, 1, block, src, dst, 2, None), "copy_blocks")
    dev.sync()
    assert np.array_equal(dev.get(C.c_void_p(slab.value + 7 * block), block, np.uint8), far)
    assert np.array_equal(dev.get(C.c_void_p(slab.value + (n - 2) * block), block, np.uint8), near)

    d, heads, small = 256, 8, 256
    entry = heads * 2 * 2 * d
    cap = (5 << 30) // entry
    rows = rng.integers(0, 256, (200, entry), dtype=np.uint8)
    sink = rng.integers(0, 256, S * heads * 4 * d, dtype=np.uint8)
    at = (cap - 300) // 128 * 128                # slot and position of the first staged row
    B = S + at
    views = [raw_view(lib, dev, (sink, rng.integers(0, 256, small * entry, dtype=np.uint8)), d, heads, 1, 0, small) for _ in range(3)]
    views[0].ring, views[0].cap = slab.value, cap
    dev.upload(slab, rows, offset=at * entry)
    sjk.check(lib.sjk_hip_fork(C.byref(views[1]), C.byref(views[0]), 1, B, B + 200, None), "fork")
    dev.sync()
    got = dev.get(C.c_void_p(views[1].ring), small * entry, np.uint8).reshape(small, entry)
    assert at * entry > 1 << 32 and np.array_equal(got[(at + np.arange(200)) % small], rows)
    dev.upload(slab, np.zeros_like(rows), offset=at * entry)
    sjk.check(lib.sjk_hip_fork(C.byref(views[0]), C.byref(views[1]), 1, B, B + 200, None), "fork back")
    dev.sync()
    assert np.array_equal(dev.get(C.c_void_p(slab.value + at * entry), rows.nbytes, np.uint8).reshape(rows.shape), rows)


def test_copy_more_blocks_than_a_launch_holds(lib, dev):
    rng = np.random.default_rng(1)
    n, block = 1500, 64
    a = rng.integers(0, 256, 2 * n * block, dtype=np.uint8)
    d = dev.put(a)
    src, dst = n + rng.permutation(n), rng.permutation(n)
    sjk.check(lib.sjk_hip_copy_blocks(d, 0, 2 * n, d, 0, 2 * n, 1, block, (C.c_uint32 * n)(*src.tolist()), (C.c_uint32 * n)(*dst.tolist()),
                                      n, None), "copy_blocks")
    dev.sync()
    a = a.reshape(2 * n, block)
    a[dst] = a[src]
    assert np.array_equal(dev.get(d, a.nbytes, np.uint8).reshape(a.shape), a)


def test_captured_fork_and_move_replay(lib, dev):
    """both calls carry all they need in the launch: captured once and replayed they copy what the buffers hold then"""
    rng = np.random.default_rng(5)
    hip = dev.hip
    for name, args in (("hipStreamBeginCapture", [C.c_void_p, C.c_int]), ("hipStreamEndCapture", [C.c_void_p, C.POINTER(C.c_void_p)]),
                       ("hipGraphInstantiate", [C.POINTER(C.c_void_p), C.c_void_p, C.c_void_p, C.c_char_p, C.c_size_t]),
                       ("hipGraphLaunch", [C.c_void_p, C.c_void_p]), ("hipGraphExecDestroy", [C.c_void_p]), ("hipGraphDestroy", [C.c_void_p])):
        getattr(hip, name).argtypes = args
    entry, cap = 2 * 98, 256
    zero = (np.zeros(S * 4 * D, np.uint8), np.zeros(cap * entry, np.uint8))
    src, dst = (raw_view(lib, dev, zero, D, 1, 0, 0, cap) for _ in range(2))
    slab = dev.put(np.zeros(8 * 1024, np.uint8))
    ids = [(C.c_uint32 * 2)(*x) for x in ((6, 7), (1, 0))]
    stream, graph, gexec = dev.stream(), C.c_void_p(), C.c_void_p()
    dev.sync()
    dev._ck(hip.hipStreamBeginCapture(stream, 2), "hipStreamBeginCapture")
    rc = lib.sjk_hip_fork(C.byref(dst), C.byref(src), 1, 256, 256 + 200, stream)
    rc2 = lib.sjk_hip_copy_blocks(slab, 0, 8, slab, 0, 8, 1, 1024, ids[0], ids[1], 2, stream)
    dev._ck(hip.hipStreamEndCapture(stream, C.byref(graph)), "hipStreamEndCapture")
    sjk.check(rc, "fork")
    sjk.check(rc2, "copy_blocks")
    dev._ck(hip.hipGraphInstantiate(C.byref(gexec), graph, None, None, 0), "hipGraphInstantiate")
    try:
        slots = (np.arange(256, 456) - S) % cap
        for _ in range(4):
            sink, ring, pages = (rng.integers(0, 256, n, dtype=np.uint8) for n in (S * 4 * D, cap * entry, 8 * 1024))
            for p, x in ((src.sink, sink), (src.ring, ring), (slab.value, pages)):
                dev.upload(C.c_void_p(p), x)
            dev._ck(hip.hipGraphLaunch(gexec, stream), "hipGraphLaunch")
            dev._ck(hip.hipStreamSynchronize(stream), "hipStreamSynchronize")
            assert np.array_equal(dev.get(C.c_void_p(dst.sink), sink.nbytes, np.uint8), sink)
            got = dev.get(C.c_void_p(dst.ring), ring.nbytes, np.uint8).reshape(cap, entry)
            assert np.array_equal(got[slots], ring.reshape(cap, entry)[slots])
            pages = pages.reshape(8, 1024)
            pages[[1, 0]] = pages[[6, 7]]
            assert np.array_equal(dev.get(slab, pages.nbytes, np.uint8).reshape(8, 1024), pages)
    finally:
        hip.hipGraphExecDestroy(gexec)
        hip.hipGraphDestroy(graph)


# ---- sequences ------------------------------------------------------------------------------------------------------

def outs(lib, dev, s, rows):
    d = dev.alloc(rows.nq)
    attend(lib, s, rows, d, None, il=0)
    a = dev.alloc(rows.nq)
    attend(lib, s, rows, a, None)
    dev.sync()
    return np.concatenate([dev.get(d, rows.nq, np.uint32), dev.get(a, rows.nq, np.uint32)])


def same(lib, dev, a, b, rows):
    assert (a.n, a.pol.B, a.pol.B_prev, a.pol.draining) == (b.n, b.pol.B, b.pol.B_prev, b.pol.draining)
    assert np.array_equal(stream_bytes(lib, a), stream_bytes(lib, b))
    if a.n >= W:
        assert np.array_equal(outs(lib, dev, a, rows), outs(lib, dev, b, rows))


def fork(lib, child, parent, pos, stream=None):
    kept = C.c_uint32(77)
    sjk.check(lib.sjk_hip_seq_fork(C.byref(child), C.byref(parent), pos, C.byref(kept), stream), "seq_fork")
    assert kept.value == child.n
    return kept.value


@pytest.mark.parametrize("bk,bv,body", [(4, 4, 0), (3, 2, 1)], ids=["4/4", "3/2t"])
@pytest.mark.parametrize("parent_pool,child_pool", [(1, 1), (1, 2), (1, 0), (0, 1), (0, 0)],
                         ids=["shared", "other-pool", "pool-alone", "alone-pool", "alone"])
def test_fork_equals_a_truncated_build(lib, dev, bk, bv, body, parent_pool, child_pool):
    """a fork at every kind of position equals a sequence built alone to the parent's end and truncated there: state
    stream, policy, attention, and all of it again after both went on; the parent is what it was"""
    cfg = config(lib, bk, bv, body)
    rows, more = Rows(dev, 3000, seed=3), Rows(dev, 3000, seed=4)
    pools = {0: None, 1: new_pool(lib, cfg), 2: new_pool(lib, cfg)}
    parent, twin = new_seq(lib, cfg, pools[parent_pool]), new_seq(lib, cfg)
    grow(lib, dev, parent, rows, 1500, 5, None, True)
    grow(lib, dev, twin, rows, 1500, 5, None, True)
    n, B = parent.n, parent.pol.B
    assert B > S + 3 * G and n > B
    for pos in (n, n - 1, B + 1, B, B - 1, S + 2 * G, S + 2 * G + 5, S + 1, S, 70, 1, 0):
        child, ref = new_seq(lib, cfg, pools[child_pool]), new_seq(lib, cfg)
        grow(lib, dev, ref, rows, 1500, 5, None, True)
        r = lib.sj_kvarn_seq_truncate(C.byref(ref), pos)
        assert fork(lib, child, parent, pos) == r == ref.n
        same(lib, dev, child, ref, rows)
        for s in (child, ref):
            for k in range(3):
                step(lib, s, more, s.n, 200, None, True)
        same(lib, dev, child, ref, more)
        if pools[child_pool] is not None and child_pool == parent_pool:
            shared = [parent.blocks[g] for g in range((min(B, max(r, S)) - S) // G)] if r < B else [parent.blocks[g] for g in range((B - S) // G)]
            assert [child.blocks[g] for g in range(len(shared))] == shared
            assert all(lib.sjk_hip_pool_refs(C.byref(pools[1]), b) == 2 for b in shared)
        lib.sj_kvarn_seq_free(C.byref(child))
        lib.sj_kvarn_seq_free(C.byref(ref))
    same(lib, dev, parent, twin, rows)
    for s in (parent, twin):
        lib.sj_kvarn_seq_free(C.byref(s))
    for p in (pools[1], pools[2]):
        assert p.n_free == p.n_blocks
        lib.sj_kvarn_pool_free(C.byref(p))


def test_fork_into_a_ring_of_another_size(lib, dev):
    """n_ubatch, and with it the ring, may differ: slots are those of the child's ring; a child too small is refused"""
    cfg = config(lib)
    rows, more = Rows(dev, 3000, seed=23), Rows(dev, 3000, seed=24)
    pool = new_pool(lib, cfg)
    parent = new_seq(lib, cfg, pool)
    grow(lib, dev, parent, rows, 1500, 5, None, True)
    for n_ubatch in (1, 64, 700):
        other = sjk.Config.from_buffer_copy(bytes(cfg))
        other.n_ubatch = n_ubatch
        child, ref = new_seq(lib, other, pool), new_seq(lib, other)
        assert child.layers[0].cap != parent.layers[0].cap
        fork(lib, child, parent, parent.n - 3)
        for p0 in range(0, 1500, 256):               # the reference's ubatches, in pieces that the smaller ring takes
            sjk.check(lib.sjk_hip_seq_begin_ubatch(C.byref(ref), p0, min(256, 1500 - p0), None), "begin")
            for il in range(NL):
                sjk.check(lib.sjk_hip_seq_store(C.byref(ref), il, p0, min(256, 1500 - p0), rows.k(p0), rows.v(p0), 1, None), "store")
        for _ in range(5):
            step(lib, ref, rows, ref.n, W, None, True)
        assert lib.sj_kvarn_seq_truncate(C.byref(ref), parent.n - 3) == parent.n - 3
        same(lib, dev, child, ref, rows)
        for s in (child, ref):
            for _ in range(200):
                step(lib, s, more, s.n, W, None, True)
        same(lib, dev, child, ref, more)
        lib.sj_kvarn_seq_free(C.byref(child))
        lib.sj_kvarn_seq_free(C.byref(ref))
    lib.sj_kvarn_seq_free(C.byref(parent))
    assert pool.n_free == pool.n_blocks
    lib.sj_kvarn_pool_free(C.byref(pool))


def test_blocks_outlive_the_sequences_that_shared_them(lib, dev):
    """parent, child and grandchild: truncations, resets and frees of the others leave a sequence's records alone, a dropped
    block is cleared and freed with its last holder, and restores count only the blocks that a reset gives back"""
    cfg = config(lib)
    rows = Rows(dev, 3000, seed=9)
    pool = new_pool(lib, cfg, 30)
    a, b, c = (new_seq(lib, cfg, pool) for _ in range(3))
    ref = new_seq(lib, cfg)
    grow(lib, dev, a, rows, 1500, 3, None, True)
    grow(lib, dev, ref, rows, 1500, 3, None, True)
    n_rec = (a.pol.B - S) // G
    blocks = [a.blocks[g] for g in range(n_rec)]
    fork(lib, b, a, a.n)
    fork(lib, c, b, S + 4 * G + 17)                          # the first four groups
    refs = lambda: [lib.sjk_hip_pool_refs(C.byref(pool), x) for x in blocks]  # noqa: E731
    assert refs() == [3] * 4 + [2] * (n_rec - 4) and pool.n_free == 30 - n_rec
    want_c = stream_bytes(lib, c)
    # the parent drops all but one group: nothing is freed or cleared
    assert lib.sj_kvarn_seq_truncate(C.byref(a), S + G) == S + G
    assert refs() == [3] + [2] * 3 + [1] * (n_rec - 4) and pool.n_free == 30 - n_rec
    same(lib, dev, b, ref, rows)
    assert np.array_equal(stream_bytes(lib, c), want_c)
    # the child drops the last two groups: it held them alone
    lay = b.layers[0].lay
    assert lib.sj_kvarn_seq_truncate(C.byref(b), S + (n_rec - 2) * G) == S + (n_rec - 2) * G
    assert refs() == [3] + [2] * 3 + [1] * (n_rec - 6) + [0, 0] and pool.n_free == 30 - n_rec + 2
    for il in range(NL):
        at = b.layers[il].body + blocks[-1] * H * lay.bytes
        assert not dev.get(C.c_void_p(at), H * lay.bytes, np.uint8).any()
        at = b.layers[il].body + blocks[0] * H * lay.bytes
        assert dev.get(C.c_void_p(at), H * lay.bytes, np.uint8).any()
    # a state stream that needs more blocks than the pool and a reset of c can give: c's own four are shared and do not count
    big = stream_bytes(lib, ref)
    taken = []
    while pool.n_free > n_rec - 3:
        taken.append(lib.sj_kvarn_pool_alloc(C.byref(pool)))
    assert lib.sj_kvarn_seq_state_read(C.byref(c), big.ctypes.data, big.nbytes) == sjk.ERR_POOL_FULL
    assert np.array_equal(stream_bytes(lib, c), want_c)
    for x in taken[:3]:
        lib.sj_kvarn_pool_release(C.byref(pool), x)
    sjk.check(lib.sj_kvarn_seq_state_read(C.byref(c), big.ctypes.data, big.nbytes), "state_read")
    same(lib, dev, c, ref, rows)
    assert refs()[:4] == [2, 1, 1, 1]
    for x in taken[3:]:
        lib.sj_kvarn_pool_release(C.byref(pool), x)
    lib.sj_kvarn_seq_reset(C.byref(a))
    assert refs()[0] == 1
    for s in (a, b, c, ref):
        lib.sj_kvarn_seq_free(C.byref(s))
    assert pool.n_free == 30 and sorted(pool.free_ids[i] for i in range(30)) == list(range(30))
    lib.sj_kvarn_pool_free(C.byref(pool))


def test_fork_refuses(lib, dev):
    cfg = config(lib)
    rows = Rows(dev, 2000, seed=11)
    pool, small = new_pool(lib, cfg), new_pool(lib, cfg, 2)
    a = new_seq(lib, cfg, pool)
    grow(lib, dev, a, rows, 1200, 1, None, True)
    want, free = stream_bytes(lib, a), pool.n_free

    def refused(child, code, pos=None):
        kept = C.c_uint32(5)
        before = bytes(child.pol), child.n
        assert lib.sjk_hip_seq_fork(C.byref(child), C.byref(a), a.n if pos is None else pos, C.byref(kept), None) == code
        assert kept.value == 5 and (bytes(child.pol), child.n) == before and pool.n_free == free

    used = new_seq(lib, cfg, pool)
    step(lib, used, rows, 0, 1, None, True)
    refused(used, -100)
    refused(a, -100)
    fresh = new_seq(lib, cfg, pool)
    refused(fresh, -100, a.n + 1)
    a.pol.B_pending = a.pol.B + G
    refused(fresh, -108)
    a.pol.B_pending = a.pol.B
    others = []
    for field, value, code in (("n_head_kv", 4, -121), ("sink", 192, -123), ("bits_v", 2, -124), ("iters", 8, -126), ("staging", 1, -127),
                               ("tail", 384, -128), ("n_ctx", 1000, -109)):
        c2 = sjk.Config.from_buffer_copy(bytes(cfg))
        setattr(c2, field, value)
        others.append(new_seq(lib, c2))
        refused(others[-1], code)
    poor = new_seq(lib, cfg, small)
    refused(poor, -110)
    assert small.n_free == 2
    buf = np.zeros(lib.sj_kvarn_seq_state_size(C.byref(a)), np.uint8)
    sjk.check(lib.sjk_hip_seq_state_read_begin(C.byref(fresh), want.ctypes.data, want.nbytes), "read_begin")
    refused(fresh, -108)                                     # a restore of the child in flight
    sjk.check(lib.sjk_hip_seq_state_finish(C.byref(fresh), None), "finish")
    free = pool.n_free
    sjk.check(lib.sjk_hip_seq_state_write_begin(C.byref(a), buf.ctypes.data, buf.nbytes), "write_begin")
    again = new_seq(lib, cfg, pool)
    fork(lib, again, a, a.n)                                 # a save of the parent in flight is no obstacle
    sjk.check(lib.sjk_hip_seq_state_finish(C.byref(a), None), "finish")
    assert np.array_equal(buf, want) and np.array_equal(stream_bytes(lib, again), want)
    for s in [a, used, fresh, poor, again] + others:
        lib.sj_kvarn_seq_free(C.byref(s))
    assert pool.n_free == pool.n_blocks
    lib.sj_kvarn_pool_free(C.byref(pool))
    lib.sj_kvarn_pool_free(C.byref(small))


def compact(lib, pool, seqs):
    moved = C.c_uint32(NO)
    arr = (C.POINTER(sjk.Seq) * max(1, len(seqs)))(*[C.pointer(s) for s in seqs])
    rc = lib.sjk_hip_pool_compact(C.byref(pool), arr, len(seqs), C.byref(moved), None)
    return rc, moved.value


def test_compaction(lib, dev):
    """sequences with shared blocks before and after a compaction: the same streams and attention, live blocks at the lowest
    ids, free ids behind them handed out lowest first; refused, changing nothing, where a holder is missing or given twice"""
    cfg = config(lib)
    rows = Rows(dev, 3000, seed=13)
    pool = new_pool(lib, cfg, 60)
    seqs = [new_seq(lib, cfg, pool) for _ in range(5)]
    for k, s in enumerate(seqs[:4]):                         # interleaved growth
        grow(lib, dev, s, rows, 900 + 150 * k, 2, None, True)
    fork(lib, seqs[4], seqs[2], S + 3 * G)
    for k in (0, 1):
        lib.sj_kvarn_seq_free(C.byref(seqs[k]))
    live = seqs[2:]
    n_live = pool.n_blocks - pool.n_free
    tables = lambda: [[s.blocks[g] for g in range(s.layers[0].n_groups)] for s in live]  # noqa: E731
    before, want, t0 = [stream_bytes(lib, s) for s in live], [outs(lib, dev, s, rows) for s in live], tables()
    assert max(b for t in t0 for b in t if b != NO) >= n_live
    for given in (live[:2], [live[0], live[2]], live + [live[0]], []):
        assert compact(lib, pool, given) == (-100, NO)
    stray = lib.sj_kvarn_pool_alloc(C.byref(pool))
    assert compact(lib, pool, live) == (-100, NO)            # a live block that no sequence holds
    lib.sj_kvarn_pool_release(C.byref(pool), stray)
    assert tables() == t0
    rc, moved = compact(lib, pool, live)
    assert rc == 0 and moved == len({b for t in t0 for b in t if b != NO and b >= n_live}) > 0
    ids = {b for t in tables() for b in t if b != NO}
    assert ids == set(range(n_live))
    assert [pool.free_ids[pool.n_free - 1 - i] for i in range(pool.n_free)] == list(range(n_live, 60))
    for t, u in zip(t0, tables()):                           # blocks that lay low stay
        assert all(v == w for v, w in zip(t, u) if v == NO or v < n_live)
    for s, x, o in zip(live, before, want):
        assert np.array_equal(stream_bytes(lib, s), x) and np.array_equal(outs(lib, dev, s, rows), o)
    assert [lib.sjk_hip_pool_refs(C.byref(pool), live[2].blocks[g]) for g in range(3)] == [2, 2, 2]
    assert compact(lib, pool, live) == (0, 0)
    ref = new_seq(lib, cfg)
    grow(lib, dev, ref, rows, 1200, 2, None, True)
    for s in (live[0], ref):
        for k in range(4):
            step(lib, s, rows, s.n, 200, None, True)
    same(lib, dev, live[0], ref, rows)
    for s in live + [ref]:
        lib.sj_kvarn_seq_free(C.byref(s))
    assert pool.n_free == 60
    assert compact(lib, pool, []) == (0, 0)
    lib.sj_kvarn_pool_free(C.byref(pool))


def test_from_projections_to_forked_sequences(lib, dev):
    """the whole path as an engine runs it, on a stream of its own: a prompt appended from projection rows (norms, turn, rotation,
    staging), committed, forked into three samples that decode different tokens in one batch, the parent freed, the pool
    compacted on the way; every step's attention and the final streams equal those of sequences run alone, step by step with
    sjk_hip_head_rows and sjk_hip_seq_store_batch"""
    cfg = config(lib)
    rng = np.random.default_rng(17)
    pool = new_pool(lib, cfg, 60)
    st = dev.stream()
    scale = 1.0 / np.sqrt(D)
    prompt = [Proj(dev, rng, 256, N_HEAD, H, D, sjk.BF16, True, D, 0, pad=8) for _ in range(5)]      # the same rows in every layer
    steps = [[Proj(dev, rng, W, N_HEAD, H, D, sjk.BF16, True, D, 0) for _ in range(3)] for _ in range(40)]
    for p in prompt[1:] + [x for r in steps for x in r]:
        p.m.d_q_norm, p.m.d_k_norm = prompt[0].m.d_q_norm, prompt[0].m.d_k_norm
    m, ms = prompt[0].m, steps[0][0].m
    noise = new_seq(lib, cfg, pool)
    rows = Rows(dev, 1200, seed=2)
    grow(lib, dev, noise, rows, 1000, 0, st, True)                                                   # blocks in front of the prompt's

    def job(s, p, n):
        q, k, v = p.ptrs()
        return sjk.SeqQkvJob(C.pointer(s), s.n if n is None else n, None, q, k, v, p.q.value)

    parent = new_seq(lib, cfg, pool)
    for i, p in enumerate(prompt):
        sjk.check(lib.sjk_hip_seq_begin_ubatch(C.byref(parent), 256 * i, 256, st), "begin")
        for il in range(NL):
            j = job(parent, p, 256 * i)
            sjk.check(lib.sjk_hip_seq_store_qkv_batch(C.byref(j), 1, il, 256, C.byref(m), st), "store")
    kids = [new_seq(lib, cfg, pool) for _ in range(3)]
    cuts = (1280, 1280, 1111)
    for s, cut in zip(kids, cuts):
        fork(lib, s, parent, cut, st)
    lib.sj_kvarn_seq_free(C.byref(parent))
    lib.sj_kvarn_seq_free(C.byref(noise))
    got = []
    for r, ps in enumerate(steps):
        if r in (0, 20):                                     # before the children take the freed blocks, and on the way
            arr = (C.POINTER(sjk.Seq) * 3)(*[C.pointer(s) for s in kids])
            moved = C.c_uint32(0)
            sjk.check(lib.sjk_hip_pool_compact(C.byref(pool), arr, 3, C.byref(moved), st), "compact")
            assert moved.value > 0 or r
        starts = [s.n for s in kids]
        for s, n in zip(kids, starts):
            sjk.check(lib.sjk_hip_seq_begin_ubatch(C.byref(s), n, W, st), "begin")
        for il in range(NL):
            jobs = (sjk.SeqQkvJob * 3)(*[job(s, p, n) for s, p, n in zip(kids, ps, starts)])
            sjk.check(lib.sjk_hip_seq_store_qkv_batch(jobs, 3, il, W, C.byref(ms), st), "store")
            aj = (sjk.SeqJob * 3)()
            for k, (s, p) in enumerate(zip(kids, ps)):
                aj[k].seq, aj[k].pos0, aj[k].d_q = C.pointer(s), starts[k], p.q.value
                aj[k].d_out = dev.alloc(W * N_HEAD * D * 4).value
                got.append(aj[k].d_out)
            sjk.check(lib.sjk_hip_seq_attend_batch(aj, 3, il, W, N_HEAD, scale, st), "attend")
    dev.sync()
    got = [dev.get(C.c_void_p(d), W * N_HEAD * D * 4, np.uint32) for d in got]

    # alone
    q, k, v, o = (dev.alloc(256 * N_HEAD * D * 4) for _ in range(4))

    def feed(s, p, n, attend_at=None):
        res = []
        jobs = (sjk.HeadJob * 3)(*[sjk.HeadJob(a, d.value, p.x.pos, D, h * D, D, sjk.BF16, sjk.F32, h, t, ro, 1e-5, w, 0) for a, d, h, t, ro, w in
                                   zip(p.ptrs(), (q, k, v), (N_HEAD, H, H), (1, 1, 0), (1, 0, 0), (p.m.d_q_norm, p.m.d_k_norm, None))])
        sjk.check(lib.sjk_hip_head_rows(jobs, 3, n, D, C.byref(p.m.rope), s.n, None, None), "head_rows")
        p0 = s.n
        sjk.check(lib.sjk_hip_seq_begin_ubatch(C.byref(s), p0, n, None), "begin")
        for il in range(NL):
            sjk.check(lib.sjk_hip_seq_store(C.byref(s), il, p0, n, k, v, 1, None), "store")
            if attend_at:
                sjk.check(lib.sjk_hip_seq_attend(C.byref(s), il, p0, n, N_HEAD, q, scale, o, None), "attend")
                dev.sync()
                res.append(dev.get(o, n * N_HEAD * D * 4, np.uint32))
        return res

    for c, (s, cut) in enumerate(zip(kids, cuts)):
        ref = new_seq(lib, cfg)
        for p in prompt:
            feed(ref, p, 256)
        assert lib.sj_kvarn_seq_truncate(C.byref(ref), cut) <= cut
        for r, ps in enumerate(steps):
            for il, want in enumerate(feed(ref, ps[c], W, True)):
                assert np.array_equal(got[(r * NL + il) * 3 + c], want), (c, r, il)
        same(lib, dev, s, ref, rows)
        lib.sj_kvarn_seq_free(C.byref(ref))
    for s in kids:
        lib.sj_kvarn_seq_free(C.byref(s))
    assert pool.n_free == 60
    lib.sj_kvarn_pool_free(C.byref(pool))
