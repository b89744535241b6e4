"""Calls between projections and cache, and those that move pages, that are refused before anything is launched (no GPU; every
device pointer is fake): positions past 32 bits, buffers that overlap, sealed positions; and pools that their caller put together."""
import ctypes as C
import sys

import cabi

sys.path.insert(0, cabi.PKG)
from test_heads_refusals import ARG, CAPACITY, FAKE, job, lib, qkv, rope, sjk, view  # noqa: E402, F401


def test_head_rows_positions_past_32_bits(lib):  # noqa: F811
    """pos0 + i ends below 2^32 - 1 (no position), as in sjk_hip_store_qkv"""
    def call(n, pos0):
        return lib.sjk_hip_head_rows(C.byref(job(rope=1)), 1, n, 128, C.byref(rope()), pos0, None, None)

    for n, pos0 in ((200, 0xFFFFFF80), (1, 0xFFFFFFFF), (2, 0xFFFFFFFE)):
        assert call(n, pos0) == ARG, (n, pos0)
    assert b"2^32" in lib.sjk_last_error() and call(0, 0xFFFFFFFF) == 0


def test_fork_refuses_buffers_that_overlap(lib):  # noqa: F811
    """a buffer of dst that is, or reaches into, another buffer of dst or one of src, of either kind, in any layer"""
    MB = 1 << 20
    sink, ring = 128 * 2 * 4 * 128, 256 * 2 * 2 * 98                    # bytes: 128 KiB, 98 KiB
    src = [view(lib, sink=i * MB, ring=i * MB + MB // 2) for i in (1, 2)]
    dst = [view(lib, sink=i * MB, ring=i * MB + MB // 2) for i in (11, 12)]

    def call(d, s, n=200):
        return lib.sjk_hip_fork((sjk.View * 2)(*d), (sjk.View * 2)(*s), 2, 128, n, None)

    assert call(dst, src, 0) == 0
    for il in (0, 1):
        for name, size, starts in (("sink", sink, [v.sink for v in src] + [v.ring for v in src] + [dst[1 - il].sink, dst[1 - il].ring, dst[il].ring]),
                                   ("ring", ring, [v.sink for v in src] + [v.ring for v in src] + [dst[1 - il].sink, dst[1 - il].ring, dst[il].sink])):
            for k, at in enumerate(starts):
                other = sink if at % MB == 0 else ring
                for p, code in ((at, ARG), (at + other - 4, ARG), (at - size + 4, ARG), (at + other, 0), (at - size, 0)):
                    d = [sjk.View.from_buffer_copy(v) for v in dst]
                    setattr(d[il], name, p)
                    assert call(d, src, 0) == code, (il, name, k, p - at)
                    assert code == 0 or call(d, src) == code
    other = [sjk.View.from_buffer_copy(v) for v in src]
    other[1].sink, other[1].ring = src[0].sink, src[0].ring              # (src's own buffers are only read)
    assert call(dst, other, 0) == 0


def test_pool_put_together_by_its_caller(lib):  # noqa: F811
    """a pool with a free list of the caller's own, n_blocks words: nothing behind the list is read or written, and every block
    has one holder"""
    for guard in (0, 1, 7, 0xFFFFFFFF):
        ids = (C.c_uint32 * 12)(*([3, 2] + [guard] * 10))
        pool = sjk.Pool()
        pool.n_layers, pool.n_blocks, pool.n_free = 1, 4, 2
        pool.free_ids = C.cast(ids, C.POINTER(C.c_uint32))
        assert [lib.sjk_hip_pool_refs(C.byref(pool), i) for i in range(5)] == [1, 1, 0, 0, 0]
        lib.sj_kvarn_pool_release(C.byref(pool), 1)
        lib.sj_kvarn_pool_release(C.byref(pool), 0)
        assert pool.n_free == 4 and list(ids) == [3, 2, 1, 0] + [guard] * 8
        lib.sj_kvarn_pool_release(C.byref(pool), 0)              # full: nothing more
        assert pool.n_free == 4 and list(ids) == [3, 2, 1, 0] + [guard] * 8
        assert [lib.sj_kvarn_pool_alloc(C.byref(pool)) for _ in range(5)] == [0, 1, 2, 3, 0xFFFFFFFF]


def test_sequence_append_below_the_sealed_end(lib):  # noqa: F811
    """positions of the sealed part whose ring slots hold staged positions are refused: storing them would write over those"""
    L = sjk.Layer()
    v = view(lib, cap=896)
    L.lay, L.cap, L.stage_bytes, L.n_groups, L.ring, L.sink, L.body = v.lay, 896, v.stage_bytes, 64, v.ring, v.sink, v.body
    L.cfg.staging, L.cfg.sink_type = v.staging, v.sink_type
    L.cfg.head_dim, L.cfg.n_head_kv, L.cfg.group, L.cfg.sink, L.cfg.n_ctx = 128, 2, 128, 128, 8192
    s = sjk.Seq()
    s.n_layers, s.layers, s.cfg = 1, C.pointer(L), L.cfg
    s.pol.sink, s.pol.group, s.pol.B, s.pol.B_pending, s.n = 128, 128, 128 + 1280, 128 + 1280, 128 + 1280 + 500
    m = qkv()

    def call(pos0, n):
        j = sjk.SeqQkvJob(C.pointer(s), pos0, None, FAKE, FAKE, FAKE, FAKE)
        return lib.sjk_hip_seq_store_qkv_batch(C.byref(j), 1, 0, n, C.byref(m), None)

    # staged slots: positions 128 + [1280, 1780) at [384, 884); the sealed positions at them are 128 + [384, 884)
    for pos0, n in ((128 + 384, 1), (128 + 883, 1), (128 + 380, 5), (128 + 883, 200), (128 + 300, 800), (0, 128 + 385)):
        assert call(pos0, n) == CAPACITY, (pos0, n)
    assert call(128 + 1280, 897) == CAPACITY and call(s.n + 1, 1) == ARG
    assert call(128 + 384, 0) == 0 and s.n == 128 + 1780
