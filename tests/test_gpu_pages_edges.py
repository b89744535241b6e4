"""Forks and compaction on a pool that its caller put together over a slab of its own (no counts of holders): records are copied,
every block has one holder, nothing behind the caller's free list is touched. Appends to a sequence's sealed positions."""
import ctypes as C

import numpy as np
import pytest

import cabi  # noqa: F401
from test_gpu_async import H, N_HEAD, NL, Rows, config, grow, new_pool, new_seq, step, stream_bytes
from test_gpu_heads import Proj
from test_gpu_pages import D, G, S, compact, dev, fork, lib, same, sjk  # noqa: F401

pytestmark = pytest.mark.gpu


def test_fork_on_a_pool_without_counts(lib, dev):  # noqa: F811
    cfg = config(lib)
    rows, more = Rows(dev, 3000, seed=31), Rows(dev, 3000, seed=32)
    slab = new_pool(lib, cfg, 30)
    pool = sjk.Pool.from_buffer_copy(bytes(slab))
    ids = (C.c_uint32 * 60)(*(list(range(29, -1, -1)) + [5] * 30))
    pool.free_ids = C.cast(ids, C.POINTER(C.c_uint32))
    parent, child, ref = new_seq(lib, cfg, pool), new_seq(lib, cfg, pool), new_seq(lib, cfg)
    for s in (parent, ref):
        grow(lib, dev, s, rows, 1500, 3, None, True)
    n_rec = (parent.pol.B - S) // G
    fork(lib, child, parent, parent.n)
    same(lib, dev, child, ref, rows)
    mine, its = ([s.blocks[g] for g in range(n_rec)] for s in (child, parent))
    assert not set(mine) & set(its) and pool.n_free == 30 - 2 * n_rec
    assert all(lib.sjk_hip_pool_refs(C.byref(pool), b) == 1 for b in mine + its)
    assert lib.sj_kvarn_seq_truncate(C.byref(parent), S + G) == S + G          # clears and frees the parent's own
    assert pool.n_free == 30 - n_rec - 1
    same(lib, dev, child, ref, rows)
    rc, moved = compact(lib, pool, [parent, child])
    assert rc == 0 and moved > 0 and {child.blocks[g] for g in range(n_rec)} | {parent.blocks[0]} == set(range(n_rec + 1))
    same(lib, dev, child, ref, rows)
    for s in (child, ref):
        step(lib, s, more, s.n, 200, None, True)
    same(lib, dev, child, ref, more)
    again = new_seq(lib, cfg, pool)
    while pool.n_free >= n_rec:
        lib.sj_kvarn_pool_alloc(C.byref(pool))
    free = pool.n_free
    assert lib.sjk_hip_seq_fork(C.byref(again), C.byref(child), child.n, None, None) == sjk.ERR_POOL_FULL and pool.n_free == free
    for s in (parent, child, again, ref):
        lib.sj_kvarn_seq_free(C.byref(s))
    assert list(ids)[30:] == [5] * 30
    lib.sj_kvarn_pool_free(C.byref(slab))


def test_append_to_sealed_positions(lib, dev):  # noqa: F811
    """a sealed position whose ring slot no staged one holds may be stored again, which changes nothing that is read; any other
    is refused and changes nothing"""
    cfg = config(lib)
    rows = Rows(dev, 4000, seed=41)
    s, ref = new_seq(lib, cfg), new_seq(lib, cfg)
    for x in (s, ref):
        grow(lib, dev, x, rows, 2500, 3, None, True)
    cap, B, n = s.layers[0].cap, s.pol.B, s.n
    assert B - S > cap and n > B
    p = Proj(dev, np.random.default_rng(41), 1, N_HEAD, H, D, sjk.BF16, True, D, 0)
    q, k, v = p.ptrs()
    held = {(x - S) % cap for x in range(B, n)}
    codes = set()
    for pos in (S, B - 1, B - G, B - cap - 1, B - cap, n - cap - 1, n - cap, n - 2 * cap, S + 1):
        if not S <= pos < B:
            continue
        j = sjk.SeqQkvJob(C.pointer(s), pos, None, q, k, v, p.q.value)
        codes.add(rc := lib.sjk_hip_seq_store_qkv_batch(C.byref(j), 1, 0, 1, C.byref(p.m), None))
        assert rc == (-109 if (pos - S) % cap in held else 0), pos
        same(lib, dev, s, ref, rows)
    assert codes == {0, -109}
    for x in (s, ref):
        lib.sj_kvarn_seq_free(C.byref(x))
