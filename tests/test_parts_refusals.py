"""What the calls on listed groups and drafted nodes refuse, before anything is launched (no GPU: every pointer is fake), and the
calls that have nothing to do."""
import ctypes as C
import sys

import pytest

import cabi

sys.path.insert(0, cabi.PKG)
import sjk  # noqa: E402

ARG, CAPACITY, UNSUPPORTED = -100, -109, -141
FAKE = 0x100000
S, G = 128, 128


@pytest.fixture(scope="module")
def lib():
    return sjk.load()


def view(lib, D=128, H=2, bits=(4, 4, 0), **kw):
    v = sjk.View()
    v.lay = sjk.layout(D, G, *bits)
    v.n_head_kv, v.staging, v.sink_type, v.S, v.cap = H, 0, 0, S, 512
    v.stage_bytes = D // 128 * 98
    v.sink = v.ring = v.body = v.work = FAKE
    v.work_bytes = 1 << 30
    for k, x in kw.items():
        setattr(v, k, x)
    return v


B, N, QPOS = S + 4 * G, S + 4 * G + 50, S + 4 * G + 49


def test_select_refusals(lib):
    def call(v=None, B=B, N=N, qpos0=QPOS, n_q=1, n_head=8, q=FAKE, top=2, sel=FAKE, stream=None):
        v = v if v is not None else view(lib)
        return lib.sjk_hip_select_groups(C.byref(v), B, N, qpos0, n_q, n_head, q, top, sel, stream)

    assert lib.sjk_hip_select_groups(None, B, N, QPOS, 1, 8, FAKE, 2, FAKE, None) == ARG
    for bad in (dict(n_q=0), dict(n_head=0), dict(n_head=7), dict(top=0), dict(top=-1), dict(q=None), dict(q=FAKE + 4), dict(sel=None),
                dict(sel=FAKE + 2), dict(B=B + 1), dict(N=B - 1), dict(qpos0=B - 2), dict(qpos0=2 ** 32 - 1), dict(qpos0=2 ** 32 - 4, n_q=5)):
        assert call(**bad) == ARG, bad
    assert call(view(lib, n_head_kv=0)) == ARG and call(view(lib, work=None)) == ARG and call(view(lib, body=None)) == ARG
    lay = view(lib)
    lay.lay.k_scale += 2
    assert call(lay) == UNSUPPORTED
    assert call(view(lib, bits=(4, 4, 0), work_bytes=4096 + 2048), top=1) == CAPACITY
    jobs = (sjk.GroupsJob * 2)(*[sjk.GroupsJob(view(lib, D=d), B, N, QPOS, FAKE, FAKE, None) for d in (128, 256)])
    assert lib.sjk_hip_select_groups_batch(jobs, 2, 1, 8, 2, None) == ARG
    assert lib.sjk_hip_select_groups_batch(None, 1, 1, 8, 2, None) == ARG and lib.sjk_hip_select_groups_batch(jobs, -1, 1, 8, 2, None) == ARG
    assert lib.sjk_hip_select_groups_batch(None, 0, 1, 8, 2, None) == 0
    v = view(lib)
    for args in ((None, N, 1, 8, FAKE, 2, FAKE), (FAKE + 2, N, 1, 8, FAKE, 2, FAKE), (FAKE, N, 1, 8, None, 2, FAKE), (FAKE, N, 1, 8, FAKE, 0, FAKE)):
        assert lib.sjk_hip_select_groups_dyn(C.byref(v), *args, None) == ARG
    assert lib.sjk_hip_select_groups_dyn(C.byref(view(lib, work=None)), FAKE, N, 1, 8, FAKE, 2, FAKE, None) == ARG


def test_attend_groups_refusals(lib):
    def call(v=None, B=B, N=N, qpos0=QPOS, n_q=1, n_head=8, q=FAKE, sel=FAKE, top=2, t=sjk.F32, out=FAKE << 4):
        v = v if v is not None else view(lib)
        return lib.sjk_hip_attend_groups(C.byref(v), B, N, qpos0, n_q, n_head, q, 0.1, sel, top, t, out, None)

    for bad in (dict(n_q=0), dict(n_head=0), dict(n_head=9), dict(top=0), dict(q=None), dict(q=FAKE + 8), dict(sel=None), dict(sel=FAKE + 1), dict(t=3),
                dict(t=-1), dict(out=None), dict(out=(FAKE << 4) + 2), dict(t=sjk.BF16, out=(FAKE << 4) + 1), dict(out=FAKE), dict(out=FAKE + 4092),
                dict(t=sjk.F16, out=FAKE - 2046), dict(B=B + 3), dict(N=B - 1), dict(qpos0=B - 2)):
        assert call(**bad) == ARG, bad
    for bad in (dict(work=None), dict(body=None), dict(ring=None), dict(sink=None), dict(cap=8), dict(work_bytes=1 << 16)):
        assert call(view(lib, **bad)) == ARG, bad
    assert call(N=B + 600, qpos0=B + 599) == CAPACITY
    assert call(view(lib, stage_bytes=99)) == UNSUPPORTED
    assert lib.sjk_hip_attend_groups_batch(None, 0, 1, 8, 0.1, 2, 0, None) == 0
    assert lib.sjk_hip_attend_groups_batch(None, 1, 1, 8, 0.1, 2, 0, None) == ARG
    v = view(lib)
    for d_desc, sel, top in ((None, FAKE, 2), (FAKE, None, 2), (FAKE, FAKE, 0)):
        assert lib.sjk_hip_attend_groups_dyn(C.byref(v), d_desc, N, 1, 8, FAKE, 0.1, sel, top, 0, FAKE << 4, None) == ARG


def test_attend_tree_refusals(lib):
    def call(v=None, B=B, base=N, n_nodes=20, n_q=20, n_head=8, q=FAKE, seen=FAKE, t=sjk.F32, out=FAKE << 4):
        v = v if v is not None else view(lib)
        return lib.sjk_hip_attend_tree(C.byref(v), B, base, n_nodes, n_q, n_head, q, 0.1, seen, t, out, None)

    for bad in (dict(n_nodes=0), dict(n_nodes=-1), dict(n_q=0), dict(n_head=3), dict(q=None), dict(seen=None), dict(seen=FAKE + 4), dict(t=7),
                dict(out=None), dict(out=FAKE), dict(base=B - 1), dict(B=B + 5), dict(base=2 ** 32 - 30), dict(base=2 ** 32 - 1)):
        assert call(**bad) == ARG, bad
    assert call(n_nodes=500) == CAPACITY
    assert call(view(lib, body=None)) == ARG
    assert lib.sjk_hip_attend_tree_batch(None, 0, 4, 4, 8, 0.1, 0, None) == 0
    assert lib.sjk_hip_attend_tree_batch(None, 2, 4, 4, 8, 0.1, 0, None) == ARG
    v = view(lib)
    for args in ((None, N, 4, 4), (FAKE, N, 0, 4), (FAKE, N, 4, 0), (FAKE, 2 ** 32 - 2, 4, 4)):
        assert lib.sjk_hip_attend_tree_dyn(C.byref(v), *args, 8, FAKE, 0.1, FAKE, 0, FAKE << 4, None) == ARG, args


def test_accept_refusals(lib):
    def call(vs, n_layers=None, base=1000, n_nodes=20, path=FAKE, n_path=4):
        a = (sjk.View * len(vs))(*vs)
        return lib.sjk_hip_accept(a, len(vs) if n_layers is None else n_layers, base, n_nodes, path, n_path, None)

    ok = view(lib)
    for bad in (dict(n_layers=-1), dict(n_nodes=-1), dict(n_path=-1), dict(path=None), dict(path=FAKE + 2), dict(base=2 ** 32 - 5)):
        assert call([ok], **bad) == ARG, bad
    for bad in (dict(ring=None), dict(sink=None), dict(ring=FAKE + 2), dict(stage_bytes=97), dict(n_head_kv=0), dict(staging=4), dict(sink_type=9)):
        assert call([view(lib, **bad)]) == ARG, bad
    for other in (view(lib, cap=256), view(lib, n_head_kv=4), view(lib, D=256), view(lib, sink_type=1)):
        assert call([ok, other]) == ARG
    assert call([ok], n_nodes=513) == CAPACITY
    assert call([ok], n_layers=0) == 0 and call([ok], n_path=0) == 0 and call([ok], n_nodes=0) == 0
    assert lib.sjk_hip_accept(None, 1, 0, 4, FAKE, 1, None) == ARG
    v = (sjk.View * 1)(ok)
    assert lib.sjk_hip_accept_dyn(v, 1, None, 4, FAKE, 1, None) == ARG and lib.sjk_hip_accept_dyn(v, 1, FAKE, 4, None, 1, None) == ARG
    assert lib.sjk_hip_accept_dyn(v, 1, FAKE, 600, FAKE, 1, None) == CAPACITY


def test_sequence_refusals(lib):
    s = sjk.Seq()
    s.n_layers, s.n = 2, 50
    j = (sjk.SeqGroupsJob * 1)(sjk.SeqGroupsJob(C.pointer(s), 49, FAKE, FAKE, FAKE))
    t = (sjk.SeqTreeJob * 1)(sjk.SeqTreeJob(C.pointer(s), 45, FAKE, FAKE, FAKE))
    for il in (-1, 2):
        assert lib.sjk_hip_seq_select_groups_batch(j, 1, il, 1, 8, 2, None) == ARG
        assert lib.sjk_hip_seq_attend_groups_batch(j, 1, il, 1, 8, 0.1, 2, 0, None) == ARG
        assert lib.sjk_hip_seq_attend_tree_batch(t, 1, il, 4, 4, 8, 0.1, 0, None) == ARG
    assert lib.sjk_hip_seq_select_groups_batch(j, 1, 0, 2, 8, 2, None) == ARG                  # past the position count
    assert lib.sjk_hip_seq_attend_tree_batch(t, 1, 0, 6, 4, 8, 0.1, 0, None) == ARG
    assert lib.sjk_hip_seq_attend_tree_batch(t, -1, 0, 4, 4, 8, 0.1, 0, None) == ARG
    assert lib.sjk_hip_seq_select_groups_batch(None, 1, 0, 1, 8, 2, None) == ARG
    assert lib.sjk_hip_seq_attend_tree_batch(None, 0, 0, 4, 4, 8, 0.1, 0, None) == 0
    assert lib.sjk_hip_seq_accept(None, 0, None, 0, None) == ARG and lib.sjk_hip_seq_accept(C.byref(s), 0, None, 0, None) == ARG
