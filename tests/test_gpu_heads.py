"""Head norms, rotary positions and the append from a projection's rows (sjk_hip_head_rows, sjk_hip_store_qkv and its dyn,
batch and sequence forms) on the GPU.

Rows against the same formulas in 64 bits (80 where the host has them), with an error bound made from the roundings the
kernel may make (below); the append bit for bit against sjk_hip_head_rows to fp32 followed by sjk_hip_layer_store, whose
bytes the oracle pins. Rows, channels and buffers that a call does not name keep what was in them."""
import ctypes as C
import sys

import numpy as np
import pytest

import cabi

sys.path.insert(0, cabi.PKG)
import sjk  # noqa: E402

pytestmark = pytest.mark.gpu
L = np.longdouble
TWO_PI = L("6.28318530717958647692528676655900577")
U = 2.0 ** -24                                   # half a step of fp32, relative
HALF = {sjk.F32: U, sjk.F16: 2.0 ** -11, sjk.BF16: 2.0 ** -8}
TINY = {sjk.F32: 2.0 ** -149, sjk.F16: 2.0 ** -24, sjk.BF16: 2.0 ** -133}
EPS = 1e-5


@pytest.fixture(scope="module")
def lib():
    return sjk.load()


@pytest.fixture
def dev():
    d = sjk.Device()
    yield d
    d.sync()
    d.free_all()


def to_bits(x, t):
    """float32 array as the element type's bits, rounded to nearest even"""
    x = np.ascontiguousarray(x, np.float32)
    if t == sjk.F32:
        return x.view(np.uint32).copy()
    if t == sjk.F16:
        with np.errstate(over="ignore"):
            return x.astype(np.float16).view(np.uint16)
    u = x.view(np.uint32).astype(np.uint64)
    r = ((u + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint16)
    return np.where(np.isnan(x), np.uint16(0x7FC0), r)


def from_bits(b, t):
    if t == sjk.F32:
        return b.view(np.float32)
    if t == sjk.F16:
        return b.view(np.float16).astype(np.float32)
    return (b.astype(np.uint32) << 16).view(np.float32)


def hadamard(D):
    i = np.arange(D)
    b = i[:, None] & i[None, :]
    return np.where(np.array([bin(x).count("1") & 1 for x in b.ravel()]).reshape(D, D), -1.0, 1.0)


def turn_table(n_rot, base=1e4):
    return base ** (-2.0 * np.arange(n_rot // 2) / max(n_rot, 1)) / (2 * np.pi)


def reference(x, pos, w=None, rope=None, rotate=False):
    """rows x [n][h][D] (exact values) -> (value, bound on the kernel's fp32 error before its last rounding).

    Counted in units of U of the magnitudes that enter: norm 12 (a tree of up to 9 sums on 1 product, the mean's product and
    sum, square root and reciprocal, halved or whole: under 10; two products); sine and cosine 6 (the reduced angle's rounding,
    the series' coefficients and steps, mscale), their two products with the pair 2; the Hadamard's log2 D sums and scale (itself
    rounded) log2 D + 2 on the sum of the magnitudes; the position's product with the table, in 64 bits, 2 pi u 2^-53."""
    x = x.astype(L)
    D = x.shape[-1]
    err = np.zeros_like(x)
    if w is not None:
        x = x / np.sqrt((x * x).sum(-1, keepdims=True) / D + L(np.float32(EPS))) * w.astype(L)
        err = 12 * U * np.abs(x)
    if rope is not None and rope["n_rot"]:
        n, half = rope["n_rot"], rope["n_rot"] // 2
        u = pos.astype(L)[:, None] * rope["turns"].astype(L)[None, :]
        ang = (u - np.rint(u)) * TWO_PI
        m = L(np.float32(rope.get("mscale", 1.0)))
        c, s = (np.cos(ang) * m)[:, None, :], (np.sin(ang) * m)[:, None, :]
        if rope.get("inverse"):
            s = -s
        i = np.arange(half)
        a, b = (2 * i, 2 * i + 1) if rope["layout"] == sjk.ROPE_PAIRS else (i, i + half)
        xa, xb = x[..., a].copy(), x[..., b].copy()
        ea, eb = err[..., a].copy(), err[..., b].copy()
        far = (np.abs(u) * TWO_PI * L(2.0 ** -53))[:, None, :]
        x[..., a], x[..., b] = xa * c - xb * s, xa * s + xb * c
        e = (8 * U + far) * np.abs(m) * (np.abs(xa) + np.abs(xb)) + np.abs(m) * (ea + eb)
        err[..., a], err[..., b] = e, e
    if rotate:
        R = hadamard(D).astype(np.float64)
        mag = np.abs(x).sum(-1, keepdims=True)
        err = err.sum(-1, keepdims=True) / np.sqrt(L(D)) + (np.log2(D) + 2) * U * mag / np.sqrt(L(D)) + np.zeros_like(x)
        lead = x.shape[:-1]
        hi = x.astype(np.float64)
        lo = (x - hi).astype(np.float64)
        x = ((hi.reshape(-1, D) @ R).astype(L) + (lo.reshape(-1, D) @ R).astype(L)).reshape(lead + (D,)) / np.sqrt(L(D))
    return x, err


def check_rows(got_bits, t, ref, err, what):
    got = from_bits(got_bits, t).astype(L)
    bound = (err + HALF[t] * (np.abs(ref) + err) + TINY[t] / 2 + 2.0 ** -126).astype(L)
    bad = ~(np.abs(got - ref) <= bound)
    assert not bad.any(), (what, int(bad.sum()), np.abs(got - ref)[bad][:4], bound[bad][:4])


class Set:
    """heads of one job: the device buffer they lie in (with guard words), their strides and values"""

    def __init__(self, dev, rng, n, heads, D, t, pos_stride=None, head_stride=None, offset=0, scale=1.0):
        self.n, self.heads, self.D, self.t, self.offset = n, heads, D, t, offset
        self.head = D if head_stride is None else head_stride
        self.pos = heads * self.head if pos_stride is None else pos_stride
        self.size = 4 if t == sjk.F32 else 2
        self.words = offset + max(1, (n - 1) * self.pos + (heads - 1) * self.head + D) + 16
        self.host = to_bits(rng.standard_normal(self.words).astype(np.float32) * scale, t)
        self.dev, self.d = dev, dev.put(self.host)
        self.ptr = self.d.value + offset * self.size

    def index(self):
        return (self.offset + np.arange(self.n)[:, None, None] * self.pos + np.arange(self.heads)[None, :, None] * self.head +
                np.arange(self.D))

    def values(self):
        return from_bits(self.host, self.t)[self.index()]

    def read(self):
        return self.dev.get(self.d, self.words * self.size, self.host.dtype)

    def set(self, at, value):
        flat = from_bits(self.host, self.t).copy()
        flat[self.index()[at]] = value
        self.host = to_bits(flat, self.t)
        self.dev.upload(self.d, self.host)


def head_job(x, out, rope=0, rotate=0, d_norm=None, norm_head=0, eps=EPS):
    return sjk.HeadJob(x.ptr, out.ptr, x.pos, x.head, out.pos, out.head, x.t, out.t, x.heads, rope, rotate, eps, d_norm, norm_head)


def make_rope(dev, r):
    return sjk.Rope(r["layout"], r["n_rot"], int(r.get("inverse", 0)), r.get("mscale", 1.0), dev.put(r["turns"]).value if r["n_rot"] else None)


def run_rows(lib, dev, jobs, n, D, rope=None, pos0=0, d_pos=None, stream=None):
    arr = (sjk.HeadJob * len(jobs))(*jobs)
    rc = lib.sjk_hip_head_rows(arr, len(jobs), n, D, C.byref(rope) if rope is not None else None, pos0, d_pos, stream)
    sjk.check(rc, "sjk_hip_head_rows")
    dev.sync()


def untouched(out):
    """what a call wrote outside its rows: nothing"""
    keep = np.ones(out.words, bool)
    keep[out.index().ravel()] = False
    now = out.read()
    assert np.array_equal(now[keep], out.host[keep])
    return now[out.index()]


# (D, n_rot, layout): whole heads, parts of a multiple of 16 and not, one pair, odd widths, widths past every lane count
SHAPES = [(128, 128, 0), (128, 128, 1), (256, 256, 0), (256, 64, 0), (256, 64, 1), (64, 64, 0), (512, 512, 0), (512, 128, 1),
          (80, 80, 0), (80, 32, 0), (96, 50, 0), (72, 72, 1), (192, 192, 0), (128, 2, 0), (128, 6, 1), (130, 70, 0), (33, 20, 0),
          (9, 8, 1), (2, 2, 0), (511, 510, 0)]


@pytest.mark.parametrize("D,n_rot,layout", SHAPES)
@pytest.mark.parametrize("t,t_out", [(0, 0), (1, 1), (2, 2), (2, 0)], ids=["f32", "f16", "bf16", "bf16-f32"])
def test_turn_against_64_bits(lib, dev, D, n_rot, layout, t, t_out):
    rng = np.random.default_rng(D * 1000 + n_rot + 10 * layout + t)
    rope = {"n_rot": n_rot, "layout": layout, "turns": turn_table(n_rot), "mscale": 1.25, "inverse": n_rot % 4 == 0}
    n = 5
    q, k = Set(dev, rng, n, 6, D, t), Set(dev, rng, n, 1, D, t)
    oq, ok = Set(dev, rng, n, 6, D, t_out), Set(dev, rng, n, 1, D, t_out)
    run_rows(lib, dev, [head_job(q, oq, rope=1), head_job(k, ok, rope=1)], n, D, make_rope(dev, rope), pos0=77777)
    pos = 77777 + np.arange(n)
    for x, o in ((q, oq), (k, ok)):
        ref, err = reference(x.values(), pos, rope=rope)
        check_rows(untouched(o), t_out, ref, err, "turn")
        if n_rot < D:                            # channels behind n_rot pass through, rounded once
            assert np.array_equal(o.read()[o.index()][..., n_rot:], to_bits(x.values()[..., n_rot:], t_out))


@pytest.mark.parametrize("D", [8, 16, 24, 32, 40, 48, 56])
@pytest.mark.parametrize("t,t_out", [(0, 0), (1, 1), (2, 2), (2, 0)], ids=["f32", "f16", "bf16", "bf16-f32"])
@pytest.mark.parametrize("n_rot", ["whole", "part", "odd", "none"])
def test_narrow_heads_against_64_bits(lib, dev, D, t, t_out, n_rot):
    """heads narrower than the lanes they are given, down to an eighth of them, with norm and turn, beside each other and apart:
    nothing but their own channels is read into them or written"""
    rng = np.random.default_rng(100 * D + 10 * t + t_out)
    n, c = 11, {"whole": D, "part": D // 16 * 16, "odd": D // 2 * 2 - (2 if D > 8 else 4), "none": 0}[n_rot]
    rope = {"n_rot": c, "layout": sjk.ROPE_HALVES, "turns": turn_table(c)}
    w = (1 + rng.standard_normal(D) / 4).astype(np.float32)
    pos = 500 + np.arange(n)
    for apart in (0, 16):
        x = Set(dev, rng, n, 3, D, t, head_stride=D + apart)
        o = Set(dev, rng, n, 3, D, t_out, head_stride=D + apart)
        run_rows(lib, dev, [head_job(x, o, rope=1, d_norm=dev.put(w).value)], n, D, make_rope(dev, rope), pos0=500)
        ref, err = reference(x.values(), pos, w=w, rope=rope)
        check_rows(untouched(o), t_out, ref, err, "narrow heads")


@pytest.mark.parametrize("D,n_rot,layout", [(128, 128, 0), (128, 96, 1), (80, 40, 0), (33, 20, 1)])
def test_inverse_turn_is_the_gradient(lib, dev, D, n_rot, layout):
    """sum(g (f(x + d) - f(x))) = sum(inverse(g) d): the turn is linear, so differences of any length show its gradient. Each
    side's error: the kernel's bound and the last rounding of each row, against the other factor"""
    rng = np.random.default_rng(D + n_rot)
    n, heads = 4, 3
    rope = {"n_rot": n_rot, "layout": layout, "turns": turn_table(n_rot), "mscale": 1.25}
    back = dict(rope, inverse=True)
    pos = 3000 + np.arange(n)
    x, x2, g = (Set(dev, rng, n, heads, D, sjk.F32) for _ in range(3))
    outs = []
    for r, s in ((rope, x), (rope, x2), (back, g)):
        o = Set(dev, rng, n, heads, D, sjk.F32)
        run_rows(lib, dev, [head_job(s, o, rope=1)], n, D, make_rope(dev, r), pos0=3000)
        ref, err = reference(s.values(), pos, rope=r)
        outs.append((untouched(o).view(np.float32).astype(L), err + U * (np.abs(ref) + err)))
    (f, ef), (f2, ef2), (dx, edx) = outs
    d, gv = x2.values().astype(L) - x.values().astype(L), g.values().astype(L)
    bound = (np.abs(gv) * (ef + ef2)).sum() + (np.abs(d) * edx).sum()
    assert abs((gv * (f2 - f)).sum() - (dx * d).sum()) <= bound


@pytest.mark.parametrize("D,rotate", [(128, 1), (256, 1), (64, 1), (512, 1), (128, 0), (80, 0), (1, 0), (7, 0), (200, 0)])
@pytest.mark.parametrize("t", [0, 1, 2], ids=["f32", "f16", "bf16"])
def test_norm_turn_rotation_against_64_bits(lib, dev, D, rotate, t):
    rng = np.random.default_rng(D * 10 + t)
    n, n_rot = 7, D // 2 * 2
    rope = {"n_rot": n_rot, "layout": D // 64 % 2, "turns": turn_table(n_rot, 1e6)}
    w = (1 + 0.3 * rng.standard_normal(3 * D)).astype(np.float32)
    dw = dev.put(w)
    x = Set(dev, rng, n, 3, D, t, scale=3.0)
    x.set((2, 1), 0.0)                           # a row of zeros stays one
    x.set((3, 2), 1e-4 if t == 1 else 1e-20)     # a row that eps outweighs
    pos = np.array([0, 1, -5, 2 ** 31 - 1, -2 ** 31, 131072, 3], np.int32)
    d_pos = dev.put(pos)
    for shared in (True, False):                 # one set of weights, or one for each head
        o = Set(dev, rng, n, 3, D, sjk.F32)
        wh = np.broadcast_to(w[:D], (3, D)) if shared else w.reshape(3, D)
        run_rows(lib, dev, [head_job(x, o, rope=1, rotate=rotate, d_norm=dw, norm_head=0 if shared else D)], n, D,
                 make_rope(dev, rope), d_pos=d_pos)
        ref, err = reference(x.values(), pos, w=wh[None], rope=rope, rotate=rotate)
        check_rows(untouched(o), sjk.F32, ref, err, (D, shared))
        assert not from_bits(o.read()[o.index()], 0)[2, 1].any()


@pytest.mark.parametrize("D", [64, 128, 256, 512])
def test_rotation_is_that_of_sjk_hip_rotate(lib, dev, D):
    """the rotation alone, fp32 to fp32, bit for bit, rows with infinities and NaNs of both signs among them"""
    rng = np.random.default_rng(D)
    x = Set(dev, rng, 6, 5, D, sjk.F32)
    for at, v in (((0, 1, 3), np.inf), ((1, 0, 0), -np.inf), ((1, 0, D - 1), np.inf), ((2, 2, 9), np.nan), ((4, 4, 5), 3e38),
                  ((4, 4, 6), 3e38)):
        x.set(at, v)
    x.host[x.index()[5, 3, 7]] |= 0x80000000 | 0x7FC00000
    dev.upload(x.d, x.host)
    o = Set(dev, rng, 6, 5, D, sjk.F32)
    run_rows(lib, dev, [head_job(x, o, rotate=1)], 6, D)
    rows = x.host[x.index()]
    d = dev.put(rows)
    sjk.check(lib.sjk_hip_rotate(d, 30, D, None), "sjk_hip_rotate")
    dev.sync()
    assert np.array_equal(untouched(o).reshape(30, D), dev.get(d, rows.nbytes, np.uint32).reshape(30, D))


@pytest.mark.parametrize("t", [0, 1, 2], ids=["f32", "f16", "bf16"])
@pytest.mark.parametrize("D", [128, 80])
def test_strides_offsets_and_in_place(lib, dev, D, t):
    """heads of a fused projection at odd offsets and strides, heads before positions, rows written over themselves: the same
    bits as from plain rows, and nothing between the rows touched"""
    rng = np.random.default_rng(5 * D + t)
    n, heads = 9, 5
    rope = {"n_rot": D - 16, "layout": 0, "turns": turn_table(D - 16)}
    dr, dw = make_rope(dev, rope), dev.put((1 + 0.1 * rng.standard_normal(D)).astype(np.float32))
    plain = Set(dev, rng, n, heads, D, t)
    want = Set(dev, rng, n, heads, D, t)
    run_rows(lib, dev, [head_job(plain, want, rope=1, d_norm=dw)], n, D, dr, pos0=11)
    want = want.read()[want.index()]
    for pos_stride, head_stride, offset in ((heads * D + 3, None, 0), (heads * D + 8, None, 8), (None, D + 1, 1), (D, n * D, 0), (heads * D, D, 3)):
        x = Set(dev, rng, n, heads, D, t, pos_stride, head_stride, offset)
        x.host[x.index()] = plain.host[plain.index()]
        dev.upload(x.d, x.host)
        o = Set(dev, rng, n, heads, D, t, offset=offset, pos_stride=heads * D + 7)
        run_rows(lib, dev, [head_job(x, o, rope=1, d_norm=dw)], n, D, dr, pos0=11)
        assert np.array_equal(untouched(o), want)
        run_rows(lib, dev, [head_job(x, x, rope=1, d_norm=dw)], n, D, dr, pos0=11)          # in place
        assert np.array_equal(untouched(x), want)


def test_rows_do_not_depend_on_their_neighbours(lib, dev):
    """a row has the same bits alone and among 3,000 positions, in a call of one job and of several types; a NaN or an infinity
    stays in its own row"""
    rng = np.random.default_rng(3)
    n, D = 3001, 128
    rope = {"n_rot": 128, "layout": 0, "turns": turn_table(128)}
    dr, dw = make_rope(dev, rope), dev.put((1 + 0.1 * rng.standard_normal(D)).astype(np.float32))
    x, o = Set(dev, rng, n, 40, D, sjk.BF16), Set(dev, rng, n, 40, D, sjk.F32)
    run_rows(lib, dev, [head_job(x, o, rope=1, rotate=1, d_norm=dw)], n, D, dr, pos0=500)
    full = untouched(o)
    for p in (0, 1, 1499, 3000):
        one, out = Set(dev, rng, 1, 40, D, sjk.BF16), Set(dev, rng, 1, 40, D, sjk.F32)
        one.host[one.index()] = x.host[x.index()[p:p + 1]]
        dev.upload(one.d, one.host)
        other, oo = Set(dev, rng, 1, 2, D, sjk.F16), Set(dev, rng, 1, 2, D, sjk.F16)
        extra = [Set(dev, rng, 1, h, D, sjk.BF16) for h in (1, 3, 0, 4, 1)]
        run_rows(lib, dev, [head_job(other, oo)] + [head_job(e, e) for e in extra] + [head_job(one, out, rope=1, rotate=1, d_norm=dw)],
                 1, D, dr, pos0=500 + p)
        assert np.array_equal(untouched(out)[0], full[p])
        assert np.array_equal(untouched(oo), other.host[other.index()])                        # no step asked for: a copy
    x.set((7, 3, 5), np.nan)
    x.set((7, 4, 0), np.inf)
    run_rows(lib, dev, [head_job(x, o, rope=1, rotate=1, d_norm=dw)], n, D, dr, pos0=500)
    again = untouched(o)
    assert np.isnan(from_bits(again[7, 3], 0)).all() and np.isnan(from_bits(again[7, 4], 0)).all()
    again[7, 3:5] = full[7, 3:5]
    assert np.array_equal(again, full)


@pytest.mark.parametrize("D,t,t_out,heads", [(128, 2, 2, 40), (128, 2, 0, 40), (80, 1, 1, 13), (256, 0, 0, 6), (64, 2, 0, 9), (96, 1, 2, 33)])
@pytest.mark.parametrize("n_rot", ["whole", "part", "odd"])
def test_rows_of_a_large_call_are_those_of_small_ones(lib, dev, D, t, t_out, heads, n_rot):
    """many positions of many heads, each head with weights of its own: wavefronts that go through runs of heads, and last
    rows and runs that are not full, against the same rows one position at a time"""
    rng = np.random.default_rng(D + heads)
    n = 1501
    n_rot = {"whole": D, "part": D // 32 * 16, "odd": D // 2 - 2}[n_rot]
    rope = {"n_rot": n_rot, "layout": 0, "turns": turn_table(n_rot)}
    dr, dw = make_rope(dev, rope), dev.put((1 + 0.3 * rng.standard_normal(heads * D)).astype(np.float32))
    x, o = Set(dev, rng, n, heads, D, t, pos_stride=heads * D + 16), Set(dev, rng, n, heads, D, t_out)
    run_rows(lib, dev, [head_job(x, o, rope=1, d_norm=dw, norm_head=D)], n, D, dr, pos0=9000)
    got = untouched(o)
    for p in (0, 1, 750, 1499, 1500):
        a, b = Set(dev, rng, 1, heads, D, t), Set(dev, rng, 1, heads, D, t_out)
        a.host[a.index()] = x.host[x.index()[p:p + 1]]
        dev.upload(a.d, a.host)
        run_rows(lib, dev, [head_job(a, b, rope=1, d_norm=dw, norm_head=D)], 1, D, dr, pos0=9000 + p)
        assert np.array_equal(untouched(b)[0], got[p]), p
        ref, err = reference(a.values(), np.array([9000 + p]), w=from_bits(dev.get(dw, heads * D * 4, np.uint32), 0).reshape(1, heads, D), rope=rope)
        check_rows(got[p:p + 1], t_out, ref, err, p)
    if t == t_out:                               # over themselves
        run_rows(lib, dev, [head_job(x, x, rope=1, d_norm=dw, norm_head=D)], n, D, dr, pos0=9000)
        assert np.array_equal(untouched(x), got)


def test_inverse_turns_back(lib, dev):
    rng = np.random.default_rng(8)
    rope = {"n_rot": 96, "layout": 0, "turns": turn_table(96)}
    x, o = Set(dev, rng, 33, 4, 128, sjk.F32), Set(dev, rng, 33, 4, 128, sjk.F32)
    r = make_rope(dev, rope)
    run_rows(lib, dev, [head_job(x, o, rope=1)], 33, 128, r, pos0=123456)
    r.inverse = 1
    run_rows(lib, dev, [head_job(o, o, rope=1)], 33, 128, r, pos0=123456)
    a, b = from_bits(x.host[x.index()], 0).astype(np.float64), from_bits(o.read()[o.index()], 0).astype(np.float64)
    half = np.concatenate([np.abs(a[..., :48]) + np.abs(a[..., 48:96])] * 2 + [0 * a[..., 96:]], -1)
    assert np.all(np.abs(a - b) <= 2 * 8 * U * np.sqrt(2) * half + 1e-30)    # two turns, each 8 U of the pair's magnitudes


# ---- the append -----------------------------------------------------------------------------------------------------

TAIL, TAIL_MAX = 256, 512


def new_layer(lib, D, H, staging, sink_type, n_ubatch=64):
    cfg = lib.sj_kvarn_config_default(D, H, 4096, n_ubatch)
    cfg.tail, cfg.tail_max, cfg.staging, cfg.sink_type = TAIL, TAIL_MAX, staging, sink_type
    PL = sjk.Layer()
    sjk.check(lib.sj_kvarn_layer_init(C.byref(PL), C.byref(cfg)), "layer_init")
    return PL


def cache_bytes(dev, v):
    sb = v.S * v.n_head_kv * (4 * v.lay.D if v.sink_type == 0 else 2 * v.stage_bytes)
    return (dev.get(C.c_void_p(v.sink), sb, np.uint8), dev.get(C.c_void_p(v.ring), v.cap * v.n_head_kv * 2 * v.stage_bytes, np.uint8))


class Proj:
    """a projection's rows [n][n_head + 2 H][D] and what a layer does with them"""

    def __init__(self, dev, rng, n, n_head, H, D, t, norm, n_rot, layout, rotate_v=1, pad=0):
        self.dev, self.n, self.n_head, self.H, self.D = dev, n, n_head, H, D
        self.x = Set(dev, rng, n, n_head + 2 * H, D, t, pos_stride=(n_head + 2 * H) * D + pad, scale=2.0)
        self.q = dev.alloc(max(1, n * n_head * D) * 4)
        m = self.m = sjk.Qkv()
        m.type, m.n_head, m.rotate_qk, m.rotate_v, m.eps = t, n_head, 1, rotate_v, EPS
        m.q_pos = m.k_pos = m.v_pos = self.x.pos
        m.q_head = m.k_head = m.v_head = D
        if norm:
            self.w = [dev.put((1 + 0.2 * rng.standard_normal(D)).astype(np.float32)) for _ in range(2)]
            m.d_q_norm, m.d_k_norm = self.w[0].value, self.w[1].value
        m.rope = make_rope(dev, {"n_rot": n_rot, "layout": layout, "turns": turn_table(n_rot)})

    def at(self, head, i=0):
        return self.x.ptr + (i * self.x.pos + head * self.D) * self.x.size

    def ptrs(self, i=0):
        return self.at(0, i), self.at(self.n_head, i), self.at(self.n_head + self.H, i)

    def q_out(self, n=None):
        n = self.n if n is None else n
        return self.dev.get(self.q, n * self.n_head * self.D * 4, np.uint32)

    def two_steps(self, lib, view, pos0, n=None, i=0, d_pos=None):
        """the same through sjk_hip_head_rows to fp32 and sjk_hip_layer_store; returns the queries' bits"""
        n, D, H, m, dev = self.n if n is None else n, self.D, self.H, self.m, self.dev
        k, v = dev.alloc(n * H * D * 4), dev.alloc(n * H * D * 4)
        q = dev.alloc(max(1, n * self.n_head * D) * 4)
        turn = int(m.rope.n_rot > 0)
        jobs = [sjk.HeadJob(self.at(0, i), q.value, self.x.pos, D, self.n_head * D, D, m.type, 0, self.n_head, turn, m.rotate_qk, EPS, m.d_q_norm, 0),
                sjk.HeadJob(self.at(self.n_head, i), k.value, self.x.pos, D, H * D, D, m.type, 0, H, turn, 0, EPS, m.d_k_norm, 0),
                sjk.HeadJob(self.at(self.n_head + H, i), v.value, self.x.pos, D, H * D, D, m.type, 0, H, 0, 0, EPS, None, 0)]
        run_rows(lib, dev, jobs, n, D, m.rope, pos0=pos0, d_pos=d_pos)
        if not m.rotate_v:                       # the store rotates both: undo the values' by rotating them first is not exact,
            sjk.check(lib.sjk_hip_rotate(k, n * H, D, None), "rotate")     # so rotate the keys here and store as they are
        sjk.check(lib.sjk_hip_layer_store(C.byref(view), pos0, n, k, v, int(m.rotate_v), None), "layer_store")
        dev.sync()
        return dev.get(q, n * self.n_head * D * 4, np.uint32)


APPENDS = [(128, 2, 8, 0, 0, 2, True, 128, 0), (256, 4, 16, 0, 0, 2, True, 256, 0), (256, 1, 5, 1, 0, 1, False, 64, 1),
           (128, 8, 32, 1, 1, 0, True, 40, 0), (128, 3, 3, 0, 1, 1, True, 128, 1), (256, 2, 0, 0, 0, 0, False, 0, 0),
           (128, 1, 1, 0, 0, 0, True, 64, 1)]


@pytest.mark.parametrize("D,H,n_head,staging,sink_type,t,norm,n_rot,layout", APPENDS)
def test_append_is_head_rows_then_layer_store(lib, dev, D, H, n_head, staging, sink_type, t, norm, n_rot, layout):
    rng = np.random.default_rng(D + H + n_head + t)
    A, B = new_layer(lib, D, H, staging, sink_type), new_layer(lib, D, H, staging, sink_type)
    va, vb = lib.sjk_layer_view(C.byref(A)), lib.sjk_layer_view(C.byref(B))
    try:
        # one position, the sink's end, a ubatch across it, odd counts, the ring's wrap and past it
        for pos0, n, pad in ((0, 1, 0), (1, 126, 0), (127, 1, 3), (100, 60, 8), (500, 37, 1), (128 + va.cap - 5, 11, 0),
                             (5 * va.cap + 60, va.cap, 0)):
            p = Proj(dev, rng, n, n_head, H, D, t, norm, n_rot, layout, rotate_v=int(n != 37), pad=pad)
            want_q = p.two_steps(lib, vb, pos0)
            q, k, v = p.ptrs()
            sjk.check(lib.sjk_hip_store_qkv(C.byref(va), pos0, n, C.byref(p.m), None, q, k, v, p.q if n_head else None, None), "store_qkv")
            dev.sync()
            assert np.array_equal(p.q_out(), want_q) if n_head else True
            for got, want in zip(cache_bytes(dev, va), cache_bytes(dev, vb)):
                assert np.array_equal(got, want), (pos0, n)
    finally:
        lib.sj_kvarn_layer_free(C.byref(A))
        lib.sj_kvarn_layer_free(C.byref(B))


@pytest.mark.parametrize("D,staging", [(128, 0), (256, 0), (128, 1)])
def test_append_of_rows_that_are_not_finite(lib, dev, D, staging):
    """infinities, NaNs of both signs, rows that overflow, zeros: the bytes of the two steps, other rows as they were"""
    rng = np.random.default_rng(D + staging)
    A, B = new_layer(lib, D, 2, staging, 0), new_layer(lib, D, 2, staging, 0)
    va, vb = lib.sjk_layer_view(C.byref(A)), lib.sjk_layer_view(C.byref(B))
    try:
        for norm in (False, True):
            p = Proj(dev, rng, 70, 4, 2, D, sjk.F32, norm, D, 0)
            x = p.x
            for i, (at, v) in enumerate((((0, 4), 0.0), ((1, 5, 3), np.inf), ((2, 6, 0), -np.inf), ((3, 7, 9), np.nan), ((4, 4, 5), 3e38),
                                         ((4, 4, 6), 3e38), ((5, 6), 1e-42), ((66, 4, 1), np.inf), ((66, 5, 2), np.nan), ((67, 7), 0.0))):
                x.set(at, v)
            x.host[x.index()[3, 6, 2]] = 0xFFC00001
            dev.upload(x.d, x.host)
            want_q = p.two_steps(lib, vb, 100)
            q, k, v = p.ptrs()
            sjk.check(lib.sjk_hip_store_qkv(C.byref(va), 100, 70, C.byref(p.m), None, q, k, v, p.q, None), "store_qkv")
            dev.sync()
            a, b = from_bits(p.q_out(), 0), from_bits(want_q, 0)
            assert np.array_equal(p.q_out(), want_q) or np.array_equal(np.isnan(a), np.isnan(b))
            for got, want in zip(cache_bytes(dev, va), cache_bytes(dev, vb)):
                assert np.array_equal(got, want), norm
    finally:
        lib.sj_kvarn_layer_free(C.byref(A))
        lib.sj_kvarn_layer_free(C.byref(B))


# whole turns, parts, parts by LDS, odd addresses; runs of 7, 5 and 6 heads of keys and values a wavefront
@pytest.mark.parametrize("D,H,n_head,n,t,n_rot,pad", [(128, 7, 2, 4211, sjk.BF16, 128, 0), (128, 5, 0, 4211, sjk.F32, 128, 0),
                                                      (256, 5, 1, 2111, sjk.F32, 40, 0), (128, 6, 1, 4211, sjk.F16, 64, 0),
                                                      (128, 7, 1, 4211, sjk.F32, 128, 3)])
def test_large_append_with_rows_that_are_not_finite(lib, dev, D, H, n_head, n, t, n_rot, pad):
    """calls so large that a wavefront stages more heads than it walks at once, and a number of them that is no multiple; rows
    with infinities and NaNs of both signs in some of them"""
    rng = np.random.default_rng(D + H + n)
    A, B = (new_layer(lib, D, H, 0, 0, n_ubatch=4352) for _ in range(2))
    va, vb = lib.sjk_layer_view(C.byref(A)), lib.sjk_layer_view(C.byref(B))
    try:
        p = Proj(dev, rng, n, n_head, H, D, t, True, n_rot, 0, pad=pad)
        for specials in (False, True):
            if specials:
                flat = from_bits(p.x.host, t).copy()
                at = rng.choice(p.x.index().ravel(), 200, replace=False)
                flat[at] = rng.choice(np.array([np.inf, -np.inf, np.nan, -np.nan, 0.0], np.float32), 200)
                p.x.host = to_bits(flat, t)
                dev.upload(p.x.d, p.x.host)
            want_q = p.two_steps(lib, vb, 100)
            q, k, v = p.ptrs()
            sjk.check(lib.sjk_hip_store_qkv(C.byref(va), 100, n, C.byref(p.m), None, q, k, v, p.q if n_head else None, None), "store_qkv")
            dev.sync()
            if n_head:
                a, b = from_bits(p.q_out(), 0), from_bits(want_q, 0)
                assert np.array_equal(p.q_out(), want_q) or (specials and np.array_equal(np.isnan(a), np.isnan(b)))
            for got, want in zip(cache_bytes(dev, va), cache_bytes(dev, vb)):
                assert np.array_equal(got, want), specials
    finally:
        lib.sj_kvarn_layer_free(C.byref(A))
        lib.sj_kvarn_layer_free(C.byref(B))


def test_append_at_positions_of_its_own_and_over_its_queries(lib, dev):
    """d_pos turns by other positions than the slots'; fp32 queries may be written over themselves"""
    rng = np.random.default_rng(21)
    D, H, n_head, n = 128, 2, 4, 19
    A, B = new_layer(lib, D, H, 0, 0), new_layer(lib, D, H, 0, 0)
    va, vb = lib.sjk_layer_view(C.byref(A)), lib.sjk_layer_view(C.byref(B))
    try:
        p = Proj(dev, rng, n, n_head, H, D, sjk.F32, True, D, 0)
        d_pos = dev.put(rng.integers(-2 ** 31, 2 ** 31, n).astype(np.int32))
        want_q = p.two_steps(lib, vb, 300, d_pos=d_pos)
        rows = from_bits(p.x.host[p.x.index()], 0)
        dq, dk, dv = (dev.put(np.ascontiguousarray(rows[:, a:b])) for a, b in ((0, 4), (4, 6), (6, 8)))
        p.m.q_pos, p.m.k_pos, p.m.v_pos = n_head * D, H * D, H * D
        sjk.check(lib.sjk_hip_store_qkv(C.byref(va), 300, n, C.byref(p.m), d_pos, dq, dk, dv, dq, None), "store_qkv")
        dev.sync()
        assert np.array_equal(dev.get(dq, want_q.nbytes, np.uint32), want_q)
        for got, want in zip(cache_bytes(dev, va), cache_bytes(dev, vb)):
            assert np.array_equal(got, want)
    finally:
        lib.sj_kvarn_layer_free(C.byref(A))
        lib.sj_kvarn_layer_free(C.byref(B))


def test_batch_of_unlike_views(lib, dev):
    """37 jobs (two launches and more): staging, sink type and capacity differ from job to job; each as by its own call"""
    rng = np.random.default_rng(2)
    D, H, n_head, n = 128, 2, 3, 5
    kinds = [(0, 0, 64), (0, 0, 128), (1, 0, 64), (1, 1, 64), (0, 1, 64)]
    layers = [[new_layer(lib, D, H, *kinds[i * 5 // 37]) for i in range(37)] for _ in range(2)]
    views = [[lib.sjk_layer_view(C.byref(PL)) for PL in side] for side in layers]
    try:
        p = Proj(dev, rng, 37 * n, n_head, H, D, sjk.BF16, True, 64, 0)
        jobs = (sjk.QkvJob * 37)()
        starts = [int(rng.integers(0, 3000)) for _ in range(37)]
        for i in range(37):
            q, k, v = p.ptrs(i * n)
            jobs[i] = sjk.QkvJob(views[0][i], starts[i], None, q, k, v, p.q.value + i * n * n_head * D * 4)
        sjk.check(lib.sjk_hip_store_qkv_batch(jobs, 37, n, C.byref(p.m), None), "store_qkv_batch")
        dev.sync()
        got = p.q_out().reshape(37, -1)
        for i in range(37):
            want = p.two_steps(lib, views[1][i], starts[i], n, i * n)
            assert np.array_equal(got[i], want), i
            for a, b in zip(cache_bytes(dev, views[0][i]), cache_bytes(dev, views[1][i])):
                assert np.array_equal(a, b), i
    finally:
        for side in layers:
            for PL in side:
                lib.sj_kvarn_layer_free(C.byref(PL))


def test_captured_append_replays_every_step(lib, dev):
    """sjk_hip_store_qkv_dyn captured once: replayed over the sink, the ring and its wrap it writes what eager calls write, and
    nothing for a negative position. sjk_hip_head_rows in the same graph reads its positions on the device."""
    rng = np.random.default_rng(12)
    D, H, n_head, w = 256, 4, 16, 3
    A, B = new_layer(lib, D, H, 0, 0), new_layer(lib, D, H, 0, 0)
    va, vb = lib.sjk_layer_view(C.byref(A)), lib.sjk_layer_view(C.byref(B))
    hip = dev.hip
    hip.hipStreamBeginCapture.argtypes = [C.c_void_p, C.c_int]
    hip.hipStreamEndCapture.argtypes = [C.c_void_p, C.POINTER(C.c_void_p)]
    hip.hipGraphInstantiate.argtypes = [C.POINTER(C.c_void_p), C.c_void_p, C.c_void_p, C.c_char_p, C.c_size_t]
    hip.hipGraphLaunch.argtypes = [C.c_void_p, C.c_void_p]
    hip.hipGraphExecDestroy.argtypes = [C.c_void_p]
    hip.hipGraphDestroy.argtypes = [C.c_void_p]
    stream, graph, gexec = dev.stream(), C.c_void_p(), C.c_void_p()
    try:
        p = Proj(dev, rng, w, n_head, H, D, sjk.BF16, True, D, 0)
        desc = np.zeros(16, np.int32)
        d_desc, d_pos = dev.put(desc), dev.put(np.zeros(w, np.int32))
        o = Set(dev, rng, w, n_head, D, sjk.F32)
        q, k, v = p.ptrs()
        hj = sjk.HeadJob(q, o.ptr, p.x.pos, D, o.pos, D, sjk.BF16, sjk.F32, n_head, 1, 1, EPS, p.m.d_q_norm, 0)
        dev.sync()
        dev._ck(hip.hipStreamBeginCapture(stream, 2), "hipStreamBeginCapture")
        rc = lib.sjk_hip_store_qkv_dyn(C.byref(va), d_desc, w, C.byref(p.m), None, q, k, v, p.q, stream)
        rc2 = lib.sjk_hip_head_rows(C.byref(hj), 1, w, D, C.byref(p.m.rope), 0, d_pos, stream)
        dev._ck(hip.hipStreamEndCapture(stream, C.byref(graph)), "hipStreamEndCapture")
        sjk.check(rc, "store_qkv_dyn")
        sjk.check(rc2, "head_rows")
        dev._ck(hip.hipGraphInstantiate(C.byref(gexec), graph, None, None, 0), "hipGraphInstantiate")
        for p0 in (0, 126, 128, 500, 128 + va.cap - 1, 70000):
            x = rng.standard_normal((w, n_head + 2 * H, D)).astype(np.float32)
            p.x.host[p.x.index()] = to_bits(x, sjk.BF16)
            dev.upload(p.x.d, p.x.host)
            desc[4] = p0
            dev.upload(d_desc, desc)
            dev.upload(d_pos, np.arange(p0, p0 + w, dtype=np.int32))
            dev._ck(hip.hipGraphLaunch(gexec, stream), "hipGraphLaunch")
            dev._ck(hip.hipStreamSynchronize(stream), "hipStreamSynchronize")
            got_q, got_o = p.q_out().copy(), o.read()[o.index()].ravel()
            sjk.check(lib.sjk_hip_store_qkv(C.byref(vb), p0, w, C.byref(p.m), None, q, k, v, p.q, None), "store_qkv")
            dev.sync()
            assert np.array_equal(got_q, p.q_out()) and np.array_equal(got_o, got_q), p0
            for a, b in zip(cache_bytes(dev, va), cache_bytes(dev, vb)):
                assert np.array_equal(a, b), p0
        desc[4] = -1
        dev.upload(d_desc, desc)
        marks = np.arange(w * n_head * D, dtype=np.uint32)
        dev.upload(p.q, marks)
        dev._ck(hip.hipGraphLaunch(gexec, stream), "hipGraphLaunch")
        dev._ck(hip.hipStreamSynchronize(stream), "hipStreamSynchronize")
        assert np.array_equal(p.q_out(), marks)
        for a, b in zip(cache_bytes(dev, va), cache_bytes(dev, vb)):
            assert np.array_equal(a, b)
    finally:
        if gexec.value:
            hip.hipGraphExecDestroy(gexec)
        if graph.value:
            hip.hipGraphDestroy(graph)
        lib.sj_kvarn_layer_free(C.byref(A))
        lib.sj_kvarn_layer_free(C.byref(B))


def test_rows_past_32_bits(lib, dev):
    """positions 3 GiB apart, read and written: the bits of rows on end"""
    rng = np.random.default_rng(3)
    n, heads, D, far = 3, 2, 128, 3 << 29        # elements of 2 bytes
    x, o = Set(dev, rng, n, heads, D, sjk.BF16), Set(dev, rng, n, heads, D, sjk.BF16)
    rope = make_rope(dev, {"n_rot": D, "layout": 0, "turns": turn_table(D)})
    run_rows(lib, dev, [head_job(x, o, rope=1)], n, D, rope, pos0=9)
    want = untouched(o)
    row = heads * D * 2
    big, out = (dev.alloc((n - 1) * far * 2 + row, zero=False).value for _ in range(2))
    for i in range(n):
        dev.upload(C.c_void_p(big + 2 * i * far), x.host[x.index()[i]])
    run_rows(lib, dev, [sjk.HeadJob(big, out, far, D, far, D, x.t, x.t, heads, 1, 0, EPS, None, 0)], n, D, rope, pos0=9)
    for i in range(n):
        assert np.array_equal(dev.get(C.c_void_p(out + 2 * i * far), row, np.uint16), want[i].ravel())


@pytest.mark.parametrize("staging", [0, 1])
def test_slots_past_32_bits(lib, dev, staging):
    """a ring of 5 GiB: the staged rows of a far slot are those of a small ring's"""
    rng = np.random.default_rng(4 + staging)
    D, H, n_head, n = 256, 8, 8, 21
    A = new_layer(lib, D, H, staging, 0)
    va = lib.sjk_layer_view(C.byref(A))
    try:
        entry = H * 2 * va.stage_bytes
        vb = sjk.View.from_buffer_copy(va)
        vb.cap = (5 << 30) // entry
        vb.ring = dev.alloc(vb.cap * entry, zero=False).value
        at = vb.cap - 40                         # its slot; the last of the n is 19 before the ring's end
        pos0 = va.S + at
        p = Proj(dev, rng, n, n_head, H, D, sjk.BF16, True, D, 0)
        want_q = p.two_steps(lib, va, pos0)
        q, k, v = p.ptrs()
        sjk.check(lib.sjk_hip_store_qkv(C.byref(vb), pos0, n, C.byref(p.m), None, q, k, v, p.q, None), "store_qkv")
        dev.sync()
        assert at * entry > 1 << 32 and np.array_equal(p.q_out(), want_q)
        small = cache_bytes(dev, va)[1].reshape(va.cap, entry)
        got = dev.get(C.c_void_p(vb.ring + at * entry), n * entry, np.uint8).reshape(n, entry)
        assert np.array_equal(got, small[(at + np.arange(n)) % va.cap])
    finally:
        lib.sj_kvarn_layer_free(C.byref(A))


def test_two_streams_at_once(lib, dev):
    """two layers' appends from two streams at once, 20 times: the bytes of one after the other"""
    rng = np.random.default_rng(31)
    D, H, n_head, n = 128, 4, 8, 200
    layers = [new_layer(lib, D, H, 0, 0, n_ubatch=256) for _ in range(4)]
    views = [lib.sjk_layer_view(C.byref(PL)) for PL in layers]
    streams = [dev.stream(), dev.stream()]
    try:
        ps = [Proj(dev, rng, n, n_head, H, D, t, True, D, 0) for t in (sjk.F16, sjk.F32)]
        dev.sync()
        for r in range(20):
            for i, p in enumerate(ps):
                q, k, v = p.ptrs()
                sjk.check(lib.sjk_hip_store_qkv(C.byref(views[i]), 100 + 200 * r, n, C.byref(p.m), None, q, k, v, p.q, streams[i]), "store")
        dev.sync()
        got = [p.q_out().copy() for p in ps]
        for i, p in enumerate(ps):
            q, k, v = p.ptrs()
            for r in range(20):
                sjk.check(lib.sjk_hip_store_qkv(C.byref(views[2 + i]), 100 + 200 * r, n, C.byref(p.m), None, q, k, v, p.q, None), "store")
            dev.sync()
            assert np.array_equal(got[i], p.q_out())
            for a, b in zip(cache_bytes(dev, views[i]), cache_bytes(dev, views[2 + i])):
                assert np.array_equal(a, b)
    finally:
        for PL in layers:
            lib.sj_kvarn_layer_free(C.byref(PL))
