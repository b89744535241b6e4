"""Small caches for the tests of listed groups and drafted nodes: layers filled through the product path (store, commit), their
rows as the device resolves them (sjk_hip_kv_rows), and attention over any of their positions in 64 bits."""
import ctypes as C
import sys

import numpy as np

import cabi
import inputs

sys.path.insert(0, cabi.PKG)
import sjk  # noqa: E402

S, G = 128, 128
U = 2.0 ** -24                                   # half a step of fp32, relative
HALF = {sjk.F32: U, sjk.F16: 2.0 ** -11, sjk.BF16: 2.0 ** -8}
TINY = {sjk.F32: 2.0 ** -149, sjk.F16: 2.0 ** -24, sjk.BF16: 2.0 ** -133}


class Ctx:
    """a layer of n_groups sealed groups and `tail` staged positions behind them (short: no group, `tail` positions in all)"""

    def __init__(self, lib, dev, D, H, bits=(4, 4, 0), staging=0, sink_type=0, n_groups=0, tail=0, seed=1, n_ubatch=256):
        self.lib, self.dev, self.D, self.H, self.n_groups = lib, dev, D, H, n_groups
        cfg = lib.sj_kvarn_config_default(D, H, S + G * n_groups + tail + 1024, n_ubatch)
        cfg.bits_k, cfg.bits_v, cfg.body = bits
        cfg.staging, cfg.sink_type, cfg.tail, cfg.tail_max = staging, sink_type, 128, 256
        self.L = sjk.Layer()
        sjk.check(lib.sj_kvarn_layer_init(C.byref(self.L), C.byref(cfg)), "layer_init")
        self.cfg, self.view = cfg, lib.sjk_layer_view(C.byref(self.L))
        self.B = S + G * n_groups
        self.N = self.B + tail if n_groups else tail
        self.seed = seed
        at = 0
        for end in ([S + G * (g + 1) for g in range(n_groups)] if n_groups else []) + [self.N]:
            self.store(at, end - at)
            if end <= self.B and n_groups:
                sjk.check(lib.sjk_hip_commit(C.byref(self.view), 1, end - G, end, 16, None), "commit")
            at = end
        dev.sync()

    def store(self, pos0, n):
        for p in range(pos0, pos0 + n, 128):
            m = min(128, pos0 + n - p)
            K, V = inputs.kv_rows(m, self.H, self.D, seed=1000 * self.seed + p)
            dK, dV = self.dev.put(K), self.dev.put(V)
            sjk.check(self.lib.sjk_hip_layer_store(C.byref(self.view), p, m, dK, dV, 1, None), "layer_store")
            self.dev.sync()
            self.dev.free(dK)
            self.dev.free(dV)

    def rows(self, end, view=None, B=None):
        """K and V [H][end][D] in 64 bits"""
        v, B = view or self.view, self.B if B is None else B
        K, V = np.empty((self.H, end, self.D)), np.empty((self.H, end, self.D))
        k, w = self.dev.alloc(end * self.D * 4), self.dev.alloc(end * self.D * 4)
        for h in range(self.H):
            sjk.check(self.lib.sjk_hip_kv_rows(C.byref(v), B, 0, end, h, k, w, None), "kv_rows")
            self.dev.sync()
            K[h] = self.dev.get(k, end * self.D * 4, np.float32).reshape(end, self.D)
            V[h] = self.dev.get(w, end * self.D * 4, np.float32).reshape(end, self.D)
        self.dev.free(k)
        self.dev.free(w)
        return K, V

    def close(self):
        self.dev.sync()
        self.lib.sj_kvarn_layer_free(C.byref(self.L))


def attention(q, K, V, seen, scale):
    """q [n_q][n_head][D] over K, V [H][n][D]; seen [n_q][H][n] -> (out, bound on an fp32 output's error), in 64 bits.

    The bound counts, in units of U: a score's terms (the products of 256 channels and the zero point, before they cancel at most
    four times |q| |K|) once for each of the D + 64 sums and roundings; twice that for the weight and the sum of weights; the
    values' products with both parts of a weight, 256 a record, each rounded at the place of a sum of at most 2.5 times the largest
    value (codes from one end of their range)."""
    n_q, n_head, D = q.shape
    H = K.shape[0]
    per = n_head // H
    out, tol = np.zeros(q.shape), np.zeros(q.shape)
    for i in range(n_q):
        for hq in range(n_head):
            h = hq // per
            m = seen[i, h]
            if not m.any():
                continue
            k, v = K[h][m], V[h][m]
            x = (k @ q[i, hq].astype(np.float64)) * scale
            p = np.exp(x - x.max())
            p /= p.sum()
            out[i, hq] = p @ v
            terms = 4 * np.abs(scale) * (np.abs(k) @ np.abs(q[i, hq].astype(np.float64)))
            w = 2 * (D + 64) * U * terms.max()
            tol[i, hq] = np.abs(v).max(0) * (w + 2.5 * 256 * U) + U * np.abs(out[i, hq])
    return out, tol


def values(bits, t):
    if t == sjk.F32:
        return bits.view(np.float32).astype(np.float64)
    if t == sjk.F16:
        return bits.view(np.float16).astype(np.float64)
    return (bits.astype(np.uint32) << 16).view(np.float32).astype(np.float64)


def out_dtype(t):
    return np.uint32 if t == sjk.F32 else np.uint16


class Out:
    """an output buffer between guard bytes"""

    def __init__(self, dev, n, t):
        self.dev, self.n, self.t, self.size = dev, n, t, n * (4 if t == sjk.F32 else 2)
        self.p = dev.put(np.full(self.size + 512, 0xA5, np.uint8))
        self.at = C.c_void_p(self.p.value + 256)

    def bits(self):
        self.dev.sync()
        b = self.dev.get(self.p, self.size + 512, np.uint8)
        assert (b[:256] == 0xA5).all() and (b[256 + self.size:] == 0xA5).all(), "written outside the output"
        return b[256:256 + self.size].view(out_dtype(self.t)).copy()

    def get(self):
        return values(self.bits(), self.t)


def check(got, want, tol, t, what=""):
    bound = tol + HALF[t] * (np.abs(want) + tol) + TINY[t]
    bad = ~(np.abs(got - want) <= bound)
    assert not bad.any(), (what, int(bad.sum()), np.abs(got - want)[bad][:4], bound[bad][:4])


def check_norm(got, want, most, what=""):
    """2-norm of the error over that of the result"""
    rel = np.linalg.norm(got - want) / np.linalg.norm(want)
    assert rel <= most, (what, rel, most)


class Graph:
    """calls captured once on a stream of their own, replayed"""

    def __init__(self, dev, stream, calls):
        hip = self.hip = dev.hip
        self.dev, self.stream = dev, stream
        hip.hipStreamBeginCapture.argtypes = [C.c_void_p, C.c_int]
        hip.hipStreamEndCapture.argtypes = [C.c_void_p, C.POINTER(C.c_void_p)]
        hip.hipGraphInstantiate.argtypes = [C.POINTER(C.c_void_p), C.c_void_p, C.c_void_p, C.c_char_p, C.c_size_t]
        hip.hipGraphLaunch.argtypes = [C.c_void_p, C.c_void_p]
        hip.hipGraphExecDestroy.argtypes = [C.c_void_p]
        hip.hipGraphDestroy.argtypes = [C.c_void_p]
        self.graph, self.exec = C.c_void_p(), C.c_void_p()
        dev._ck(hip.hipStreamBeginCapture(stream, 2), "hipStreamBeginCapture")
        for call in calls:
            sjk.check(call(), "captured call")
        dev._ck(hip.hipStreamEndCapture(stream, C.byref(self.graph)), "hipStreamEndCapture")
        dev._ck(hip.hipGraphInstantiate(C.byref(self.exec), self.graph, None, None, 0), "hipGraphInstantiate")

    def replay(self):
        self.dev._ck(self.hip.hipGraphLaunch(self.exec, self.stream), "hipGraphLaunch")
        self.dev._ck(self.hip.hipStreamSynchronize(self.stream), "hipStreamSynchronize")

    def close(self):
        self.hip.hipGraphExecDestroy(self.exec)
        self.hip.hipGraphDestroy(self.graph)


def descriptor(B, N, qpos0):
    d = np.zeros(16, np.int32)
    d[2], d[3], d[4] = B, N, qpos0
    return d
