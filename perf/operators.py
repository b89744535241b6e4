"""The steps of an engine on either side of this library's cache, as measurable cases.

Between a layer's projections and its attention, and between one sequence and another, an engine runs:

* "rope":   rotary positions of query and key heads (sjk_hip_head_rows without norm weights): the rows of a fused
            projection output turned by their positions, halves or pairs, the whole head or its first n_rot channels,
            plain frequencies or frequencies scaled for long contexts;
* "heads":  the norm of every query and key head, the same turn, and the rotation into the cache's basis, in one pass
            (sjk_hip_head_rows);
* "append": the same for the queries, and the keys and values straight into the cache (sjk_hip_store_qkv, _batch):
            norm, turn, rotation and staging of a projection's rows in one launch;
* "fork":   a second sequence that goes on from the first one's positions (sjk_hip_fork): sink and staged rows of every
            layer copied, the sealed records shared through the block table;
* "blocks": record blocks of a paged pool moved in every layer (sjk_hip_copy_blocks), as compacting a pool does.

With `own` false an operator is computed in elementary torch operations, angles in 64 bits and sums in 32. The staged
rows of "append" are fp16 (SJKVARN_STAGING_F16): the 6-bit codes of the other staging type turn at borders, where the last
bit of a sum decides.
"""
import ctypes as C
import math
import os
import sys

import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, os.path.join(ROOT, "sj-kvarn-codec_amd"))
import sjk  # noqa: E402

own = False

S, G = 128, 128                        # sink positions and tokens per sealed group (the format's defaults)
EPS = 1e-6
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
TYPE_IDS = {"f32": 0, "f16": 1, "bf16": 2}
# frequency scalings: (kind, base, factor, original context, low, high)
SCALINGS = {"plain": (0, 1e4, 1.0, 0, 0, 0), "far": (0, 1e6, 1.0, 0, 0, 0), "linear": (1, 1e4, 4.0, 0, 0, 0),
            "ntk": (2, 1e4, 8.0, 0, 0, 0), "ramp": (3, 1e4, 16.0, 4096, 1, 32), "bands": (4, 5e5, 8.0, 8192, 1, 4)}
MOST_VALUES = 8192 * 40 * 128          # of a drawn case's rows: those of the largest listed ones
MOST_BYTES = 16 * 256 * 4 * 35072      # of a drawn case's pages


def listed():
    return [
        # one decode step of one layer, one token: the smallest call, launch-bound
        {"name": "rope_step", "kind": "rope", "D": 256, "n_head": 16, "H": 4, "n_pos": 1, "type": "f32", "out": "f32",
         "layout": "halves", "n_rot": 256, "scaling": "plain", "pos0": 5000, "ragged": False, "rotate": False},
        # a decode batch of 37 sequences at positions of their own, a quarter of the head turned
        {"name": "rope_batch_ragged", "kind": "rope", "D": 256, "n_head": 16, "H": 2, "n_pos": 37, "type": "f16", "out": "f16",
         "layout": "pairs", "n_rot": 64, "scaling": "linear", "pos0": 0, "ragged": True, "rotate": False},
        # the rows of an 8,192-position prompt of a head-dimension-128 model, frequencies scaled by wavelength
        {"name": "rope_8192", "kind": "rope", "D": 128, "n_head": 32, "H": 8, "n_pos": 8192, "type": "bf16", "out": "bf16",
         "layout": "halves", "n_rot": 128, "scaling": "bands", "pos0": 100000, "ragged": False, "rotate": False},
        # one decode step of 8 sequences: norms, turn and basis rotation of 40 heads each, queries as the attention takes them
        {"name": "heads_step_8", "kind": "heads", "D": 128, "n_head": 32, "H": 8, "n_pos": 8, "type": "bf16", "out": "f32",
         "layout": "halves", "n_rot": 128, "scaling": "far", "pos0": 0, "ragged": True, "rotate": True},
        # a ragged ubatch of heads of an odd width, no basis rotation
        {"name": "heads_1237_d80", "kind": "heads", "D": 80, "n_head": 32, "H": 32, "n_pos": 1237, "type": "f16", "out": "f16",
         "layout": "halves", "n_rot": 80, "scaling": "ramp", "pos0": 30000, "ragged": False, "rotate": False},
        # one decode step of 8 sequences straight into their caches
        {"name": "append_step_8", "kind": "append", "D": 256, "n_head": 16, "H": 4, "n_pos": 1, "jobs": 8, "type": "bf16",
         "norm": True, "layout": "halves", "n_rot": 256, "scaling": "plain", "pos0": 700, "ragged": False},
        # a prefill ubatch, no norms, interleaved pairs, from the sink into the ring
        {"name": "append_512", "kind": "append", "D": 128, "n_head": 32, "H": 8, "n_pos": 512, "jobs": 1, "type": "f16",
         "norm": False, "layout": "pairs", "n_rot": 128, "scaling": "plain", "pos0": 0, "ragged": False},
        # the largest ubatch: 4,096 positions of a head-dimension-128 model
        {"name": "append_4096", "kind": "append", "D": 128, "n_head": 32, "H": 8, "n_pos": 4096, "jobs": 1, "type": "bf16",
         "norm": True, "layout": "halves", "n_rot": 128, "scaling": "far", "pos0": 60000, "ragged": False},
        # a chat's first turns forked: everything still in sink and ring
        {"name": "fork_short", "kind": "fork", "D": 256, "H": 4, "layers": 16, "N": 391, "B": 128, "staging": 0, "cap": 9344},
        # a full adaptive tail of 16 layers, the ring wrapped
        {"name": "fork_tail", "kind": "fork", "D": 256, "H": 4, "layers": 16, "N": 40123, "B": 32128, "staging": 0, "cap": 9344},
        # a few blocks of a 16-layer pool
        {"name": "blocks_5", "kind": "blocks", "D": 256, "H": 4, "layers": 16, "n": 5, "n_blocks": 64, "bits": 3},
        # a pool of 16 layers compacted: a quarter of its blocks moved
        {"name": "blocks_256", "kind": "blocks", "D": 256, "H": 4, "layers": 16, "n": 256, "n_blocks": 1024, "bits": 4},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["rope", "rope", "heads", "heads", "append", "append", "fork", "blocks"])
    if kind in ("fork", "blocks"):
        D, H, layers = rng.choice([128, 256]), rng.choice([1, 2, 4, 8]), _log_int(rng, 1, 32)
        if kind == "fork":
            cap, staging = rng.choice([896, 4480, 9344]), rng.choice([0, 0, 1])
            row = H * 2 * _stage_bytes(staging, D) * layers
            tail = _log_int(rng, 1, max(2, min(cap, MOST_BYTES // row)))
            B = S + G * rng.choice([0, 0, _log_int(rng, 1, 700)])
            N = rng.randrange(1, S + 1) if B == S and rng.random() < 0.2 else B + tail
            return {"kind": kind, "D": D, "H": H, "layers": layers, "N": N, "B": B, "staging": staging, "cap": cap}
        bits = rng.choice([2, 3, 4])
        most = max(2, MOST_BYTES // (4 * layers * H * D * 137))
        n = _log_int(rng, 1, min(256, most))
        return {"kind": kind, "D": D, "H": H, "layers": layers, "n": n, "n_blocks": 2 * n + rng.randrange(0, 2 * n + 1), "bits": bits}
    H = rng.choice([1, 2, 4, 8])
    n_head = H * rng.choice([1, 2, 4, 5, 8])
    c = {"kind": kind, "D": rng.choice([128, 256]), "n_head": n_head, "H": H, "type": rng.choice(["f32", "f16", "bf16", "bf16"]),
         "layout": rng.choice(["halves", "halves", "pairs"]), "scaling": rng.choice(sorted(SCALINGS)),
         "pos0": rng.choice([0, rng.randrange(1, 5000), rng.randrange(5000, 1000000)]), "ragged": rng.random() < 0.3}
    if kind == "append":
        c["jobs"] = rng.choice([1, 1, _log_int(rng, 2, 16)])
        c["norm"] = rng.random() < 0.6
    else:
        c["rotate"] = kind == "heads" and rng.random() < 0.5
        if not c["rotate"]:
            c["D"] = rng.choice([64, 72, 80, 96, 128, 128, 192, 256, 256, 512])
        c["out"] = rng.choice([c["type"], "f32"])
    D = c["D"]
    most = min(8192, MOST_VALUES // ((n_head + (1 if kind != "append" else 2) * H) * D * c.get("jobs", 1)))
    c["n_pos"] = _log_int(rng, 1, min(most, 4096 if kind == "append" else most))
    c["n_rot"] = rng.choice([D, D, D // 2, 2 * rng.randrange(1, D // 2)])
    return c


def _stage_bytes(staging, D):
    return 2 * D if staging else D // 128 * 98


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    return g


# ---- what a program has in hand -------------------------------------------------------------------------------------

def _turns(case):
    """turns per position of every turned pair of channels (float64 [n_rot / 2]), and the magnitude that the scaling asks for"""
    kind, base, factor, n_orig, low, high = SCALINGS[case["scaling"]]
    n = case["n_rot"]
    i = torch.arange(n // 2, dtype=torch.float64, device="cuda")
    if kind == 2 and n > 2:
        base = base * factor ** (n / (n - 2))
    f = base ** (-2.0 * i / n)
    mscale = 1.0
    if kind == 1 or (kind == 2 and n == 2):
        f = f / factor
    if kind == 3:
        a, b = (n * math.log(n_orig / (r * 2 * math.pi)) / (2 * math.log(base)) for r in (high, low))
        a, b = max(math.floor(a), 0), min(math.ceil(b), n - 1)
        ramp = ((i - a) / max(b - a, 0.001)).clamp(0, 1)
        f = f / factor * ramp + f * (1 - ramp)
        mscale = 0.1 * math.log(factor) + 1
    if kind == 4:
        wave = 2 * math.pi / f
        smooth = ((n_orig / wave - low) / (high - low)).clamp(0, 1)
        f = f / factor * (1 - smooth) + f * smooth
    return f / (2 * math.pi), mscale


def _hadamard(D):
    """the rotation into the cache's basis as a [D, D] matrix (Sylvester order, over sqrt(D)); symmetric"""
    i = torch.arange(D, device="cuda")
    bits = i[:, None] & i[None, :]
    for s in (8, 4, 2, 1):
        bits = bits ^ (bits >> s)
    return (1.0 - 2.0 * (bits & 1)).float() / math.sqrt(D)


def _rows(case, g, n):
    """a fused projection output [n][n_head + 2 H][D]: heads of different sizes, a few outlier channels"""
    D, heads = case["D"], case["n_head"] + 2 * case["H"]
    x = torch.randn((n, heads, D), generator=g, device="cuda")
    x *= torch.exp(0.4 * torch.randn((1, heads, 1), generator=g, device="cuda"))
    x[:, :, 3::50] *= 6.0
    return x.to(DTYPES[case["type"]])


def _positions(case, g, n):
    if case["ragged"]:
        return torch.randint(0, 131072, (n,), generator=g, device="cuda", dtype=torch.int32)
    return torch.arange(case["pos0"], case["pos0"] + n, dtype=torch.int32, device="cuda")


def _weights(case, g):
    return [1.0 + 0.2 * torch.randn(case["D"], generator=g, device="cuda") for _ in range(2)]


def _layout(case):
    b = case["bits"]
    return sjk.layout(case["D"], G, b, b, 0 if b == 4 else 1)


def _inputs(case, seed):
    """the inputs alone, the same for the operator and for its exact results"""
    g, kind, D = _gen(seed), case["kind"], case["D"]
    if kind == "fork":
        H, L, cap = case["H"], case["layers"], case["cap"]
        sb = _stage_bytes(case["staging"], D)
        ring = torch.randint(-2 ** 31, 2 ** 31, (L, cap, H * 2 * sb // 4), generator=g, device="cuda", dtype=torch.int32)
        sink = torch.randint(-2 ** 31, 2 ** 31, (L, S, H * D), generator=g, device="cuda", dtype=torch.int32)
        return {"ring": ring, "sink": sink}
    if kind == "blocks":
        lay = _layout(case)
        nb = case["H"] * lay.bytes
        body = torch.randint(-2 ** 31, 2 ** 31, (case["layers"], case["n_blocks"], nb // 4), generator=g, device="cuda",
                             dtype=torch.int32)
        # live blocks from the pool's upper half into holes of its lower half
        half = case["n_blocks"] // 2
        src = half + torch.randperm(case["n_blocks"] - half, generator=g, device="cuda")[:case["n"]]
        dst = torch.randperm(half, generator=g, device="cuda")[:case["n"]].sort().values
        return {"body": body, "src": src, "dst": dst}
    turns, mscale = _turns(case)
    n = case["n_pos"]
    seqs = []
    for j in range(case.get("jobs", 1)):
        first = case["pos0"] + 37 * j
        x = _rows(case, g, n)
        pos = _positions(dict(case, pos0=first), g, n)
        seqs.append((x, pos, first))
    norm = case["norm"] if kind == "append" else kind == "heads"
    return {"seqs": seqs, "turns": turns, "mscale": mscale, "w": _weights(case, g) if norm else None}


def _cap(case):
    """ring capacity of an append case: a small adaptive tail and the case's own ubatch"""
    return int(sjk.load().sj_kvarn_ring_capacity(256, 512, G, case["n_pos"]))


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"], kind, D = case, case["kind"], case["D"]
    if kind == "fork":
        cap, B, N = case["cap"], case["B"], case["N"]
        s["to_ring"], s["to_sink"] = torch.zeros_like(s["ring"]), torch.zeros_like(s["sink"])
        a, n = (B - S) % cap, max(0, N - B)
        s["runs"] = ((a, min(cap, a + n)), (0, max(0, a + n - cap)))       # slots of the staged positions, wrapped once
    elif kind == "blocks":
        s["ids"] = [(C.c_uint32 * case["n"])(*s[k].tolist()) for k in ("src", "dst")]
        s["long"] = s["body"].view(torch.int64) if s["body"].shape[2] % 2 == 0 else s["body"]
    else:
        if kind == "append" or case["rotate"]:
            s["R"] = _hadamard(D)
        n, H = case["n_pos"], case["H"]
        s["outs"] = []
        for x, pos, first in s["seqs"]:
            if kind == "append":
                cap = _cap(case)
                p = torch.arange(first, first + n, device="cuda")
                s["outs"].append({"q": torch.empty((n, case["n_head"], D), device="cuda"),
                                  "sink": torch.zeros((S, H, 2, D), dtype=torch.float16, device="cuda"),
                                  "ring": torch.zeros((cap, H, 2, D), dtype=torch.float16, device="cuda"),
                                  "n_sink": max(0, min(n, S - first)), "slots": torch.remainder(p[p >= S] - S, cap)})
            else:
                o = DTYPES[case["out"]]
                s["outs"].append({"q": torch.empty((n, case["n_head"], D), dtype=o, device="cuda"),
                                  "k": torch.empty((n, H, D), dtype=o, device="cuda")})
    if own:
        s["call"] = _call(s)              # the argument structures that a program keeps for its layer
    return s


# ---- the framework's calls ------------------------------------------------------------------------------------------

def _view(case, lay, cap, sink, ring, staging):
    v = sjk.View()
    v.lay, v.n_head_kv, v.staging, v.sink_type, v.S, v.cap = lay, case["H"], staging, 0, S, cap
    v.stage_bytes = _stage_bytes(staging, case["D"])
    v.sink, v.ring, v.body, v.blocks, v.work, v.work_bytes = sink.data_ptr(), ring.data_ptr(), ring.data_ptr(), None, None, 0
    return v


def _rope(s):
    case = s["case"]
    r = sjk.Rope()
    r.layout, r.n_rot, r.inverse = (1 if case["layout"] == "pairs" else 0), case["n_rot"], 0
    r.mscale, r.d_turns = s["mscale"], s["turns"].data_ptr()
    return r


def _call(s):
    case, lib = s["case"], sjk.load()
    kind, D, H = case["kind"], case["D"], case.get("H")
    if kind == "fork":
        lay = sjk.layout(D, G, 4, 4, 0)
        views = []
        for sink, ring in ((s["to_sink"], s["to_ring"]), (s["sink"], s["ring"])):
            vs = (sjk.View * case["layers"])()
            for i in range(case["layers"]):
                vs[i] = _view(case, lay, case["cap"], sink[i], ring[i], case["staging"])
            views.append(vs)
        return lambda st: lib.sjk_hip_fork(views[0], views[1], case["layers"], case["B"], case["N"], st)
    if kind == "blocks":
        body, nb, layer = s["body"].data_ptr(), 4 * s["body"].shape[2], 4 * s["body"].shape[1] * s["body"].shape[2]
        src, dst = s["ids"]
        return lambda st: lib.sjk_hip_copy_blocks(body, layer, case["n_blocks"], body, layer, case["n_blocks"], case["layers"], nb,
                                                  src, dst, case["n"], st)
    heads, n, t = case["n_head"], case["n_pos"], TYPE_IDS[case["type"]]
    rope, w = _rope(s), s["w"]
    stride, size = (heads + 2 * H) * D, DTYPES[case["type"]].itemsize
    if kind == "append":
        m = sjk.Qkv()
        m.type, m.n_head, m.rotate_qk, m.rotate_v, m.eps, m.norm_head = t, heads, 1, 1, EPS, 0
        m.q_pos = m.k_pos = m.v_pos = stride
        m.q_head = m.k_head = m.v_head = D
        m.d_q_norm, m.d_k_norm = (w[0].data_ptr(), w[1].data_ptr()) if w else (None, None)
        m.rope = rope
        lay = sjk.layout(D, G, 4, 4, 0)
        jobs = (sjk.QkvJob * case["jobs"])()
        for j, ((x, pos, first), o) in enumerate(zip(s["seqs"], s["outs"])):
            jobs[j].v = _view(case, lay, o["ring"].shape[0], o["sink"], o["ring"], 1)
            jobs[j].pos0, jobs[j].d_pos = first, pos.data_ptr() if case["ragged"] else None
            jobs[j].d_q, jobs[j].d_k = x.data_ptr(), x.data_ptr() + heads * D * size
            jobs[j].d_v, jobs[j].d_q_out = x.data_ptr() + (heads + H) * D * size, o["q"].data_ptr()
        if case["jobs"] == 1:
            j, v = jobs[0], C.pointer(jobs[0].v)
            return lambda st: lib.sjk_hip_store_qkv(v, j.pos0, n, C.byref(m), j.d_pos, j.d_q, j.d_k, j.d_v, j.d_q_out, st)
        return lambda st: lib.sjk_hip_store_qkv_batch(jobs, len(jobs), n, C.byref(m), st)
    x, pos, first = s["seqs"][0]
    jobs = (sjk.HeadJob * 2)()
    for k, (at, n_heads, out) in enumerate(((0, heads, s["outs"][0]["q"]), (heads, H, s["outs"][0]["k"]))):
        j = jobs[k]
        j.d_x, j.d_out = x.data_ptr() + at * D * size, out.data_ptr()
        j.x_pos, j.x_head, j.out_pos, j.out_head = stride, D, n_heads * D, D
        j.x_type, j.out_type, j.n_heads, j.rope, j.rotate = t, TYPE_IDS[case["out"]], n_heads, 1, int(case["rotate"])
        j.d_norm, j.norm_head, j.eps = (w[k].data_ptr() if w else None), 0, EPS
    d_pos = pos.data_ptr() if case["ragged"] else None
    return lambda st: lib.sjk_hip_head_rows(jobs, 2, n, D, C.byref(rope), first, d_pos, st)


# ---- the plain form -------------------------------------------------------------------------------------------------

def _plain_head(x, w, cos, sin, layout, n_rot, R):
    """rows [n, heads, D] in 32 bits: norm with weights w, turn by cos / sin [n, 1, n_rot / 2], product with R"""
    x = x.float()
    if w is not None:
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * w
    if cos is not None:
        r = x[..., :n_rot]
        a, b = (r[..., 0::2], r[..., 1::2]) if layout == "pairs" else (r[..., :n_rot // 2], r[..., n_rot // 2:])
        a, b = a * cos - b * sin, a * sin + b * cos
        r = torch.stack([a, b], -1).flatten(-2) if layout == "pairs" else torch.cat([a, b], -1)
        x = torch.cat([r, x[..., n_rot:]], -1) if n_rot < x.shape[-1] else r
    return x if R is None else x @ R


def _plain(s):
    case, kind = s["case"], s["case"]["kind"]
    if kind == "fork":
        n = min(case["N"], S)
        s["to_sink"][:, :n] = s["sink"][:, :n]
        (a, b), (c, d) = s["runs"]
        s["to_ring"][:, a:b] = s["ring"][:, a:b]
        if d > c:
            s["to_ring"][:, c:d] = s["ring"][:, c:d]
        return
    if kind == "blocks":
        s["long"][:, s["dst"]] = s["long"][:, s["src"]]
        return
    heads, H, layout, n_rot, R = case["n_head"], case["H"], case["layout"], case["n_rot"], s.get("R")
    wq, wk = s["w"] if s["w"] is not None else (None, None)
    for (x, pos, first), o in zip(s["seqs"], s["outs"]):
        angle = pos.double()[:, None, None] * s["turns"] * (2 * math.pi)
        cos, sin = (angle.cos() * s["mscale"]).float(), (angle.sin() * s["mscale"]).float()
        q = _plain_head(x[:, :heads], wq, cos, sin, layout, n_rot, R)
        k = _plain_head(x[:, heads:heads + H], wk, cos, sin, layout, n_rot, R)
        o["q"].copy_(q)
        if kind != "append":
            o["k"].copy_(k)
            continue
        v = _plain_head(x[:, heads + H:], None, None, None, layout, n_rot, R)
        kv = torch.stack([k, v], 2).half()
        m = o["n_sink"]
        o["sink"][first:first + m] = kv[:m]
        o["ring"][o["slots"]] = kv[m:]


def run(state):
    if own:
        rc = state["call"](torch.cuda.current_stream().cuda_stream)
        if rc:
            sjk.check(rc, state["case"]["kind"])
    else:
        _plain(state)
    kind = state["case"]["kind"]
    if kind == "fork":
        return state["to_sink"], state["to_ring"]
    if kind == "blocks":
        return state["body"]
    if kind == "append":
        return [[o["q"], o["sink"], o["ring"]] for o in state["outs"]]
    return state["outs"][0]["q"], state["outs"][0]["k"]


def work(case):
    kind, D, H = case["kind"], case["D"], case["H"]
    if kind == "fork":
        n = case["layers"] * H * (min(case["N"], S) * 4 * D + max(0, case["N"] - case["B"]) * 2 * _stage_bytes(case["staging"], D))
        return {"bytes": 2 * n, "flops": 0}
    if kind == "blocks":
        return {"bytes": 2 * case["layers"] * case["n"] * H * _layout(case).bytes, "flops": 0}
    n, heads, size = case["n_pos"] * case.get("jobs", 1), case["n_head"], DTYPES[case["type"]].itemsize
    if kind == "append":
        return {"bytes": n * D * ((heads + 2 * H) * size + heads * 4 + 2 * H * 2),
                "flops": n * D * ((heads + H) * (4 * case["norm"] + 3) + (heads + 2 * H) * math.log2(D))}
    out = DTYPES[case["out"]].itemsize
    return {"bytes": n * D * (heads + H) * (size + out),
            "flops": n * D * (heads + H) * ((4 if kind == "heads" else 0) + 3 * case["n_rot"] / D + case["rotate"] * math.log2(D))}


# ---- the same results in 64 bits ------------------------------------------------------------------------------------

def _exact_head(x, w, unit, layout, n_rot, rotate):
    """rows [n, heads, D] in 64 bits: the turn as a product of complex numbers, the rotation by sums and differences"""
    x = x.double()
    D = x.shape[-1]
    if w is not None:
        x = x / torch.sqrt((x * x).sum(-1, keepdim=True) / D + EPS) * w.double()
    if unit is not None:
        i = torch.arange(n_rot // 2, device="cuda")
        a, b = (2 * i, 2 * i + 1) if layout == "pairs" else (i, i + n_rot // 2)
        z = torch.complex(x[..., a].contiguous(), x[..., b].contiguous()) * unit
        x = x.clone()
        x[..., a], x[..., b] = z.real, z.imag
    if rotate:
        h = 1
        while h < D:
            y = x.reshape(x.shape[:-1] + (D // (2 * h), 2, h))
            x = torch.stack([y[..., 0, :] + y[..., 1, :], y[..., 0, :] - y[..., 1, :]], -2).reshape(x.shape)
            h *= 2
        x = x / math.sqrt(D)
    return x


def exact(case, seed):
    if case["kind"] in ("fork", "blocks"):
        return None                       # bytes
    s = _inputs(case, seed)
    heads, H, n = case["n_head"], case["H"], case["n_pos"]
    append = case["kind"] == "append"
    rotate = append or case["rotate"]
    wq, wk = s["w"] if s["w"] is not None else (None, None)
    outs = []
    for x, pos, first in s["seqs"]:
        turn = torch.remainder(pos.double()[:, None] * s["turns"][None, :], 1.0)
        unit = torch.polar(torch.full_like(turn, s["mscale"]), 2 * math.pi * turn)[:, None, :]
        args = (unit, case["layout"], case["n_rot"], rotate)
        q, k = _exact_head(x[:, :heads], wq, *args), _exact_head(x[:, heads:heads + H], wk, *args)
        if not append:
            return q, k
        v = _exact_head(x[:, heads + H:], None, None, None, 0, True)
        cap = _cap(case)
        sink = torch.zeros((S, H, 2, case["D"]), dtype=torch.float64, device="cuda")
        ring = torch.zeros((cap, H, 2, case["D"]), dtype=torch.float64, device="cuda")
        m = max(0, min(n, S - first))
        sink[first:first + m, :, 0], sink[first:first + m, :, 1] = k[:m], v[:m]
        at = torch.remainder(torch.arange(first + m, first + n, device="cuda") - S, cap)
        ring[at, :, 0], ring[at, :, 1] = k[m:], v[m:]
        outs.append([q, sink, ring])
    return outs
