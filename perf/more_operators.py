"""Long contexts and drafted tokens on this library's cache, as measurable cases.

A decode step over a long context need not read all of it, and several drafted tokens can be checked in one step. Around the
attention (sjk_hip_attend) an engine then runs:

* "select": for every query position and KV head the `top` sealed groups of 128 positions whose keys can reach the highest
            scores (sjk_hip_select_groups, _batch). The bound comes from the record's own scale tables: with codes c in [0, L],
            K[t, d] = (c Kscale[d] + Kzero[d]) Ktok[t], so q.K[t] is at most u max Ktok for
            u = sum_d q_d Kzero_d + max(q_d, 0) L Kscale_d (u min Ktok where u < 0). A group's score is the largest bound of the
            KV head's query heads; ties go to the lower group; the list comes out in ascending order, -1 behind its end;
* "groups": attention over the sink, the listed groups and the staged tail (sjk_hip_attend_groups, _batch);
* "tree":   attention of drafted nodes, staged behind the context, each over the whole context and the nodes that its mask
            names (sjk_hip_attend_tree, _batch);
* "accept": the staged rows of the accepted path moved to the positions behind the context, in every layer (sjk_hip_accept).

With `own` false an operator is computed in elementary torch operations on the cache's bytes, sums in 32 bits, the scores that
decide a selection in 64.
"""
import ctypes as C
import math
import os
import sys

import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

own = False

S, G = 128, 128                        # sink positions and tokens per sealed group (the format's defaults)
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
TYPE_IDS = {"f32": 0, "f16": 1, "bf16": 2}
# the 64 levels of the 6-bit staging rows (format data), upper half; the lower is its mirror image
LEVELS = (0x3B41871E, 0x3C11361E, 0x3C72452C, 0x3CA9D841, 0x3CDACEEE, 0x3D060ED8, 0x3D1EEAA7, 0x3D380779, 0x3D5170D6, 0x3D6B3355,
          0x3D82AE4B, 0x3D8FFEB0, 0x3D9D92B8, 0x3DAB73D2, 0x3DB9AD86, 0x3DC84BE4, 0x3DD75C8E, 0x3DE6F156, 0x3DF71E2A, 0x3E03FD0D,
          0x3E0CD142, 0x3E161E4F, 0x3E1FFAC2, 0x3E2A84BE, 0x3E35E397, 0x3E424E9C, 0x3E501472, 0x3E5FAD6D, 0x3E71DDE3, 0x3E8406E2,
          0x3E92A540, 0x3EA97050)


def listed():
    return [
        # one decode step of one sequence a few thousand positions long: the smallest selection, launch-bound
        {"name": "select_step", "kind": "select", "D": 256, "H": 4, "n_head": 16, "bk": 4, "bv": 4, "jobs": 1, "n_q": 1, "groups": 53,
         "top": 16, "paged": False},
        # a decode batch of 7 sequences of different lengths in one pool, 3-bit records
        {"name": "select_batch_7", "kind": "select", "D": 128, "H": 8, "n_head": 32, "bk": 3, "bv": 3, "jobs": 7, "n_q": 1,
         "groups": 301, "top": 64, "paged": True},
        # four query positions over a million
        {"name": "select_1m", "kind": "select", "D": 128, "H": 8, "n_head": 32, "bk": 4, "bv": 4, "jobs": 1, "n_q": 4, "groups": 8000,
         "top": 256, "paged": True},
        # one decode step at 100,000 positions, an eleventh of the sealed groups read, and the staged tail
        {"name": "groups_step", "kind": "groups", "D": 256, "H": 4, "n_head": 16, "bk": 4, "bv": 4, "jobs": 1, "n_q": 1, "groups": 736,
         "top": 64, "tail": 5664, "paged": False, "staging": 0, "out": "f32"},
        # a decode batch of 8 sequences in one pool, 3-bit records, short tails
        {"name": "groups_batch_8", "kind": "groups", "D": 128, "H": 8, "n_head": 32, "bk": 3, "bv": 3, "jobs": 8, "n_q": 1, "groups": 230,
         "top": 32, "tail": 517, "paged": True, "staging": 0, "out": "bf16"},
        # three query positions over 400,000
        {"name": "groups_400k", "kind": "groups", "D": 128, "H": 8, "n_head": 64, "bk": 4, "bv": 4, "jobs": 1, "n_q": 3, "groups": 3100,
         "top": 384, "tail": 4321, "paged": True, "staging": 0, "out": "f16"},
        # a chain of four drafted tokens behind a short chat
        {"name": "tree_chain_4", "kind": "tree", "D": 256, "H": 4, "n_head": 16, "bk": 4, "bv": 4, "jobs": 1, "nodes": 4, "n_q": 4,
         "groups": 0, "tail": 391, "paged": False, "staging": 0, "out": "f32"},
        # a tree of 21 nodes, the last level of 9 asking, fp16 staging and 3-bit records
        {"name": "tree_level_9_of_21", "kind": "tree", "D": 128, "H": 2, "n_head": 10, "bk": 4, "bv": 3, "jobs": 1, "nodes": 21, "n_q": 9,
         "groups": 87, "tail": 777, "paged": True, "staging": 1, "out": "f32"},
        # a decode batch of 4 sequences with trees of 12 nodes
        {"name": "tree_batch_4", "kind": "tree", "D": 128, "H": 8, "n_head": 32, "bk": 4, "bv": 4, "jobs": 4, "nodes": 12, "n_q": 12,
         "groups": 61, "tail": 900, "paged": True, "staging": 0, "out": "bf16"},
        # a tree of 64 nodes at 100,000 positions
        {"name": "tree_64_100k", "kind": "tree", "D": 256, "H": 4, "n_head": 16, "bk": 4, "bv": 4, "jobs": 1, "nodes": 64, "n_q": 64,
         "groups": 736, "tail": 5600, "paged": False, "staging": 0, "out": "bf16"},
        # a path of 5 of 16 nodes in 16 layers
        {"name": "accept_5", "kind": "accept", "D": 256, "H": 4, "layers": 16, "cap": 896, "base": 5000, "nodes": 16, "path": 5,
         "staging": 0},
        # a long path through a tree of 200 nodes in 64 layers, across the end of the ring
        {"name": "accept_90", "kind": "accept", "D": 128, "H": 8, "layers": 64, "cap": 1024, "base": 6200, "nodes": 200, "path": 90,
         "staging": 0},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["select", "groups", "groups", "tree", "tree", "tree", "accept"])
    D, H = rng.choice([128, 256]), rng.choice([1, 2, 3, 4, 8])
    if kind == "accept":
        nodes = _log_int(rng, 2, 200)
        return {"kind": kind, "D": D, "H": H, "layers": _log_int(rng, 1, 64 * 8 * 128 // (H * D)), "cap": rng.choice([384, 896, 1024]),
                "base": rng.choice([rng.randrange(0, S), rng.randrange(S, 100000)]), "nodes": nodes, "path": _log_int(rng, 1, min(nodes, 90)),
                "staging": rng.choice([0, 0, 1])}
    c = {"kind": kind, "D": D, "H": H, "n_head": H * rng.choice([1, 2, 4, 5, 8]), "bk": rng.choice([4, 4, 3, 2]), "bv": rng.choice([4, 4, 3, 2]),
         "jobs": rng.choice([1, 1, _log_int(rng, 2, 9)]), "paged": rng.random() < 0.6}
    if rng.random() < 0.5:
        c["bk"] = c["bv"] = 4
    if kind == "select":
        c["n_q"] = rng.choice([1, 1, 2, 3, 4])
        c["groups"] = _log_int(rng, 32, 8000 * 8 * 128 // (c["H"] * D * c["jobs"] * (2 if c["n_head"] > 4 * H else 1)))
        c["top"] = _log_int(rng, 4, min(512, c["groups"] // 2))
        return c
    c["staging"], c["out"] = rng.choice([0, 0, 1]), rng.choice(["f32", "f16", "bf16"])
    c["tail"] = _log_int(rng, 1, 4096 // c["jobs"])
    if kind == "groups":
        c["n_q"] = rng.choice([1, 1, 2, 3])
        c["groups"] = _log_int(rng, 1, 3100 * 8 * 128 // (H * D * c["jobs"]))
        c["top"] = _log_int(rng, 1, min(384 * 8 * 128 * 3 // (H * D * c["jobs"] * c["n_q"]), 2 * c["groups"]))
        c["tail"] = max(c["tail"], c["n_q"])
        return c
    c["nodes"] = _log_int(rng, 1, 100)
    c["n_q"] = rng.choice([c["nodes"], c["nodes"], rng.randrange(1, c["nodes"] + 1)])
    most = 64 * 16 * 736 * 256 // (c["n_q"] * c["n_head"] * D * c["jobs"])
    c["groups"] = rng.choice([0, _log_int(rng, 1, max(1, min(736, most)))])
    return c


# ---- the cache's bytes ----------------------------------------------------------------------------------------------

def _offsets(c):
    """record offsets: K codes, V codes, Kscale[D], Kzero[D], Ktok[G], Vch[D], Vscale[G], Vzero[G], bytes"""
    D, vp = c["D"], 16 * c["D"] * c["bk"]
    ks = vp + 16 * D * c["bv"]
    return {"v": vp, "ks": ks, "kz": ks + 2 * D, "kt": ks + 4 * D, "vc": ks + 4 * D + 256, "vs": ks + 6 * D + 256, "vz": ks + 6 * D + 512,
            "bytes": ks + 6 * D + 768}


def _stage_bytes(c):
    return 2 * c["D"] if c["staging"] else c["D"] // 128 * 98


def _half_bytes(x):
    return x.half().contiguous().view(torch.uint8)


def _records(c, g, n):
    """n x H records: codes near the middle of their range (4 bits), scales by channel and token, group means by channel"""
    D, H, o = c["D"], c["H"], _offsets(c)
    body = torch.randint(0, 256, (n, H, o["bytes"]), generator=g, device="cuda", dtype=torch.uint8)
    spans = [(a, b) for a, b, bits in ((0, o["v"], c["bk"]), (o["v"], o["ks"], c["bv"])) if bits == 4]
    if spans:                          # the sum of two nibbles of 0 .. 7
        a, b = spans[0][0], spans[-1][1]
        body[..., a:b] = ((body[..., a:b] >> 1) & 0x77) + (torch.randint(0, 256, (n, H, b - a), generator=g, device="cuda", dtype=torch.uint8) & 0x77)
    r = lambda *shape: torch.randn(shape, generator=g, device="cuda")  # noqa: E731
    tops = [float(2 ** c[k] - 1) for k in ("bk", "bv")]
    ks = 4.5 / tops[0] * torch.exp(0.3 * r(1, H, D) + 0.2 * r(n, H, D))
    vs = 4.5 / tops[1] * torch.exp(0.2 * r(n, H, G))
    kz = 0.5 * r(n, H, D) + 0.7 * r(1, H, D) - 0.47 * tops[0] * ks
    table = torch.cat([_half_bytes(ks), _half_bytes(kz), _half_bytes(torch.exp(0.1 * r(n, H, G))), _half_bytes(torch.exp(0.3 * r(n, H, D))),
                       _half_bytes(vs), _half_bytes(0.1 * r(n, H, G) - 0.47 * tops[1] * vs)], -1)
    body[..., o["ks"]:] = table
    return body


def _staged(c, g, n):
    """n slots x H x (K row | V row) of the staging type"""
    D, H = c["D"], c["H"]
    if c["staging"]:
        return _half_bytes(torch.randn((n, H, 2 * D), generator=g, device="cuda"))
    x = torch.randint(0, 256, (n, H, 2 * D // 128, 98), generator=g, device="cuda", dtype=torch.uint8)
    x[..., :2] = _half_bytes(7.0 * torch.exp(0.2 * torch.randn((n, H, 2 * D // 128, 1), generator=g, device="cuda")))
    return x.reshape(n, H, 2 * _stage_bytes(c))


def _cache(c, g, n_rows):
    """one sequence's cache: sink, sealed groups through a block table, a ring that holds the last n_rows positions"""
    D, H, n = c["D"], c["H"], c["groups"]
    s = {"body": _records(c, g, max(n, 1)), "groups": n, "B": S + G * n}
    s["blocks"] = (torch.randperm(max(n, 1), generator=g, device="cuda") if c["paged"] else torch.arange(max(n, 1), device="cuda")).int()
    if c["kind"] != "select":
        s["sink"] = torch.randn((S, H, 2, D), generator=g, device="cuda").half()
        cap = -(-max(n_rows, 16) // 128) * 128
        s["ring"], s["cap"] = _staged(c, g, cap), cap
    return s


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    return g


def _inputs(case, seed):
    """the inputs alone, the same for the operator and for its exact results"""
    c, g = case, _gen(seed)
    D, H = c["D"], c["H"]
    if c["kind"] == "accept":
        ring = torch.stack([_staged(c, g, c["cap"]) for _ in range(c["layers"])])
        sink = torch.randint(0, 256, (c["layers"], S, H, 4 * D), generator=g, device="cuda", dtype=torch.uint8)
        path = torch.randperm(c["nodes"], generator=g, device="cuda")[:c["path"]].sort().values.int()
        return {"ring": ring, "sink": sink, "path": path}
    seqs = []
    for j in range(c["jobs"]):
        cj = dict(c, groups=max(1, c["groups"] - (c["groups"] // 11) * j) if c["groups"] else 0)
        rows = c.get("tail", 0) + c.get("nodes", 0)
        s = _cache(cj, g, rows)
        # the context ends `tail` staged positions behind the sealed part; without one, partly or wholly inside the sink
        s["N"] = s["B"] + c.get("tail", 0) if s["groups"] else max(c.get("tail", 0) - 37 * j, 1)
        s["q"] = torch.randn((c["n_q"], c["n_head"], D), generator=g, device="cuda") * torch.exp(0.3 * torch.randn((1, c["n_head"], 1), generator=g, device="cuda"))
        if c["kind"] == "groups":
            k = min(c["top"], s["groups"])
            pick = torch.rand((c["n_q"], H, s["groups"]), generator=g, device="cuda").argsort(-1)[..., :k].sort(-1).values
            s["sel"] = torch.full((c["n_q"], H, c["top"]), -1, device="cuda", dtype=torch.int32)
            s["sel"][..., :k] = pick.int()
        if c["kind"] == "tree":
            t = c["nodes"]
            parent = (torch.arange(t, device="cuda") - 1 - (torch.rand(t, generator=g, device="cuda") ** 2 * min(t, 8)).long()).clamp(min=-1)
            step = torch.zeros((t, t + 1), device="cuda", dtype=torch.float64)
            step[torch.arange(t, device="cuda"), parent + 1] = 1
            walk = torch.eye(t, device="cuda", dtype=torch.float64) + step[:, 1:]
            seen = torch.linalg.matrix_power(walk, t) > 0
            seen[3::17] = False                                    # padding of a tree of fixed size: such a node sees the context only
            s["seen"] = seen[t - c["n_q"]:]
            bits = torch.zeros((c["n_q"], -(-t // 64) * 64), device="cuda", dtype=torch.int64)
            bits[:, :t] = s["seen"].long()
            s["words"] = (bits.view(c["n_q"], -1, 64) << torch.arange(64, device="cuda")).sum(-1)
        seqs.append(s)
    return {"seqs": seqs}


def prepare(case, seed):
    s, c = _inputs(case, seed), case
    s["case"] = c
    lv = torch.tensor(LEVELS, dtype=torch.int32, device="cuda").view(torch.float32)
    s["levels"] = torch.cat([-lv.flip(0), lv])
    if c["kind"] == "accept":
        i = torch.arange(c["path"], device="cuda")
        s["rows"] = tuple(_row_of(c, s, p) for p in (c["base"] + s["path"].long(), c["base"] + i))
    else:
        for q in s["seqs"]:
            if c["kind"] == "select":
                q["sel"] = torch.empty((c["n_q"], c["H"], c["top"]), dtype=torch.int32, device="cuda")
            else:
                q["out"] = torch.empty((c["n_q"], c["n_head"], c["D"]), dtype=TYPES[c["out"]], device="cuda")
    if own:
        s["call"] = _call(s)           # the argument structures and the workspace that a program keeps for its layer
    return s


def _row_of(c, s, pos):
    """whether positions lie in the sink, their rows there and their slots of the ring"""
    return pos < S, pos.clamp(max=S - 1), torch.remainder(pos - S, c["cap"])


# ---- the framework's calls ------------------------------------------------------------------------------------------

def _sjk():
    if os.path.join(ROOT, "sj-kvarn-codec_amd") not in sys.path:
        sys.path.insert(0, os.path.join(ROOT, "sj-kvarn-codec_amd"))
    import sjk
    return sjk


def _view(sjk, c, q, work):
    v = sjk.View()
    v.lay = sjk.layout(c["D"], G, c.get("bk", 4), c.get("bv", 4), 0)
    v.n_head_kv, v.staging, v.sink_type, v.S, v.cap = c["H"], c.get("staging", 0), 0, S, q.get("cap", 0)
    v.stage_bytes = _stage_bytes(dict(c, staging=c.get("staging", 0)))
    v.sink, v.ring = (q["sink"].data_ptr(), q["ring"].data_ptr()) if "ring" in q else (None, None)
    v.body = q["body"].data_ptr() if "body" in q else None
    v.blocks = q["blocks"].data_ptr() if c.get("paged") else None
    v.work, v.work_bytes = (work.data_ptr(), work.numel()) if work is not None else (None, 0)
    return v


def _call(s):
    c, sjk = s["case"], _sjk()
    lib, kind = sjk.load(), c["kind"]
    if kind == "accept":
        views = (sjk.View * c["layers"])(*[_view(sjk, c, {"sink": s["sink"][i], "ring": s["ring"][i], "cap": c["cap"]}, None) for i in range(c["layers"])])
        return lambda st: lib.sjk_hip_accept(views, c["layers"], c["base"], c["nodes"], s["path"].data_ptr(), c["path"], st)
    lay = sjk.layout(c["D"], G, c["bk"], c["bv"], 0)
    size = lib.sjk_hip_workspace_bytes(C.byref(lay), c["H"])
    s["work"] = [torch.empty(size, dtype=torch.uint8, device="cuda") for _ in s["seqs"]]
    scale, n, top = 1.0 / math.sqrt(c["D"]), len(s["seqs"]), c.get("top")
    if kind == "tree":
        jobs = (sjk.TreeJob * n)(*[sjk.TreeJob(_view(sjk, c, q, w), q["B"], q["N"], q["words"].data_ptr(), q["q"].data_ptr(), q["out"].data_ptr())
                                   for q, w in zip(s["seqs"], s["work"])])
        j, t = jobs[0], TYPE_IDS[c["out"]]
        if n == 1:
            v = C.pointer(j.v)
            return lambda st: lib.sjk_hip_attend_tree(v, j.B, j.base, c["nodes"], c["n_q"], c["n_head"], j.d_q, scale, j.d_seen, t, j.d_out, st)
        return lambda st: lib.sjk_hip_attend_tree_batch(jobs, n, c["nodes"], c["n_q"], c["n_head"], scale, t, st)
    jobs = (sjk.GroupsJob * n)(*[sjk.GroupsJob(_view(sjk, c, q, w), q["B"], q["N"], q["N"] - c["n_q"] if kind == "groups" else q["N"],
                                               q["q"].data_ptr(), q["sel"].data_ptr(), q["out"].data_ptr() if kind == "groups" else None)
                                 for q, w in zip(s["seqs"], s["work"])])
    j = jobs[0]
    v = C.pointer(j.v)
    if kind == "select":
        if n == 1:
            return lambda st: lib.sjk_hip_select_groups(v, j.B, j.N, j.qpos0, c["n_q"], c["n_head"], j.d_q, top, j.d_sel, st)
        return lambda st: lib.sjk_hip_select_groups_batch(jobs, n, c["n_q"], c["n_head"], top, st)
    t = TYPE_IDS[c["out"]]
    if n == 1:
        return lambda st: lib.sjk_hip_attend_groups(v, j.B, j.N, j.qpos0, c["n_q"], c["n_head"], j.d_q, scale, j.d_sel, top, t, j.d_out, st)
    return lambda st: lib.sjk_hip_attend_groups_batch(jobs, n, c["n_q"], c["n_head"], scale, top, t, st)


# ---- the plain form -------------------------------------------------------------------------------------------------

def _codes(p, D, bits, is_v):
    """codes [n, G, D] (int32) of payload bytes p [n, 16 D bits]: 4 bits in 16 x 16 tiles of fragment order, fewer token by token"""
    n = p.shape[0]
    if bits == 4:
        w = p.contiguous().view(torch.int32).view(n, 8, D // 16, 8, 4)          # token tile, channel tile, a % 8, (b / 2) % 4
        c = (w[..., None] >> torch.arange(0, 32, 4, device=p.device, dtype=torch.int32)) & 15
        c = c.view(n, 8, D // 16, 8, 4, 2, 2, 2)                               # ..., b % 2, b / 8, a / 8
        # a is the token on the K side, the channel on the V side
        return c.permute((0, 1, 6, 4, 5, 2, 7, 3) if is_v else (0, 1, 7, 3, 2, 6, 4, 5)).reshape(n, G, D)
    if bits == 2:
        return ((p.int()[..., None] >> torch.arange(0, 8, 2, device=p.device, dtype=torch.int32)) & 3).reshape(n, G, D)
    b = p.view(n, -1, 3).int()
    x = b[..., 0] | (b[..., 1] << 8) | (b[..., 2] << 16)
    return ((x[..., None] >> torch.arange(0, 24, 3, device=p.device, dtype=torch.int32)) & 7).reshape(n, G, D)


def _halves(r, at, n):
    return r[:, at:at + 2 * n].contiguous().view(torch.float16).float()


def _channel(c, side, device):
    """where a channel's scale lies in its table"""
    d = torch.arange(c["D"], device=device)
    if c["b" + side] != 4:
        return d
    if side == "v":
        return (d & 7) * (c["D"] // 8) + (d >> 4) * 2 + ((d >> 3) & 1)
    j = (d & 15) >> 1
    return (j & 3) * (c["D"] // 4) + (d >> 4) * 4 + (j >> 2) * 2 + (d & 1)


def _decode(c, r):
    """K and V [n, G, D] in 32 bits of records r [n, bytes]"""
    D, o = c["D"], _offsets(c)
    ik, iv = _channel(c, "k", r.device), _channel(c, "v", r.device)
    k = _codes(r[:, :o["v"]], D, c["bk"], False).float()
    k = (k * _halves(r, o["ks"], D)[:, None, ik] + _halves(r, o["kz"], D)[:, None, ik]) * _halves(r, o["kt"], G)[:, :, None]
    v = _codes(r[:, o["v"]:o["ks"]], D, c["bv"], True).float()
    v = (v * _halves(r, o["vs"], G)[:, :, None] + _halves(r, o["vz"], G)[:, :, None]) * _halves(r, o["vc"], D)[:, None, iv]
    return k, v


def _unstage(c, levels, x):
    """K and V [H, n, D] in 32 bits of staged rows x [n, H, 2 rows]"""
    n, H, D = x.shape[0], c["H"], c["D"]
    if c["staging"]:
        y = x.contiguous().view(torch.float16).float().view(n, H, 2, D)
    else:
        b = x.reshape(n, H, 2 * D // 128, 98)
        lo = ((b[..., 2:66, None] >> torch.tensor([0, 4], device=x.device, dtype=torch.uint8)) & 15).flatten(3)
        hi = ((b[..., 66:98, None] >> torch.tensor([0, 2, 4, 6], device=x.device, dtype=torch.uint8)) & 3).flatten(3)
        y = levels[(lo | (hi << 4)).int()] * b[..., :2].contiguous().view(torch.float16).float()
        y = y.view(n, H, 2, D)
    return y[:, :, 0].transpose(0, 1), y[:, :, 1].transpose(0, 1)


def _rows(c, s, levels, end):
    """K and V [H, n, D] of the sink's and the tail's positions before `end`, and the positions"""
    k, v = (s["sink"][:min(end, S), :, i].float().transpose(0, 1) for i in (0, 1))
    pos = torch.arange(s["B"], max(end, s["B"]), device=k.device)
    tk, tv = _unstage(c, levels, s["ring"][torch.remainder(pos - S, s["cap"])])
    return torch.cat([k, tk], 1), torch.cat([v, tv], 1), torch.cat([torch.arange(min(end, S), device=k.device), pos])


def _attention(q, k, v, seen, scale):
    """rows q [..., R, D] over k, v [..., M, D]; seen (broadcast to [..., R, M]) or None; a row that sees nothing gives zeros"""
    x = (q @ k.transpose(-1, -2)) * scale
    if seen is not None:
        x = x.masked_fill(~seen, -math.inf)
    m = x.amax(-1, keepdim=True)
    p = torch.exp(x - torch.where(m == -math.inf, 0.0, m))
    t = p.sum(-1, keepdim=True)
    return (p @ v) / torch.where(t == 0, 1.0, t)


def _by_kv_head(c, x):
    """[n_q, n_head, D] -> [H, n_q * heads of a KV head, D]"""
    n = x.shape[0]
    return x.view(n, c["H"], -1, c["D"]).transpose(0, 1).reshape(c["H"], -1, c["D"])


def _by_head(c, x):
    n = c["n_q"]
    return x.view(c["H"], n, -1, c["D"]).transpose(0, 1).reshape(n, c["n_head"], c["D"])


def _scores(c, s):
    """the bound of every group [n_q, H, groups], in 64 bits"""
    o, D, H, n = _offsets(c), c["D"], c["H"], s["groups"]
    table = s["body"][s["blocks"][:n].long(), :, o["ks"]:o["vc"]].contiguous().view(torch.float16).double()
    ik = _channel(c, "k", table.device)
    ks, kz, kt = table[..., :D][..., ik], table[..., D:2 * D][..., ik], table[..., 2 * D:]
    q = s["q"].view(c["n_q"], H, -1, D).double().permute(1, 0, 2, 3).reshape(H, -1, D)
    u = q @ kz.permute(1, 2, 0) + (q.clamp(min=0) * float(2 ** c["bk"] - 1)) @ ks.permute(1, 2, 0)
    u = torch.where(u >= 0, u * kt.amax(-1).t()[:, None], u * kt.amin(-1).t()[:, None])
    return u.view(H, c["n_q"], -1, n).amax(2).transpose(0, 1)


def _plain_select(c, s):
    k = min(c["top"], s["groups"])
    best = torch.sort(_scores(c, s), dim=-1, descending=True, stable=True).indices[..., :k].sort(-1).values
    s["sel"].fill_(-1)
    s["sel"][..., :k] = best.int()
    return s["sel"]


def _plain_groups(c, s, levels):
    D, H, n_q = c["D"], c["H"], c["n_q"]
    k, v, pos = _rows(c, s, levels, s["N"])
    live = s["sel"] >= 0
    blk = s["blocks"][s["sel"].clamp(min=0).long()].long()
    r = s["body"][blk, torch.arange(H, device=blk.device)[None, :, None]]
    rk, rv = (x.view(n_q, H, -1, D) for x in _decode(c, r.reshape(-1, r.shape[-1])))
    seen = torch.cat([live[..., None].expand(-1, -1, -1, G).reshape(n_q, H, 1, -1),
                      (pos[None, :] <= (s["N"] - n_q + torch.arange(n_q, device=pos.device))[:, None])[:, None, None].expand(-1, H, -1, -1)], -1)
    x = _attention(s["q"].view(n_q, H, -1, D), torch.cat([rk, k.expand(n_q, -1, -1, -1)], 2), torch.cat([rv, v.expand(n_q, -1, -1, -1)], 2),
                   seen, 1.0 / math.sqrt(D))
    return s["out"].copy_(x.reshape(n_q, c["n_head"], D))


def _plain_tree(c, s, levels):
    D, H, n_q = c["D"], c["H"], c["n_q"]
    k, v, pos = _rows(c, s, levels, s["N"] + c["nodes"])
    if s["groups"]:
        r = s["body"][s["blocks"][:s["groups"]].long()].transpose(0, 1)
        rk, rv = (x.view(H, -1, D) for x in _decode(c, r.reshape(-1, r.shape[-1])))
        k, v = torch.cat([rk, k], 1), torch.cat([rv, v], 1)
    seen = torch.ones((n_q, k.shape[1]), dtype=torch.bool, device=k.device)
    seen[:, -c["nodes"]:] = s["seen"]
    x = _attention(_by_kv_head(c, s["q"]), k, v, seen.repeat_interleave(c["n_head"] // H, 0), 1.0 / math.sqrt(D))
    return s["out"].copy_(_by_head(c, x))


def _plain_accept(c, s):
    (a, sa, ra), (b, sb, rb) = s["rows"]
    if c["base"] >= S:
        s["ring"][:, rb] = s["ring"][:, ra]
    else:                                # nodes in the sink, the ring or both: sink rows are fp16, ring rows the staging type
        _across(c, s, a, sa, ra, b, sb, rb)


def _across(c, s, a, sa, ra, b, sb, rb):
    """a move whose source is staged in the ring and whose destination lies in the sink takes the row's values to fp16"""
    sink, ring = s["sink"][:, sa], s["ring"][:, ra]
    lv, L, n = s["levels"], c["layers"], len(sa)
    k, v = _unstage(c, lv, ring.reshape(L * n, c["H"], -1))
    y = torch.stack([k.transpose(0, 1), v.transpose(0, 1)], 2).half().view(torch.uint8).view(L, n, c["H"], 4 * c["D"])
    x = torch.where(a[None, :, None, None], sink, y)
    s["sink"][:, sb[b]] = x[:, b]
    s["ring"][:, rb[~b]] = ring[:, ~b]


def run(state):
    c = state["case"]
    if own:
        rc = state["call"](torch.cuda.current_stream().cuda_stream)
        if rc:
            _sjk().check(rc, c["kind"])
    elif c["kind"] == "accept":
        _plain_accept(c, state)
    elif c["kind"] == "select":
        return [_plain_select(c, s) for s in state["seqs"]]
    else:
        f = _plain_groups if c["kind"] == "groups" else _plain_tree
        return [f(c, s, state["levels"]) for s in state["seqs"]]
    if c["kind"] == "accept":
        return state["sink"], state["ring"]
    return [s["sel" if c["kind"] == "select" else "out"] for s in state["seqs"]]


def work(case):
    c = case
    D, H = c["D"], c["H"]
    row = 2 * _stage_bytes(dict(c, staging=c.get("staging", 0)))
    if c["kind"] == "accept":
        return {"bytes": 2 * c["layers"] * H * c["path"] * row, "flops": 0}
    n = [max(1, c["groups"] - (c["groups"] // 11) * j) if c["groups"] else 0 for j in range(c["jobs"])]
    heads, n_q, q = c["n_head"], c["n_q"], c["n_q"] * c["n_head"] * D
    if c["kind"] == "select":
        return {"bytes": sum(n) * H * (4 * D + 2 * G) + c["jobs"] * (4 * q + 4 * n_q * H * c["top"]), "flops": 4 * sum(n) * q}
    rec, size = _offsets(c)["bytes"], TYPES[c["out"]].itemsize
    if c["kind"] == "groups":
        read = [n_q * min(c["top"], k) for k in n]
        tail, dense = [c["tail"]] * c["jobs"], [S + c["tail"]] * c["jobs"]
        flops = sum(4 * heads * D * (k * G + n_q * d) for k, d in zip(read, dense))
        recs = sum(min(r, k) for r, k in zip(read, n))              # a group that several positions list is read once at least
        return {"bytes": recs * H * rec + H * (c["jobs"] * S * 4 * D + sum(tail) * row) + c["jobs"] * q * (4 + size) + 4 * H * c["jobs"] * n_q * c["top"],
                "flops": flops}
    end = [c["tail"] + c["nodes"] + (S + G * k if k else -37 * j) for j, k in enumerate(n)]
    end = [max(e, c["nodes"] + 1) for e in end]
    tail = [max(0, e - S - G * k) for e, k in zip(end, n)]
    return {"bytes": sum(n) * H * rec + H * (sum(min(e, S) for e in end) * 4 * D + sum(tail) * row) + c["jobs"] * (q * (4 + size) + 8 * n_q * -(-c["nodes"] // 64)),
            "flops": 4 * q * sum(end)}


# ---- the same results in 64 bits ------------------------------------------------------------------------------------

def _exact_code(c, r, side):
    """codes [n, G, D] of records r [n, bytes], each by the place of its bits"""
    D, bits, v = c["D"], c["b" + side], side == "v"
    at = _offsets(c)["v"] if v else 0
    t, d = torch.meshgrid(torch.arange(G, device=r.device), torch.arange(D, device=r.device), indexing="ij")
    if bits == 4:
        a, b = (d % 16, t % 16) if v else (t % 16, d % 16)
        word = ((t // 16) * (D // 16) + d // 16) * 32 + 4 * (a % 8) + (b // 2) % 4
        bit = 32 * word + 4 * (a // 8 + 2 * (b // 8) + 4 * (b % 2))
    else:
        bit = (t * D + d) * bits
    lo, hi = r[:, at + bit // 8].long(), r[:, at + bit // 8 + 1].long()     # the scales follow the codes: the next byte is there
    return ((lo + 256 * hi) // 2 ** (bit % 8)) % 2 ** bits


def _exact_table(c, r, at, side=None):
    n = c["D"] if side else G
    h = r[:, at:at + 2 * n].reshape(-1, n, 2).long()
    h = (h[..., 0] + 256 * h[..., 1]).to(torch.int16).view(torch.float16).double()
    if side is None or c["b" + side] != 4:
        return h
    d = torch.arange(n, device=r.device)
    if side == "v":
        i = (d % 8) * (n // 8) + 2 * (d // 16) + (d // 8) % 2
    else:
        i = ((d // 2) % 4) * (n // 4) + 4 * (d // 16) + 2 * ((d // 8) % 2) + d % 2
    return h[:, i]


def _exact_records(c, r):
    """K and V [n G, D]"""
    o = _offsets(c)
    t = lambda name, side=None: _exact_table(c, r, o[name], side)  # noqa: E731
    k = (_exact_code(c, r, "k") * t("ks", "k")[:, None] + t("kz", "k")[:, None]) * t("kt")[..., None]
    v = (_exact_code(c, r, "v") * t("vs")[..., None] + t("vz")[..., None]) * t("vc", "v")[:, None]
    return k.reshape(-1, c["D"]), v.reshape(-1, c["D"])


def _exact_row(c, x):
    """values [n, D] of staged rows [n, row bytes]"""
    if c["staging"]:
        return x.contiguous().view(torch.float16).double()
    lv = torch.tensor(LEVELS, dtype=torch.int32, device=x.device).view(torch.float32).double()
    lv = torch.cat([-lv.flip(0), lv])
    out = []
    for b in x.split(98, 1):
        j = torch.arange(128, device=x.device)
        code = (b[:, 2 + j // 2].long() // 16 ** (j % 2)) % 16 + 16 * ((b[:, 66 + j // 4].long() // 4 ** (j % 4)) % 4)
        out.append(lv[code] * b[:, :2].contiguous().view(torch.float16).double())
    return torch.cat(out, 1)


def exact(case, seed):
    c = case
    if c["kind"] in ("accept", "select"):
        return None                       # bytes and whole numbers
    D, H, per = c["D"], c["H"], c["n_head"] // c["H"]
    outs = []
    for s in _inputs(case, seed)["seqs"]:
        y = torch.empty((c["n_q"], c["n_head"], D), dtype=torch.float64, device="cuda")
        end = s["N"] + c.get("nodes", 0)
        slots = torch.remainder(torch.arange(s["B"], max(end, s["B"]), device="cuda") - S, s["cap"])
        first = min(end, S)
        for h in range(H):
            ring = s["ring"][slots, h]
            rows = [torch.cat([s["sink"][:first, h, i].double(), _exact_row(c, ring[:, i * _stage_bytes(c):(i + 1) * _stage_bytes(c)])]) for i in (0, 1)]
            n = rows[0].shape[0]
            every = _exact_records(c, s["body"][s["blocks"][:s["groups"]].long(), h]) if c["kind"] == "tree" and s["groups"] else None
            for i in range(c["n_q"]):
                k, v = rows
                if c["kind"] == "tree":
                    keep = torch.ones(n, dtype=torch.bool, device="cuda")
                    keep[n - c["nodes"]:] = s["seen"][i]
                    k, v = k[keep], v[keep]
                else:
                    n_see = n - (c["n_q"] - 1 - i)
                    k, v = k[:n_see], v[:n_see]
                    ids = s["sel"][i, h]
                    every = _exact_records(c, s["body"][s["blocks"][ids[ids >= 0].long()].long(), h])
                q = s["q"][i, h * per:(h + 1) * per].double() / math.sqrt(D)
                x = [q @ k.t()] + ([q @ every[0].t()] if every is not None else [])
                m = torch.cat(x, 1).amax(1, keepdim=True)
                p = [(z - m).exp() for z in x]
                o = p[0] @ v + (p[1] @ every[1] if every is not None else 0.0)
                y[i, h * per:(h + 1) * per] = o / sum(z.sum(1, keepdim=True) for z in p)
        outs.append(y)
    return outs
