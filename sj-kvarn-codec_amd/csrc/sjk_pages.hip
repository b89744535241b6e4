// sjk_pages.hip - pages of a cache from one place to another: the sink and staged rows of a fork (sjk_hip_fork),
// record blocks of a pool (sjk_hip_copy_blocks), and the rows of accepted drafted tokens (sjk_hip_accept).
//
// Both are copies bound by HBM (6.0 TB/s read and written for 574 MB of blocks, where a large plain copy reaches 4.7-5.4).
// A workgroup takes one tile of one run, each thread TILE_U 16-byte loads in flight before its stores (two or eight of them: 3%
// slower and the same); the run and its place come from the kernel arguments, so a call needs no device table and no host wait.
// Runs are 4-byte aligned (a tq6_0 slot is 196 bytes a head), the accesses 16 bytes wide at that alignment.
#include <stdlib.h>

#include "sjk_dev.h"

namespace sjk {

typedef uint32_t word4_t __attribute__((ext_vector_type(4), aligned(4)));

constexpr int TILE_U = 4, TILE_WORDS = 256 * 4 * TILE_U;       // 16 KB

// words [tile * TILE_WORDS, + TILE_WORDS) of a run of n; STREAM: loads and stores that do not displace what the caches hold
template <bool STREAM> SJK_DEV void copy_tile(uint32_t * dst, const uint32_t * src, uint64_t n, uint64_t tile) {
    const uint64_t w0 = tile * TILE_WORDS + 4u * threadIdx.x;
    if ((tile + 1) * TILE_WORDS <= n) {
        word4_t v[TILE_U];
#pragma unroll
        for (int i = 0; i < TILE_U; ++i) {
            const word4_t * p = (const word4_t *) (src + w0 + i * 1024u);
            v[i] = STREAM ? __builtin_nontemporal_load(p) : *p;
        }
#pragma unroll
        for (int i = 0; i < TILE_U; ++i) {
            word4_t * p = (word4_t *) (dst + w0 + i * 1024u);
            if (STREAM) __builtin_nontemporal_store(v[i], p);
            else *p = v[i];
        }
        return;
    }
    for (uint64_t w = w0; w < n; w += 1024u) {
        if (w + 4 <= n) *(word4_t *) (dst + w) = *(const word4_t *) (src + w);
        else for (uint64_t k = w; k < n; ++k) dst[k] = src[k];
    }
}

// ---- fork: every layer has the same runs, relative to its sink and ring ----
constexpr int FORK_LAYERS = 64, FORK_RUNS = 4;                 // the sink; the staged range, cut where either ring wraps
struct ForkRun { uint64_t src, dst, words, tile0; };
struct ForkBatch {
    struct { const uint8_t * sink, * ring; uint8_t * to_sink, * to_ring; } layer[FORK_LAYERS];
    ForkRun run[FORK_RUNS];
    int n_runs;
};
static_assert(sizeof(ForkBatch) <= 4096, "the table travels in the kernel arguments");

template <bool STREAM> __global__ __launch_bounds__(256) void fork_kernel(const ForkBatch bt) {
    int r = 0;
    while (r + 1 < bt.n_runs && blockIdx.x >= bt.run[r + 1].tile0) ++r;
    const ForkRun & R = bt.run[r];
    const auto & L = bt.layer[blockIdx.y];
    copy_tile<STREAM>((uint32_t *) ((r ? L.to_ring : L.to_sink) + R.dst), (const uint32_t *) ((r ? L.ring : L.sink) + R.src), R.words,
              blockIdx.x - R.tile0);
}

// ---- blocks ----
constexpr int BLOCK_PAIRS = 448;
struct BlockBatch {
    uint32_t src[BLOCK_PAIRS], dst[BLOCK_PAIRS];
    uint8_t * to;
    const uint8_t * from;
    uint64_t to_layer, from_layer, block;
};
static_assert(sizeof(BlockBatch) <= 4096, "the table travels in the kernel arguments");

template <bool STREAM> __global__ __launch_bounds__(256) void copy_blocks_kernel(const BlockBatch bt) {
    const uint32_t p = blockIdx.y, il = blockIdx.z;
    copy_tile<STREAM>((uint32_t *) (bt.to + il * bt.to_layer + bt.dst[p] * bt.block),
              (const uint32_t *) (bt.from + il * bt.from_layer + bt.src[p] * bt.block), bt.block / 4, blockIdx.x);
}

// A copy that the caches cannot hold beside its source takes loads and stores that leave them alone. Forks of a tail of 16
// layers, plain / streamed, alone and with a reader of the copy behind: 50 MB 22.8 / 22.1 and 39.1 / 42.3 us, 100 MB 43.1 / 37.9
// and 79.1 / 73.9, 200 MB 77.7 / 70.0 and 126.6 / 115.8; 574 MB of blocks 224 / 191 alone.
static bool stream_past(uint64_t bytes) { return bytes > ((uint64_t) 64 << 20); }

static uint64_t tiles(uint64_t words) { return (words + TILE_WORDS - 1) / TILE_WORDS; }

// ---- accept: rows base + path[i] to positions base + i, in place ----
//
// path ascends, so path[i] >= i: a row is never written before those that are copied from it at lower positions have been
// read, if a workgroup reads ACC_ROWS rows of its columns, waits, writes them and goes on. A call moves little (5 rows of 16 layers
// of 4 KV heads of 256: 125 KB, 3.5 us on the device; 90 of 64 layers of 8 of 128: 9 MB, 7.7) and is bound by its launch and two
// round trips; a column is 16 bytes of one row of one layer.
constexpr int ACC_LAYERS = 160, ACC_COLS = 16, ACC_U = 8, ACC_ROWS = 256 / ACC_COLS * ACC_U, ACC_PATH = 512;
struct AcceptBatch {
    struct { uint8_t * sink, * ring; } layer[ACC_LAYERS];
    const int32_t * path;                        // device, or null: the list below
    const int32_t * desc;                        // base from the device descriptor, or null
    uint32_t base, S, cap, n_nodes, n_path, to;  // rows go to base + to + i
    uint32_t sink_row, ring_row;                 // bytes of a position's row
    int D, H, side;                              // (rows of two formats) channels, KV heads, staged bytes of K or V
    uint32_t list0;                              // the list's first node; its entries count from there
    uint16_t list[ACC_PATH];
};
constexpr int ACC_HELD = 1024;                   // path entries that a workgroup holds in LDS
static_assert(ACC_PATH <= ACC_HELD, "a list is held whole");
static_assert(sizeof(AcceptBatch) <= 4096, "the table travels in the kernel arguments");

// A workgroup's place in the call: its first position, that position's slot, and the path's first entries in LDS
struct AccPlace {
    const AcceptBatch & b;
    uint32_t base, slot0;
    const uint32_t * held;
    __device__ __forceinline__ uint32_t node(uint32_t i) const { return i < (uint32_t) ACC_HELD ? held[i] : (uint32_t) b.path[i]; }
    // slot of position base + k; k is less than the ring's slots
    __device__ __forceinline__ uint32_t slot(uint32_t k) const {
        const uint32_t s = base < b.S ? base + k - b.S : slot0 + k;
        return s < b.cap ? s : s - b.cap;
    }
};
// the call's first position; false: it moves nothing
SJK_DEV bool acc_base(const AcceptBatch & b, uint32_t & base) {
    base = b.base;
    if (!b.desc) return true;
    const int32_t q = b.desc[SJK_DESC_QPOS0];
    base = (uint32_t) q;
    return q >= 0;
}
// entries of the path up to the first that is no node above the one before it
SJK_DEV uint32_t acc_len(const AcceptBatch & b, uint32_t * held, uint32_t * s_len) {
    auto entry = [&](uint32_t i) { return b.path ? (uint32_t) b.path[i] : b.list0 + b.list[i]; };
    if (threadIdx.x == 0) *s_len = b.n_path;
    __syncthreads();
    uint32_t first = b.n_path;
    for (uint32_t i = threadIdx.x; i < b.n_path; i += blockDim.x) {
        const uint32_t e = entry(i);
        const int64_t x = (int32_t) e, before = i ? (int64_t) (int32_t) entry(i - 1) : -1;
        if (i < (uint32_t) ACC_HELD) held[i] = e;
        if ((x <= before || x >= (int64_t) b.n_nodes) && i < first) first = i;
    }
    if (first < b.n_path) atomicMin(s_len, first);
    __syncthreads();
    return *s_len;
}
// rows [from, to) of the path, n words of each, columns of this thread's workgroup: dst and src rows of i by row(i)
template <typename Src, typename Dst>
SJK_DEV void acc_move(uint32_t from, uint32_t to, uint32_t words, uint32_t col0, Src src, Dst dst) {
    const uint32_t w = 4u * (col0 + threadIdx.x % ACC_COLS), r = threadIdx.x / ACC_COLS;
    const bool in = w < words, whole = w + 4u <= words;
    for (uint32_t i0 = from; i0 < to; i0 += ACC_ROWS) {
        uint32_t v[ACC_U][4];
#pragma unroll
        for (int u = 0; u < ACC_U; ++u) {
            const uint32_t i = i0 + u * (256 / ACC_COLS) + r;
            if (i >= to || !in) continue;
            const uint32_t * p = (const uint32_t *) src(i) + w;
            if (whole) {
                const word4_t x = *(const word4_t *) p;
#pragma unroll
                for (int k = 0; k < 4; ++k) v[u][k] = x[k];
            } else {
#pragma unroll
                for (int k = 0; k < 4; ++k) v[u][k] = w + k < words ? p[k] : 0u;
            }
        }
        __syncthreads();                         // every row of this turn has been read
#pragma unroll
        for (int u = 0; u < ACC_U; ++u) {
            const uint32_t i = i0 + u * (256 / ACC_COLS) + r;
            if (i >= to || !in) continue;
            uint32_t * p = (uint32_t *) dst(i) + w;
            if (whole) {
                *(word4_t *) p = word4_t{v[u][0], v[u][1], v[u][2], v[u][3]};
            } else {
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    if (w + k < words) p[k] = v[u][k];
            }
        }
    }
}

// sink and ring rows of one format, or a path that lies in one of them: grid (columns, layers)
__global__ __launch_bounds__(256) void accept_kernel(const AcceptBatch b) {
    __shared__ uint32_t s_len, held[ACC_HELD];
    uint32_t base;
    if (!acc_base(b, base)) return;
    const uint32_t len = acc_len(b, held, &s_len);
    const int il = (int) blockIdx.y;
    const AccPlace P = {b, base, base < b.S ? 0u : (base - b.S) % b.cap, held};
    uint8_t * sink = b.layer[il].sink, * ring = b.layer[il].ring;
    auto row = [&](uint32_t k) { return base + k < b.S ? sink + (size_t) (base + k) * b.sink_row : ring + (size_t) P.slot(k) * b.ring_row; };
    acc_move(0, len, (base < b.S ? b.sink_row : b.ring_row) / 4u, blockIdx.x * ACC_COLS, [&](uint32_t i) { return row(P.node(i)); },
             [&](uint32_t i) { return row(b.to + i); });
}

// An fp16 sink in front of a ring of 6-bit rows, nodes on both sides of its end: grid (KV heads, layers). Sink rows first, then the
// ring's rows that go to the sink, as fp16 values of what the ring holds (centroid x norm, one rounding to fp32 and one to
// fp16), then the rest; a step reads what the one before it does not write.
__global__ __launch_bounds__(256) void accept_mixed_kernel(const AcceptBatch b) {
    __shared__ uint32_t s_len, s_ns, held[ACC_HELD];
    uint32_t base;
    if (!acc_base(b, base)) return;
    const uint32_t len = acc_len(b, held, &s_len);
    const int h = (int) blockIdx.x, il = (int) blockIdx.y;
    const AccPlace P = {b, base, base < b.S ? 0u : (base - b.S) % b.cap, held};
    const uint32_t S = b.S, first = base + b.to;
    if (threadIdx.x == 0) s_ns = 0;
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < len; i += 256)
        if (base + P.node(i) < S) atomicMax(&s_ns, i + 1u);            // nodes ascend: a prefix of the path
    __syncthreads();
    const uint32_t ns = s_ns, nd = first >= S ? 0u : S - first < len ? S - first : len;      // destinations in the sink
    const uint32_t sw = (uint32_t) b.D, rw = (uint32_t) b.side / 2u;       // words of a head's sink and ring rows (K | V)
    auto sink = [&](uint32_t k) { return b.layer[il].sink + (size_t) (base + k) * b.sink_row + (size_t) h * 4u * (size_t) b.D; };
    auto ring = [&](uint32_t k) { return b.layer[il].ring + (size_t) P.slot(k) * b.ring_row + (size_t) h * 2u * (size_t) b.side; };
    for (uint32_t c = 0; 4u * c < sw; c += ACC_COLS)
        acc_move(0, ns, sw, c, [&](uint32_t i) { return sink(P.node(i)); }, [&](uint32_t i) { return sink(b.to + i); });
    __syncthreads();
    const uint32_t nv = 2u * (uint32_t) b.D;
    for (uint32_t e = threadIdx.x; e < (nd > ns ? nd - ns : 0u) * nv; e += 256) {
        const uint32_t i = ns + e / nv, d = e % nv, side = d / (uint32_t) b.D, j = d % (uint32_t) b.D;
        const uint8_t * blk = ring(P.node(i)) + side * (uint32_t) b.side + (j >> 7) * SJKVARN_TQ6_BLOCK_BYTES;
        const uint32_t k = j & 127u;
        const int code = ((blk[2 + (k >> 1)] >> (4 * (k & 1))) & 15) | (((blk[66 + (k >> 2)] >> (2 * (k & 3))) & 3) << 4);
        ((uint16_t *) sink(b.to + i))[d] = f32_to_f16(xmul(tq6_cent(code), f16_to_f32((uint16_t) (blk[0] | (blk[1] << 8)))));
    }
    __syncthreads();
    const uint32_t from = nd > ns ? nd : ns;
    for (uint32_t c = 0; 4u * c < rw; c += ACC_COLS)
        acc_move(from, len, rw, c, [&](uint32_t i) { return ring(P.node(i)); }, [&](uint32_t i) { return ring(b.to + i); });
}

}  // namespace sjk

using namespace sjk;

extern "C" int sjk_hip_fork(const sjk_hip_view * dst, const sjk_hip_view * src, int n_layers, uint32_t B, uint32_t N, void * stream) {
    if (n_layers < 0 || (n_layers > 0 && (!dst || !src))) return SJKVARN_ERR_ARG;
    if (!n_layers) return 0;
    const sjk_hip_view & s0 = src[0], & d0 = dst[0];
    if (s0.n_head_kv <= 0 || s0.lay.D <= 0 || s0.lay.G <= 0 || s0.cap == 0 || d0.cap == 0) return SJKVARN_ERR_ARG;
    if ((s0.staging != SJKVARN_STAGING_TQ6_0 && s0.staging != SJKVARN_STAGING_F16) ||
        s0.stage_bytes != sj_kvarn_stage_row_bytes(s0.staging, s0.lay.D) || s0.stage_bytes == 0 ||
        (s0.sink_type != SJKVARN_SINK_F16 && s0.sink_type != SJKVARN_SINK_INHERIT))
        return SJKVARN_ERR_ARG;
    if (B < s0.S || (B - s0.S) % (uint32_t) s0.lay.G || (N < B && B > s0.S))
        return refuse("sjk_hip_fork: B below S, inside a group or past N");
    for (int il = 0; il < n_layers; ++il)
        for (const sjk_hip_view * v : {dst + il, src + il}) {
            const sjk_hip_view & w = v == src + il ? s0 : d0;
            if (!v->sink || !v->ring || (((uintptr_t) v->sink | (uintptr_t) v->ring) & 3u)) return SJKVARN_ERR_ARG;
            if (v->lay.D != s0.lay.D || v->lay.G != s0.lay.G || v->n_head_kv != s0.n_head_kv || v->staging != s0.staging ||
                v->sink_type != s0.sink_type || v->stage_bytes != s0.stage_bytes || v->S != s0.S || v->cap != w.cap)
                return refuse("sjk_hip_fork: the views differ in layout, heads, staging, sink or (on one side) capacity");
        }
    const uint64_t H = (uint64_t) s0.n_head_kv, entry = H * 2 * s0.stage_bytes;
    const uint64_t sink_entry = s0.sink_type == SJKVARN_SINK_F16 ? H * 4 * (uint64_t) s0.lay.D : entry;
    // each buffer of dst against every other buffer: none may be written twice, or written and read
    const uint64_t ss = s0.S * sink_entry, sr = s0.cap * entry, dr = d0.cap * entry;
    auto meet = [](const uint8_t * p, uint64_t np, const uint8_t * q, uint64_t nq) {
        return (uint64_t) ((uintptr_t) p - (uintptr_t) q) + np - 1 < np + nq - 1;      // -np < p - q < nq
    };
    for (int i = 0; i < n_layers; ++i) {
        const sjk_hip_view & d = dst[i];
        bool bad = meet(d.sink, ss, d.ring, dr);
        for (int k = 0; k < n_layers; ++k)
            bad |= meet(d.sink, ss, src[k].sink, ss) | meet(d.sink, ss, src[k].ring, sr) | meet(d.ring, dr, src[k].sink, ss) |
                   meet(d.ring, dr, src[k].ring, sr);
        for (int k = 0; k < i; ++k)
            bad |= meet(d.sink, ss, dst[k].sink, ss) | meet(d.sink, ss, dst[k].ring, dr) | meet(d.ring, dr, dst[k].sink, ss) |
                   meet(d.ring, dr, dst[k].ring, dr);
        if (bad) return refuse("sjk_hip_fork: a buffer of dst overlaps another of dst, or one of src");
    }
    const uint32_t n = N > B ? N - B : 0;
    if (n > s0.cap || n > d0.cap) {
        set_error("sjk_hip_fork: the staged positions do not fit the ring");
        return SJKVARN_ERR_CAPACITY;
    }
    ForkBatch bt;
    const uint64_t sink = (uint64_t) (N < s0.S ? N : s0.S) * sink_entry, bytes = sink + n * entry;     // of a layer
    uint64_t at = tiles(sink / 4);
    bt.run[0] = ForkRun{0, 0, sink / 4, 0};
    bt.n_runs = 1;
    for (uint32_t pos = B; pos < B + n;) {
        const uint32_t a = sj_kvarn_ring_slot(s0.S, s0.cap, pos), b = sj_kvarn_ring_slot(s0.S, d0.cap, pos);
        uint32_t k = B + n - pos;
        if (k > s0.cap - a) k = s0.cap - a;
        if (k > d0.cap - b) k = d0.cap - b;
        bt.run[bt.n_runs++] = ForkRun{a * entry, b * entry, k * entry / 4, at};
        at += tiles(k * entry / 4);
        pos += k;
    }
    if (!at) return 0;
    if (at > 0x7fffffffu) return refuse("sjk_hip_fork: too large");
    for (int i0 = 0; i0 < n_layers; i0 += FORK_LAYERS) {
        const int nl = n_layers - i0 < FORK_LAYERS ? n_layers - i0 : FORK_LAYERS;
        for (int k = 0; k < nl; ++k) {
            bt.layer[k].sink = src[i0 + k].sink; bt.layer[k].ring = src[i0 + k].ring;
            bt.layer[k].to_sink = dst[i0 + k].sink; bt.layer[k].to_ring = dst[i0 + k].ring;
        }
        hipLaunchKernelGGL(stream_past((uint64_t) n_layers * bytes) ? fork_kernel<true> : fork_kernel<false>,
                           dim3((unsigned) at, (unsigned) nl), dim3(256), 0, (hipStream_t) stream, bt);
        if (SJK_CHECK_LAUNCH()) return SJK_ERR_DEVICE;
    }
    return 0;
}

// a set of block ids of a slab
static bool mark(uint64_t * set, uint32_t id) {        // false: it was in the set
    const uint64_t b = 1ull << (id & 63u);
    const bool fresh = !(set[id >> 6] & b);
    set[id >> 6] |= b;
    return fresh;
}

extern "C" int sjk_hip_copy_blocks(uint8_t * d_dst, size_t dst_layer_bytes, uint32_t dst_blocks, const uint8_t * d_src,
                                   size_t src_layer_bytes, uint32_t src_blocks, int n_layers, size_t block_bytes,
                                   const uint32_t * src_ids, const uint32_t * dst_ids, uint32_t n, void * stream) {
    if (!d_dst || !d_src || n_layers < 0 || (n > 0 && (!src_ids || !dst_ids))) return SJKVARN_ERR_ARG;
    if (!n || !n_layers) return 0;
    if (block_bytes == 0 || ((uintptr_t) d_dst | (uintptr_t) d_src | dst_layer_bytes | src_layer_bytes | block_bytes) & 3u)
        return refuse("sjk_hip_copy_blocks: addresses and sizes in multiples of 4");
    if (n_layers > 65535 || (n_layers > 1 && (dst_layer_bytes / block_bytes < dst_blocks || src_layer_bytes / block_bytes < src_blocks)))
        return refuse("sjk_hip_copy_blocks: the slabs' layers overlap (or more than 65,535)");
    const bool same = d_dst == d_src && (n_layers == 1 || dst_layer_bytes == src_layer_bytes);
    const uintptr_t d0 = (uintptr_t) d_dst, d1 = d0 + (n_layers - 1) * dst_layer_bytes + dst_blocks * block_bytes;
    const uintptr_t s0 = (uintptr_t) d_src, s1 = s0 + (n_layers - 1) * src_layer_bytes + src_blocks * block_bytes;
    if (!same && d0 < s1 && s0 < d1) return refuse("sjk_hip_copy_blocks: the slabs overlap");
    const size_t words = ((size_t) dst_blocks + 63u) / 64u;
    uint64_t * set = (uint64_t *) calloc(words ? words : 1, 8);
    if (!set) return SJKVARN_ERR_NOMEM;
    bool ok = true;
    for (uint32_t i = 0; ok && i < n; ++i) ok = src_ids[i] < src_blocks && dst_ids[i] < dst_blocks && mark(set, dst_ids[i]);
    for (uint32_t i = 0; ok && same && i < n; ++i) ok = src_ids[i] >= dst_blocks || !(set[src_ids[i] >> 6] >> (src_ids[i] & 63u) & 1u);
    free(set);
    if (!ok) return refuse("sjk_hip_copy_blocks: an id outside its slab, a destination twice, or one that is also a source");
    const uint64_t t = tiles(block_bytes / 4);
    if (t > 0x7fffffffu) return refuse("sjk_hip_copy_blocks: too large");
    BlockBatch bt;
    bt.to = d_dst; bt.from = d_src; bt.to_layer = dst_layer_bytes; bt.from_layer = src_layer_bytes; bt.block = block_bytes;
    for (uint32_t i0 = 0; i0 < n; i0 += BLOCK_PAIRS) {
        const uint32_t k = n - i0 < (uint32_t) BLOCK_PAIRS ? n - i0 : (uint32_t) BLOCK_PAIRS;
        for (uint32_t i = 0; i < k; ++i) { bt.src[i] = src_ids[i0 + i]; bt.dst[i] = dst_ids[i0 + i]; }
        hipLaunchKernelGGL(stream_past((uint64_t) n * (uint64_t) n_layers * block_bytes) ? copy_blocks_kernel<true>
                                                                                         : copy_blocks_kernel<false>,
                           dim3((unsigned) t, k, (unsigned) n_layers), dim3(256), 0, (hipStream_t) stream, bt);
        if (SJK_CHECK_LAUNCH()) return SJK_ERR_DEVICE;
    }
    return 0;
}

// The checks of an accept and its launches. host: the path (then d_path is null), in pieces that the arguments hold; a piece's rows go
// where the ones before it end.
namespace sjk {
int accept_rows(const sjk_hip_view * views, int n_layers, const int32_t * d_desc, uint32_t base, int n_nodes, const int32_t * d_path,
                const int32_t * host, int n_path, hipStream_t st) {
    if (n_layers < 0 || (n_layers > 0 && !views) || n_nodes < 0 || n_path < 0) return SJKVARN_ERR_ARG;
    if (!n_layers || !n_path || !n_nodes) return 0;
    if ((!d_path && !host) || ((uintptr_t) d_path & 3u) || ((uintptr_t) d_desc & 3u)) return SJKVARN_ERR_ARG;
    const sjk_hip_view & v0 = views[0];
    if (v0.n_head_kv <= 0 || v0.n_head_kv > 65535 || v0.lay.D <= 0 || (v0.staging != SJKVARN_STAGING_TQ6_0 && v0.staging != SJKVARN_STAGING_F16) ||
        v0.stage_bytes != sj_kvarn_stage_row_bytes(v0.staging, v0.lay.D) || v0.stage_bytes == 0 ||
        (v0.sink_type != SJKVARN_SINK_F16 && v0.sink_type != SJKVARN_SINK_INHERIT))
        return SJKVARN_ERR_ARG;
    for (int il = 0; il < n_layers; ++il) {
        const sjk_hip_view & v = views[il];
        if ((v.S && !v.sink) || (v.cap && !v.ring) || (((uintptr_t) v.sink | (uintptr_t) v.ring) & 3u)) return SJKVARN_ERR_ARG;
        if (v.lay.D != v0.lay.D || v.n_head_kv != v0.n_head_kv || v.staging != v0.staging || v.sink_type != v0.sink_type ||
            v.stage_bytes != v0.stage_bytes || v.S != v0.S || v.cap != v0.cap)
            return refuse("sjk_hip_accept: the views differ in heads, staging, sink or capacity");
    }
    const uint64_t end = (uint64_t) base + (uint64_t) n_nodes;
    if (!d_desc && end > 0xFFFFFFFFull) return SJKVARN_ERR_ARG;
    // staged nodes have a slot each (a descriptor's nodes may all be staged)
    const uint64_t staged = d_desc ? (uint64_t) n_nodes : end <= v0.S ? 0 : end - (base > v0.S ? base : v0.S);
    if (staged > v0.cap) {
        set_error("sjk_hip_accept: more nodes than the ring holds");
        return SJKVARN_ERR_CAPACITY;
    }
    AcceptBatch b;
    const uint32_t H = (uint32_t) v0.n_head_kv;
    b.path = d_path; b.desc = d_desc;
    b.base = base; b.S = v0.S; b.cap = v0.cap ? v0.cap : 1u; b.n_nodes = (uint32_t) n_nodes;
    b.D = v0.lay.D; b.H = v0.n_head_kv; b.side = (int) v0.stage_bytes;
    b.ring_row = H * 2u * (uint32_t) v0.stage_bytes;
    b.sink_row = v0.sink_type == SJKVARN_SINK_F16 ? H * 4u * (uint32_t) b.D : b.ring_row;
    const bool mixed = b.sink_row != b.ring_row && v0.S && (d_desc ? true : base < v0.S && end > v0.S);
    const uint32_t row = b.sink_row > b.ring_row ? b.sink_row : b.ring_row, cols = (row / 4u + 4u * ACC_COLS - 1u) / (4u * ACC_COLS);
    for (int i0 = 0, k; i0 < n_path; i0 += k) {
        k = n_path - i0;
        if (host) {                              // what the list holds: ACC_PATH entries, 65,536 nodes from its first on
            if (k > ACC_PATH) k = ACC_PATH;
            while (host[i0 + k - 1] - host[i0] > 65535) --k;
        }
        b.n_path = (uint32_t) k;
        b.to = (uint32_t) i0;
        b.list0 = host ? (uint32_t) host[i0] : 0u;
        for (int i = 0; host && i < k; ++i) b.list[i] = (uint16_t) (host[i0 + i] - host[i0]);
        for (int l0 = 0; l0 < n_layers; l0 += ACC_LAYERS) {
            const int nl = n_layers - l0 < ACC_LAYERS ? n_layers - l0 : ACC_LAYERS;
            for (int il = 0; il < nl; ++il) { b.layer[il].sink = views[l0 + il].sink; b.layer[il].ring = views[l0 + il].ring; }
            if (mixed) hipLaunchKernelGGL(accept_mixed_kernel, dim3(H, (unsigned) nl), dim3(256), 0, st, b);
            else hipLaunchKernelGGL(accept_kernel, dim3(cols, (unsigned) nl), dim3(256), 0, st, b);
            if (SJK_CHECK_LAUNCH()) return SJK_ERR_DEVICE;
        }
    }
    return 0;
}
}  // namespace sjk

extern "C" int sjk_hip_accept(const sjk_hip_view * views, int n_layers, uint32_t base, int n_nodes, const int32_t * d_path, int n_path,
                              void * stream) {
    if (n_path > 0 && !d_path) return SJKVARN_ERR_ARG;
    return accept_rows(views, n_layers, nullptr, base, n_nodes, d_path, nullptr, n_path, (hipStream_t) stream);
}

extern "C" int sjk_hip_accept_dyn(const sjk_hip_view * views, int n_layers, const int32_t * d_desc, int n_nodes, const int32_t * d_path,
                                  int n_path, void * stream) {
    if (!d_desc || (n_path > 0 && !d_path)) return SJKVARN_ERR_ARG;
    return accept_rows(views, n_layers, d_desc, 0, n_nodes, d_path, nullptr, n_path, (hipStream_t) stream);
}
