// sjk_pages.hip - pages of a cache from one place to another: the sink and staged rows of a fork (sjk_hip_fork) and
// record blocks of a pool (sjk_hip_copy_blocks).
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
