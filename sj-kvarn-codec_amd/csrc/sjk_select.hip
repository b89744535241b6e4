// sjk_select.hip - which sealed groups a query position reads (sjk_hip_select_groups and its batch and descriptor forms).
//
// A record's scale tables bound its keys: with codes c in [c0, c1] (0 .. 2^bits - 1, or the trellis codebook's range),
// K[t, d] = (c Kscale[d] + Kzero[d]) Ktok[t], so for every token t of the group
//   q . K[t] <= u max Ktok (u >= 0) or u min Ktok (u < 0),   u = sum_d q_d Kzero_d + max(c1 q_d, c0 q_d) Kscale_d.
// That needs (4 D + 256) bytes of a record and no memory of its own, so commits, forks, truncations and compaction have nothing to
// keep in step. A group's score for a KV head is the largest bound of its query heads; the `top` largest scores are taken,
// of equal ones the lower group.
//
// Sums are 64-bit, on the fp64 matrix unit (v_mfma_f64_16x16x4: 16 groups x 16 query rows x 4 channels): a list is whole
// numbers, and two scores next to its border must not change places with the order of a sum.
//
// What bounds it: few groups, its two launches (5.7 + 3.9 us); 8,000 groups of 8 KV heads of 128 for 4 positions, 22.8 us of scores (49 MB of
// tables in pieces of 768 bytes, 9.5 us at a copy's rate, beside 6.9 us of fp64 products and as much of conversions) and 11.9 of lists (32
// workgroups, counts and barriers).
#include "sjk_mfma.h"

namespace sjk {

typedef double d4 __attribute__((ext_vector_type(4)));

constexpr int SEL_MAXJ = 16;
constexpr int SEL_NT = 256;
constexpr int SEL_GT = 16;                       // groups of a score tile

struct SelJob {
    const uint8_t * body;
    const uint32_t * blocks;
    const float * q;                             // [n_q][n_head][D]
    int32_t * sel;                               // [n_q][H][top]
    double * score;                              // [n_pos][H][stride], of the launch's positions
    uint32_t n;                                  // sealed groups
};
struct SelArgs {
    SelJob job[SEL_MAXJ];
    const int32_t * desc;                        // one job whose groups and place come from the device, or null
    uint32_t n_max, S, cap;                      // for desc
    uint32_t rec_bytes, k_scale, stride;
    int H, n_head, gq, n_q, top, frag;
    int pos0, n_pos;                             // the launch's positions [pos0, pos0 + n_pos) of n_q
    int pb;                                      // positions of a score tile: 16 / gq, at least one
    int tpw;                                     // score tiles of a workgroup
    double c0, c1;
};
static_assert(sizeof(SelArgs) <= 4096, "the jobs travel in the kernel arguments");

// sealed groups of job j; a descriptor that the view cannot hold has none
SJK_DEV uint32_t sel_groups(const SelArgs & a, int j) {
    if (!a.desc) return a.job[j].n;
    const int32_t B = a.desc[SJK_DESC_B], N = a.desc[SJK_DESC_N], Q = a.desc[SJK_DESC_QPOS0];
    const uint32_t b = (uint32_t) B;
    const bool ok = B >= 0 && N >= 0 && Q >= 0 && b <= (uint32_t) N && (uint32_t) N <= a.n_max && b > a.S && (b - a.S) % 128u == 0u &&
                    (uint32_t) Q + 1u >= b;
    // staged positions that the call's rows see: as many as the ring holds
    const uint64_t last = (uint64_t) (uint32_t) Q + (uint32_t) a.n_q, end = (uint64_t) (uint32_t) N < last ? (uint32_t) N : last;
    if (ok && end > b && end - b > a.cap) return 0u;
    return ok ? (b - a.S) / 128u : 0u;
}

// where channel d of the K side lies in the scale tables
SJK_DEV int k_index(int d, int D, int frag) {
    const int j = (d & 15) >> 1;
    return frag ? (j & 3) * (D / 4) + (d >> 4) * 4 + (j >> 2) * 2 + (d & 1) : d;
}

// least and greatest Ktok of a group from the eighths that its 16 lanes (a DPP row) hold; bad: a NaN if one of them is
SJK_DEV void tok_range(const u4 & kt, float & lo, float & hi, float & bad) {
    lo = __builtin_inff(); hi = -__builtin_inff(); bad = 0.0f;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const float x = h2f((kt[e >> 1] >> (16 * (e & 1))) & 0xFFFFu);
        lo = fminf(lo, x);
        hi = fmaxf(hi, x);
        if (x != x) bad = x;
    }
    lo = fminf(lo, dpp<0x128>(lo)); hi = fmaxf(hi, dpp<0x128>(hi)); bad += dpp<0x128>(bad);
    lo = fminf(lo, dpp<0x124>(lo)); hi = fmaxf(hi, dpp<0x124>(hi)); bad += dpp<0x124>(bad);
    lo = fminf(lo, dpp<0x122>(lo)); hi = fmaxf(hi, dpp<0x122>(hi)); bad += dpp<0x122>(bad);
    lo = fminf(lo, dpp<0x121>(lo)); hi = fmaxf(hi, dpp<0x121>(hi)); bad += dpp<0x121>(bad);
}

// scores: grid (runs of tpw 16-group tiles, KV heads, jobs x position tiles). The wavefronts of a workgroup take a quarter of the
// channels each; lane (m, k) loads group m's tables at channels 8 k .. 8 k + 7 of every 32, its A operands. Four workgroups a CU hide
// each other's loads at D = 128 (tables loaded a tile ahead took registers for three: no faster).
template <int D>
__global__ __launch_bounds__(SEL_NT) __attribute__((amdgpu_waves_per_eu(D == 128 ? 4 : 2))) void score_kernel(const SelArgs a) {
    constexpr int NC = D / 128;                  // 8-channel loads of a lane per table
    __shared__ float qs[16][D + 4];              // query rows in the tables' channel order
    __shared__ double part[2][4][16][17];        // (two tiles' sums: one barrier a tile)
    __shared__ double bound[16][17];             // [group][row]
    const int tid = threadIdx.x, lane = tid & 63, m = lane & 15, k = lane >> 4;
    const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int n_pt = (a.n_pos + a.pb - 1) / a.pb, j = (int) blockIdx.z / n_pt, pt = (int) blockIdx.z % n_pt;
    const int h = (int) blockIdx.y;
    const uint32_t n = sel_groups(a, j), first = blockIdx.x * (uint32_t) a.tpw * SEL_GT;
    if (first >= n || n <= (uint32_t) a.top) return;                   // (all of its groups are listed, without scores)
    const uint32_t end = first + (uint32_t) a.tpw * SEL_GT < n ? first + (uint32_t) a.tpw * SEL_GT : n;
    const SelJob & J = a.job[j];
    auto table = [&](uint32_t gi) {              // groups past the end repeat the last one
        gi = gi < n ? gi : n - 1;
        const uint32_t blk = J.blocks ? J.blocks[gi] : gi;
        return J.body + ((size_t) blk * a.H + h) * a.rec_bytes + a.k_scale;
    };
    const int gi = tid >> 4, r16 = tid & 15;     // (group, row) of the sums; (group, sixteenth of its Ktok)
    u4 ks[NC], kz[NC], kt;
    auto load = [&](uint32_t g0) {
        const uint8_t * tb = table(g0 + (uint32_t) m);
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            const int i = (D / 4) * w + 32 * c + 8 * k;
            ks[c] = *(const u4 *) (tb + 2 * i);
            kz[c] = *(const u4 *) (tb + 2 * D + 2 * i);
        }
        kt = *(const u4 *) (table(g0 + (uint32_t) gi) + 4 * D + 16 * r16);
    };
    load(first);
    // query rows of the tile's positions: 16 at a time (one position of more than 16 heads takes several turns)
    const int p0 = a.pos0 + pt * a.pb, np = a.pos0 + a.n_pos - p0 < a.pb ? a.pos0 + a.n_pos - p0 : a.pb;
    const int rows = np * a.gq;
    auto stage = [&](int r0) {
        constexpr int PT = D / 16;
        const int r = r0 + gi < rows ? r0 + gi : rows - 1;
        const float * src = J.q + ((size_t) (p0 + r / a.gq) * a.n_head + h * a.gq + r % a.gq) * D + PT * r16;
#pragma unroll
        for (int e = 0; e < PT; e += 4) {
            const float4 x = *(const float4 *) (src + e);
            const float v[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
            for (int u = 0; u < 4; ++u) qs[gi][k_index(PT * r16 + e + u, D, a.frag)] = v[u];
        }
    };
    stage(0);
    // B operands, of all tiles while a position tile has no more than 16 rows
    double qd[NC][8], wd[NC][8];
    auto rows_to_regs = [&]() {
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            const float * qr = &qs[m][(D / 4) * w + 32 * c + 8 * k];
            const f4 q0 = *(const f4 *) qr, q1 = *(const f4 *) (qr + 4);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                qd[c][e] = (double) (e < 4 ? q0[e & 3] : q1[e & 3]);
                wd[c][e] = qd[c][e] > 0.0 ? qd[c][e] * a.c1 : qd[c][e] * a.c0;       // exact: 24 and 11 bits
            }
        }
    };
    __syncthreads();
    rows_to_regs();
    int turn = 0;
    for (uint32_t g0 = first; g0 < end; g0 += SEL_GT) {
        float lo, hi, bad;
        tok_range(kt, lo, hi, bad);
        double best = -__builtin_inf();          // thread (group gi, position r16 < np)
        for (int r0 = 0; r0 < rows; r0 += 16) {
            if (rows > 16 && (g0 > first || r0 > 0)) {
                __syncthreads();                 // the rows before these have been read
                stage(r0);
                __syncthreads();
                rows_to_regs();
            }
            d4 acc = {0.0, 0.0, 0.0, 0.0}, acw = acc;
#pragma unroll
            for (int c = 0; c < NC; ++c)
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const uint32_t sh = 16 * (e & 1);
                    uint32_t z = kz[c][e >> 1], s = ks[c][e >> 1];
                    asm volatile("" : "+v"(z), "+v"(s));               // converted here: 32 registers of doubles less, no spill
                    acc = __builtin_amdgcn_mfma_f64_16x16x4f64((double) h2f((z >> sh) & 0xFFFFu), qd[c][e], acc, 0, 0, 0);
                    acw = __builtin_amdgcn_mfma_f64_16x16x4f64((double) h2f((s >> sh) & 0xFFFFu), wd[c][e], acw, 0, 0, 0);
                }
            // lane (row m, k): groups 4 i + k
            double (*pw)[16][17] = part[turn & 1];
            ++turn;
#pragma unroll
            for (int i = 0; i < 4; ++i) pw[w][4 * i + k][m] = acc[i] + acw[i];
            __syncthreads();
            const double u = (pw[0][gi][r16] + pw[1][gi][r16]) + (pw[2][gi][r16] + pw[3][gi][r16]);
            wave_sync();                         // a group's rows stay in its wavefront
            bound[gi][r16] = bad != 0.0f ? (double) bad : u >= 0.0 ? u * (double) hi : u * (double) lo;
            wave_sync();
            const int nr = rows - r0 < 16 ? rows - r0 : 16;
            if (r16 < np) {                      // the rows of position r16 in this turn (all of them, unless there are several)
                const int a0 = a.gq <= 16 ? r16 * a.gq : 0, a1 = a.gq <= 16 ? a0 + a.gq : nr;
#pragma unroll 1
                for (int r = a0; r < a1; ++r) {
                    const double x = bound[gi][r];
                    best = x > best || x != x ? x : best;              // a NaN stays: no number is greater
                }
            }
        }
        if (g0 + SEL_GT < end) load(g0 + SEL_GT);
        if (r16 < np && g0 + (uint32_t) gi < n)
            J.score[((size_t) (p0 - a.pos0 + r16) * a.H + h) * a.stride + g0 + gi] = best;
    }
}

// scores as unsigned numbers of the same order; -0 counts as 0, a NaN is above all (a group whose bound is not a number is
// read, so that it shows in the attention)
SJK_DEV uint64_t sel_key(double x) {
    if (x != x) return ~0ull;
    const uint64_t b = (uint64_t) __double_as_longlong(x + 0.0);
    return (b >> 63) ? ~b : b | 0x8000000000000000ull;
}

// The list of one (position, KV head): the border is found digit by digit from the highest bit in which the keys differ, until the
// keys that share the border's digits are just those still wanted; then the places of the taken ones in order of the groups.
// NT threads; KPT: keys per thread, adjacent groups, in registers, or 0: read again for every digit.
template <int NT, int KPT>
__global__ __launch_bounds__(NT) void pick_kernel(const SelArgs a) {
    constexpr int NW = NT / 64, NK = KPT ? KPT : 8;
    constexpr int HC = NT > 256 ? 8 : 1;         // counts per digit, one for every eighth lane: the first digits of most keys are alike
    __shared__ uint32_t hist[256 * HC];
    __shared__ unsigned long long s_or;
    __shared__ uint32_t s_digit, s_left, s_all;
    __shared__ uint32_t w_sel[NW], w_tie[NW];
    const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
    const int j = (int) blockIdx.y, list = (int) blockIdx.x;           // list = position x H + KV head
    const SelJob & J = a.job[j];
    const uint32_t n = sel_groups(a, j), top = (uint32_t) a.top;
    int32_t * out = J.sel + ((size_t) a.pos0 * a.H + list) * top;
    const double * sc = J.score + (size_t) list * a.stride;
    if (n <= top) {
        for (uint32_t i = tid; i < top; i += NT) out[i] = i < n ? (int32_t) i : -1;
        return;
    }
    // keys of a turn of NT x NK groups; keys past the end are 0, below every key of a number
    uint64_t key[NK];
    auto load = [&](uint32_t i0) {
#pragma unroll
        for (int e = 0; e < NK; ++e) {
            const uint32_t i = i0 + (uint32_t) tid * NK + e;
            key[e] = i < n ? sel_key(sc[i]) : 0;
        }
    };
    const uint64_t first = sel_key(sc[0]);
    load(0);
    if (tid == 0) s_or = 0;
    __syncthreads();
    {   // the bits in which any key differs from the first
        uint64_t d = 0;
        for (uint32_t i0 = 0; i0 < n; i0 += NT * NK) {
            if (!KPT && i0) load(i0);
#pragma unroll
            for (int e = 0; e < NK; ++e)
                if (i0 + (uint32_t) tid * NK + e < n) d |= key[e] ^ first;
        }
#pragma unroll
        for (int s = 1; s < 64; s <<= 1) {
            const uint32_t lo = __shfl_xor((uint32_t) d, s, 64), hi = __shfl_xor((uint32_t) (d >> 32), s, 64);
            d |= lo | ((uint64_t) hi << 32);
        }
        if (lane == 0 && d) atomicOr(&s_or, (unsigned long long) d);
    }
    __syncthreads();
    // border: keys with key >> shift above pre are taken, of those equal to it the first `left`
    int shift = s_or ? 64 - (int) __clzll((long long) s_or) : 0;       // the digits above are the same in all keys
    uint64_t pre = shift < 64 ? first >> shift : 0;
    uint32_t left = top;
    while (shift > 0) {
        const int bits = shift < 8 ? shift : 8, sh = shift - bits;
        for (int i = tid; i < 256 * HC; i += NT) hist[i] = 0;
        __syncthreads();
        for (uint32_t i0 = 0; i0 < n; i0 += NT * NK) {
            if (!KPT) load(i0);
#pragma unroll
            for (int e = 0; e < NK; ++e)
                if (i0 + (uint32_t) tid * NK + e < n && (shift == 64 || (key[e] >> shift) == pre))
                    atomicAdd(&hist[((uint32_t) (key[e] >> sh) & ((1u << bits) - 1u)) * HC + (lane & (HC - 1))], 1u);
        }
        __syncthreads();
        if (tid < 64) {                          // digits 4 lane .. 4 lane + 3: how many keys have a higher one
            uint32_t c[4], sum = 0;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                c[e] = 0;
#pragma unroll
                for (int k = 0; k < HC; ++k) c[e] += hist[(4 * lane + e) * HC + k];
                sum += c[e];
            }
            uint32_t above = sum;                // of this lane and the ones after it
#pragma unroll
            for (int s = 1; s < 64; s <<= 1) {
                const uint32_t o = __shfl_down(above, s, 64);
                if (lane + s < 64) above += o;
            }
            above -= sum;
#pragma unroll
            for (int e = 3; e >= 0; --e) {
                if (above < left && left <= above + c[e]) { s_digit = (uint32_t) (4 * lane + e); s_left = left - above; s_all = c[e]; }
                above += c[e];
            }
        }
        __syncthreads();
        pre = (shift == 64 ? 0 : pre << bits) | s_digit;
        left = s_left;
        shift = sh;
        if (s_all == left) break;                // (the next writes of s_* are two barriers away)
    }
    uint32_t done = 0, ties = 0;
    for (uint32_t i0 = 0; i0 < n; i0 += NT * NK) {
        if (!KPT) load(i0);
        // this thread's counts of taken and of equal keys, and those of the threads before it
        uint32_t nt = 0, ng = 0;
#pragma unroll
        for (int e = 0; e < NK; ++e) {
            const bool in = i0 + (uint32_t) tid * NK + e < n;
            nt += in && (key[e] >> shift) == pre;
            ng += in && (key[e] >> shift) > pre;
        }
        uint32_t both = ng | (nt << 16), inc = both;                   // at most 512 of a wavefront
#pragma unroll
        for (int s = 1; s < 64; s <<= 1) {
            const uint32_t o = __shfl_up(inc, s, 64);
            if (lane >= s) inc += o;
        }
        __syncthreads();                         // the last turn's counts have been read
        if (lane == 63) { w_sel[w] = inc & 0xFFFFu; w_tie[w] = inc >> 16; }
        __syncthreads();
        uint32_t g = done + (inc & 0xFFFFu) - ng, t = ties + (inc >> 16) - nt;
#pragma unroll
        for (int x = 0; x < NW; ++x) {
            if (x < w) { g += w_sel[x]; t += w_tie[x]; }
            done += w_sel[x];
            ties += w_tie[x];
        }
#pragma unroll
        for (int e = 0; e < NK; ++e) {
            const uint32_t i = i0 + (uint32_t) tid * NK + e;
            if (i >= n) continue;
            const uint64_t kk = key[e] >> shift;
            if (kk > pre || (kk == pre && t < left)) out[g + (t < left ? t : left)] = (int32_t) i;
            g += kk > pre;
            t += kk == pre;
        }
    }
}

// range of a K side's code values
static void code_range(const sj_kvarn_layout & l, double & c0, double & c1) {
    c0 = 0.0;
    c1 = (double) ((1 << l.bits_k) - 1);
    if (l.body != SJKVARN_BODY_TRELLIS) return;
    static const uint16_t cb3[] = SJK_CB3_K_INIT, cb2[] = SJK_CB2_K_INIT;
    const uint16_t * cb = l.bits_k == 3 ? cb3 : cb2;
    const int n = l.bits_k == 3 ? 512 : 256;
    c0 = c1 = (double) sj_kvarn_f16_to_f32(cb[0]);
    for (int i = 1; i < n; ++i) {
        const double x = (double) sj_kvarn_f16_to_f32(cb[i]);
        if (x < c0) c0 = x;
        if (x > c1) c1 = x;
    }
}

}  // namespace sjk

using namespace sjk;

extern "C" int sjk_attend3_supported(const sjk_hip_view * v);

// what every form asks of a view and its call
static int sel_args(const sjk_hip_view & v, int n_q, int n_head, const float * q, int top, const int32_t * sel) {
    if (!q || !sel || ((uintptr_t) q & 15u) || ((uintptr_t) sel & 3u) || n_q <= 0 || n_head <= 0 || top <= 0 || v.n_head_kv <= 0 ||
        n_head % v.n_head_kv)
        return SJKVARN_ERR_ARG;
    if (!sjk_attend3_supported(&v)) {
        set_error("the view is not one the attention kernels are built for (a layer's own layout)");
        return SJK_ERR_UNSUPPORTED;
    }
    if (v.n_head_kv > n_cus() || (int64_t) n_q * v.n_head_kv > 0x7fffffff) return SJKVARN_ERR_ARG;
    return 0;
}

static size_t sel_room(const sjk_hip_view & v) { return ws_part_slots(v) * ws_slot_floats(v.lay.D) * sizeof(float) / sizeof(double); }

static int sel_full() {
    set_error("sjk_hip_select_groups: the scores of one position do not fit the view's workspace");
    return SJKVARN_ERR_CAPACITY;
}

// n_jobs <= SEL_MAXJ jobs of one shape; most: the largest number of groups any of them can have
static int sel_launch(SelArgs & a, const sjk_hip_view & v, int n_jobs, size_t room, uint32_t most, hipStream_t st) {
    const sj_kvarn_layout & l = v.lay;
    a.S = v.S; a.cap = v.cap;
    a.rec_bytes = l.bytes;
    a.k_scale = l.k_scale;
    a.H = v.n_head_kv;
    a.gq = a.n_head / a.H;
    a.frag = l.body == SJKVARN_BODY_SCALAR && l.bits_k == 4;
    a.pb = a.gq < 16 ? 16 / a.gq : 1;
    code_range(l, a.c0, a.c1);
    const bool scored = most > (uint32_t) a.top; // else every list is all groups
    a.stride = scored ? most : 0;
    int chunk = a.n_q;                           // positions whose scores the workspaces hold at once
    if (scored) {
        const size_t fit = room / ((size_t) a.H * most);
        if (fit == 0) return sel_full();
        if ((size_t) chunk > fit) chunk = (int) fit;
    }
    if (chunk > 2048) chunk = 2048;              // grid z: jobs x position tiles
    for (a.pos0 = 0; a.pos0 < a.n_q; a.pos0 += chunk) {
        a.n_pos = a.n_q - a.pos0 < chunk ? a.n_q - a.pos0 : chunk;
        if (scored) {
            // a tile a workgroup up to 8 of them a CU (two rounds), then runs of up to 16 that are all on the device at once
            // (1M positions of 8 KV heads, 4,000 tiles: runs of 4 25.6 -> 22 us)
            const uint64_t tiles = (most + SEL_GT - 1) / SEL_GT, others = (uint64_t) a.H * (uint64_t) (n_jobs * ((a.n_pos + a.pb - 1) / a.pb));
            const uint64_t cus = (uint64_t) n_cus(), run = (tiles * others + 4u * cus - 1) / (4u * cus);
            a.tpw = tiles * others <= 8u * cus ? 1 : run > 16 ? 16 : (int) run;
            const dim3 grid((unsigned) ((tiles + a.tpw - 1) / a.tpw), (unsigned) a.H, (unsigned) (others / (uint64_t) a.H));
            if (l.D == 128) hipLaunchKernelGGL(score_kernel<128>, grid, dim3(SEL_NT), 0, st, a);
            else hipLaunchKernelGGL(score_kernel<256>, grid, dim3(SEL_NT), 0, st, a);
        }
        const dim3 lists((unsigned) (a.n_pos * a.H), (unsigned) n_jobs);
        if (most <= 256u) hipLaunchKernelGGL((pick_kernel<256, 1>), lists, dim3(256), 0, st, a);
        else if (most <= 1024u) hipLaunchKernelGGL((pick_kernel<256, 4>), lists, dim3(256), 0, st, a);
        else if (most <= 8192u) hipLaunchKernelGGL((pick_kernel<1024, 8>), lists, dim3(1024), 0, st, a);
        else hipLaunchKernelGGL((pick_kernel<1024, 0>), lists, dim3(1024), 0, st, a);
        if (SJK_CHECK_LAUNCH()) return SJK_ERR_DEVICE;
    }
    return 0;
}

extern "C" int sjk_hip_select_groups_batch(const sjk_hip_groups_job * jobs, int n_jobs, int n_q, int n_head, int top, void * stream) {
    if (n_jobs < 0 || (n_jobs > 0 && !jobs)) return SJKVARN_ERR_ARG;
    for (int k = 0; k < n_jobs; ++k) {
        const sjk_hip_groups_job & J = jobs[k];
        const sjk_hip_view & v = J.v, & v0 = jobs[0].v;
        if (const int rc = sel_args(v, n_q, n_head, J.d_q, top, J.d_sel)) return rc;
        if (const int rc = groups_ok(v, J.B, J.N, J.qpos0, n_q)) return rc;
        const uint32_t bend = J.B > v.S ? J.B : v.S, last = J.qpos0 + (uint32_t) n_q, end = J.N < last ? J.N : last;
        if (end > bend && end - bend > v.cap) {
            set_error("sjk_hip_select_groups: more staged positions than the ring holds");
            return SJKVARN_ERR_CAPACITY;
        }
        if (J.B > v.S && (J.B - v.S) / 128u > (uint32_t) top && !v.work) return SJKVARN_ERR_ARG;
        if (v.lay.D != v0.lay.D || v.lay.bits_k != v0.lay.bits_k || v.lay.bits_v != v0.lay.bits_v || v.lay.body != v0.lay.body ||
            v.n_head_kv != v0.n_head_kv)
            return refuse("sjk_hip_select_groups_batch: the views differ in layout or KV heads");
    }
    auto groups = [&](int k) { return jobs[k].B > jobs[k].v.S ? (jobs[k].B - jobs[k].v.S) / 128u : 0u; };
    auto scored = [&](int k) { return groups(k) > (uint32_t) top; };
    // before the first launch: every job's scores of one position fit its workspace
    for (int k = 0; k < n_jobs; ++k)
        if (scored(k) && sel_room(jobs[k].v) < (size_t) jobs[k].v.n_head_kv * groups(k)) return sel_full();
    // Jobs with scores that share a workspace (the layers of a sequence) share its room: the scores that each of the n jobs from k0 on
    // may hold; most: the groups of the longest
    auto share = [&](int k0, int n, uint32_t & most) {
        size_t room = ~(size_t) 0;
        most = 0;
        for (int k = k0; k < k0 + n; ++k) {
            if (groups(k) > most) most = groups(k);
            if (!scored(k)) continue;
            size_t on_it = 0;
            for (int i = k0; i < k0 + n; ++i) on_it += scored(i) && jobs[i].v.work == jobs[k].v.work;
            const size_t r = sel_room(jobs[k].v) / on_it;
            if (r < room) room = r;
        }
        return room;
    };
    for (int k0 = 0, n; k0 < n_jobs; k0 += n) {
        // as many jobs a launch as have room for the longest one's scores of a position; the next launch follows on the stream
        uint32_t most;
        n = n_jobs - k0 < SEL_MAXJ ? n_jobs - k0 : SEL_MAXJ;
        size_t room = share(k0, n, most);
        while (n > 1 && most > (uint32_t) top && room < (size_t) jobs[0].v.n_head_kv * most) room = share(k0, --n, most);
        SelArgs a = {};
        a.n_q = n_q; a.n_head = n_head; a.top = top;
        for (int k = 0; k < n; ++k) {
            const sjk_hip_groups_job & J = jobs[k0 + k];
            SelJob & s = a.job[k];
            s.body = J.v.body; s.blocks = J.v.blocks; s.q = J.d_q; s.sel = J.d_sel;
            s.n = groups(k0 + k);
            if (!scored(k0 + k)) continue;
            size_t rank = 0;
            for (int i = k0; i < k0 + k; ++i) rank += scored(i) && jobs[i].v.work == J.v.work;
            s.score = (double *) ws_part(J.v) + rank * room;
        }
        if (const int rc = sel_launch(a, jobs[k0].v, n, room, most, (hipStream_t) stream)) return rc;
    }
    return 0;
}

extern "C" int sjk_hip_select_groups(const sjk_hip_view * v, uint32_t B, uint32_t N, uint32_t qpos0, int n_q, int n_head, const float * d_q,
                                     int top, int32_t * d_sel, void * stream) {
    if (!v) return SJKVARN_ERR_ARG;
    sjk_hip_groups_job J = {};
    J.v = *v; J.B = B; J.N = N; J.qpos0 = qpos0; J.d_q = d_q; J.d_sel = d_sel;
    return sjk_hip_select_groups_batch(&J, 1, n_q, n_head, top, stream);
}

extern "C" int sjk_hip_select_groups_dyn(const sjk_hip_view * v, const int32_t * d_desc, uint32_t n_max, int n_q, int n_head,
                                         const float * d_q, int top, int32_t * d_sel, void * stream) {
    if (!v || !d_desc || ((uintptr_t) d_desc & 3u)) return SJKVARN_ERR_ARG;
    if (const int rc = sel_args(*v, n_q, n_head, d_q, top, d_sel)) return rc;
    const uint32_t most = n_max > v->S ? (n_max - v->S) / 128u : 0u;
    if (most && !v->body) return SJKVARN_ERR_ARG;
    if (most > (uint32_t) top && !v->work) return SJKVARN_ERR_ARG;
    SelArgs a = {};
    a.n_q = n_q; a.n_head = n_head; a.top = top;
    a.desc = d_desc; a.n_max = n_max;
    a.job[0].body = v->body; a.job[0].blocks = v->blocks; a.job[0].q = d_q; a.job[0].sel = d_sel;
    a.job[0].score = v->work ? (double *) ws_part(*v) : nullptr;
    return sel_launch(a, *v, 1, sel_room(*v), most, (hipStream_t) stream);
}
