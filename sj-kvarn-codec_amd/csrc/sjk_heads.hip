// sjk_heads.hip - rows between a layer's projections and its cache: head norms, rotary positions, the rotation into the
// cache's basis, and the append, in one pass over the rows (sjk_hip_head_rows, sjk_hip_store_qkv).
//
// A row (one head at one position) lies 8 consecutive channels a lane in LPR lanes, so a wavefront holds 64 / LPR rows and
// reads and writes 16 or 32 bytes a lane. The rows are the same head at adjacent positions, or adjacent heads of one position
// (HF_BY_HEAD), and the wavefront goes through a run of heads of one set, the next loads issued before the current rows'
// arithmetic: a lane keeps its position, whose sines, cosines and cache slot it works out once.
//   * norm: the sum of squares is a fixed tree (pairs in the lane, then lanes 1, 2, 4, ... apart), so a row's bits do not
//     depend on the rows beside it.
//   * turn: u = position * turns per position in double, reduced to (-1/2, 1/2] turns and then to an eighth of one either
//     side of a quarter before it becomes a float: nothing is lost at far positions, and the sine and cosine are short
//     polynomials; no table of positions is read. Where the halves of a whole head are paired, the two lanes of a pair make
//     half of their sines and cosines each and exchange them.
//   * the Hadamard and the staging are those of the row kernel (sjk_rows.hip): the same bytes.
#include "sjk_dev.h"
#include "sjk_row.h"

namespace sjk {

constexpr int HW = 4;                  // wavefronts a workgroup
constexpr int HEAD_PARTS = 3;          // sets of heads a launch: q, k, v
constexpr int HEAD_SEQS = 32;          // sequences a launch
constexpr int HEAD_ITERS = 8;          // heads a wavefront goes through at most
constexpr int TQ_BATCH = 4;            // of them staged as tq6_0 together
enum { HP_ROWS = 0, HP_K = 1, HP_V = 2 };                               // where a part's rows go
enum { HF_ROPE = 1, HF_ROT = 2, HF_BY_HEAD = 4 };
enum { HM_ROWS = 0, HM_F16 = 1, HM_TQ6 = 2 };                           // a launch: plain rows only, or a cache's staging
enum { HO_F32 = 0, HO_HALF = 1, HO_CACHE = 2 };                         // a wavefront's rows
template <int N> struct Int { static constexpr int value = N; };

struct HeadPart {
    int64_t x_pos, x_head, o_pos, o_head, w_head;
    const float * w;
    float eps;
    int n_heads, n_iters, n_chunks, n_units, flags, kind, o_type;      // iterations of a wavefront, runs of heads, wavefronts
};

struct HeadSeq {
    const void * x[HEAD_PARTS];
    void * o[HEAD_PARTS];              // HP_ROWS: the part's rows; of a cache also [1] sink, [2] ring
    const int32_t * pos;
    uint32_t pos0, S, cap;
};

struct HeadBatch {
    HeadPart part[HEAD_PARTS];
    HeadSeq seq[HEAD_SEQS];
    const double * turns;
    const int32_t * desc;
    size_t stage_bytes;
    int n_parts, n_seqs, n_pos, D, units;              // units: wavefronts of one sequence
    int layout, n_rot, H, sink_type;
    float mscale, sine, rot_scale, inv_D;              // sine: the sign of sines (inverse)
};

static_assert(sizeof(HeadBatch) <= 4096, "the table travels in the kernel arguments");

// sine and cosine of u turns, times m (sines also times sg)
SJK_DEV void turn(double u, float m, float sg, float & s, float & c) {
    u -= __builtin_rint(u);
    const float q = __builtin_rintf(4.0f * (float) u);
    const float r = (float) __builtin_fma((double) q, -0.25, u);        // |r| <= 1/8 (and an ulp)
    const float z = r * r;
    // Taylor series in r, coefficients (2 pi)^k / k!: the first term left out is below 3e-9 of the
    // sine, 2e-10 of the cosine
    float p = __builtin_fmaf(z, 42.058693944897654f, -76.70585975306138f);
    p = __builtin_fmaf(z, p, 81.60524927607504f);
    p = __builtin_fmaf(z, p, -41.341702240399755f);
    const float sn = __builtin_fmaf(r * z, p, r * 6.283185307179586f);
    p = __builtin_fmaf(z, -26.426256783374398f, 60.24464137187666f);
    p = __builtin_fmaf(z, p, -85.45681720669373f);
    p = __builtin_fmaf(z, p, 64.93939402266829f);
    p = __builtin_fmaf(z, p, -19.739208802178716f);
    const float cs = __builtin_fmaf(z, p, 1.0f);
    const int k = (int) q;                                              // quarter turns, -2 .. 2
    const float a = k & 1 ? cs : sn, b = k & 1 ? sn : cs;
    s = (k & 2 ? -a : a) * m * sg;
    c = ((k + 1) & 2 ? -b : b) * m;
    __builtin_amdgcn_sched_barrier(0);       // one after the other: interleaved, their temporaries set the kernel's registers
}

// tq6_level by one look into a table: the line is cut into LV_CELLS cells so narrow that each holds at most one midpoint, which a
// comparison then decides exactly. The cell of a value is a monotone function of it, the same for midpoints and values, so every
// midpoint of a lower cell is below the value and every one of a higher cell above. (With the search's six dependent
// reads 4,096 positions of 32 + 8 heads of 128 to tq6_0 take 6 us more.) Cells are counted downwards, by the negated value: the
// hardware's median of a NaN and two others is their lesser, so a NaN (infinity * 0 where a block's norm is infinite) falls in the
// highest cell, where the comparison is false, and gets level 63, as in the search (with a test of its own in its place, 16-bit rows
// of 128 turned in part have 12 wavefronts a CU for 16: 2,048 positions 24.6 us for 19.5, 512 12.9 for 10.0).
constexpr int LV_CELLS = 128;
constexpr float LV_SCALE = 200.0f;
struct LevelCell { float mid; int base; };                 // the cell's midpoint, the midpoints of lower cells (a cell without one:
                                                           // -infinity, and one fewer)
struct LevelTable { LevelCell cell[LV_CELLS]; };
constexpr float level_at(float v) { return v * LV_SCALE + 64.0f; }
constexpr int level_cell(float v) { const float t = level_at(v); return t < 0.0f ? 0 : t > 127.0f ? 127 : (int) t; }
constexpr LevelTable level_table() {
    constexpr uint32_t bits[63] = SJK_TQ6_MIDPOINT_BITS_INIT;
    LevelTable t = {};
    for (int c = 0; c < LV_CELLS; ++c) {
        t.cell[c].mid = -__builtin_inff();
        t.cell[c].base = -1;
        for (int i = 0; i < 63; ++i) {
            const float m = __builtin_bit_cast(float, bits[i]);
            if (level_cell(-m) >= c) ++t.cell[c].base;
            if (level_cell(-m) == c) t.cell[c].mid = m;
        }
    }
    return t;
}
constexpr bool level_table_ok() {                          // no cell with two midpoints, midpoints in ascending order
    constexpr uint32_t bits[63] = SJK_TQ6_MIDPOINT_BITS_INIT;
    for (int i = 1; i < 63; ++i)
        if (level_cell(-__builtin_bit_cast(float, bits[i])) >= level_cell(-__builtin_bit_cast(float, bits[i - 1]))) return false;
    return true;
}
static_assert(level_table_ok(), "one midpoint a cell");
static __constant__ LevelTable c_levels = level_table();

SJK_DEV int level_of(float v, const LevelCell * cells) {
    const LevelCell c = cells[(int) __builtin_amdgcn_fmed3f(level_at(-v), 0.0f, 127.0f)];
    return c.base + (v < c.mid ? 0 : 1);
}

// 8 channels of a row from its element e0 on, as raw words. WIDE: 16 bytes at a time, else element by element up to D.
template <typename T> struct Raw { uint32_t w[2 * sizeof(T)]; };
template <typename T, bool WIDE> SJK_DEV void load_row(Raw<T> & r, const T * p, int e0, int D) {
    constexpr int NW = 2 * (int) sizeof(T);
    if constexpr (WIDE) {
#pragma unroll
        for (int i = 0; i < NW; i += 4) {
            const uint4 v = *(const uint4 *) ((const uint32_t *) (p + e0) + i);
            r.w[i] = v.x; r.w[i + 1] = v.y; r.w[i + 2] = v.z; r.w[i + 3] = v.w;
        }
    } else {
#pragma unroll
        for (int i = 0; i < NW; ++i) r.w[i] = 0;
#pragma unroll
        for (int m = 0; m < 8; ++m)
            if (e0 + m < D) {
                if constexpr (sizeof(T) == 4) r.w[m] = __builtin_bit_cast(uint32_t, p[e0 + m]);
                else r.w[m >> 1] |= (uint32_t) __builtin_bit_cast(uint16_t, p[e0 + m]) << (16 * (m & 1));
            }
    }
}
template <typename T> SJK_DEV float raw_at(const Raw<T> & r, int m) {
    if constexpr (sizeof(T) == 4) return bits_f(r.w[m]);
    else if constexpr (__is_same(T, __bf16)) return bits_f(m & 1 ? r.w[m >> 1] & 0xFFFF0000u : r.w[m >> 1] << 16);
    else return (float) __builtin_bit_cast(T, (uint16_t) (r.w[m >> 1] >> (16 * (m & 1))));
}

typedef float float2_t __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2_t __attribute__((ext_vector_type(2)));

SJK_DEV uint32_t pack_f16(float a, float b) {
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((float2_t{a, b}), f16x2_t));
}
SJK_DEV uint32_t pack_bf16(float a, float b) {
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((float2_t{a, b}), bf16x2_t));
}

template <bool WIDE> SJK_DEV void store_halves(uint16_t * o, const uint32_t (&h)[4], int e0, int D) {
    if constexpr (WIDE) {
        *(uint4 *) o = uint4{h[0], h[1], h[2], h[3]};
    } else {
#pragma unroll
        for (int m = 0; m < 8; ++m) if (e0 + m < D) o[m] = (uint16_t) (h[m >> 1] >> (16 * (m & 1)));
    }
}

// whether v is an infinity or a NaN
SJK_DEV bool nonfinite(float v) { return __builtin_amdgcn_classf(v, 0x207); }

// The rotation with the host's NaN rule in the rows where xn is set, through the wavefront's LDS (512 floats), a lane four pairs
// of every stage: such rows are rare, so this is short rather than fast. The values of the other rows are hadamard_row's, signs of
// NaNs included: as it is compiled, of two NaNs a sum keeps the upper one, a difference the lower one where the partner comes by
// DPP (LPR / 8 values a lane in 64 lanes there) and the upper one where it comes by a row swap, and an upper one's sign is turned.
template <int LPR> SJK_DEV void hadamard_rows_x(float (&x)[8], float * buf, int lane, float scale, bool xn) {
    const int l = lane % LPR;
    float * row = buf + lane / LPR * (8 * LPR);
    wave_sync();
#pragma unroll
    for (int m = 0; m < 8; ++m) row[8 * l + m] = x[m];
    wave_sync();
#pragma unroll 1
    for (int h = 1; h < 8 * LPR; h *= 2) {
#pragma unroll 1
        for (int k = 4 * l; k < 4 * l + 4; ++k) {
            const int j = 2 * (k & -h) + (k & (h - 1));
            const float a = row[j], b = row[j + h];
            const float n = -b;
            const bool swap = h >= 16 * (LPR / 8);
            row[j] = xn ? xadd(a, b) : b != b ? b : a + b;
            row[j + h] = xn ? xsub(a, b) : swap && b != b ? n : a != a ? a : b != b ? n : a - b;
        }
        wave_sync();
    }
#pragma unroll
    for (int m = 0; m < 8; ++m) {
        const float v = row[8 * l + m];
        x[m] = xn ? xmul(v, scale) : v * scale;
    }
    wave_sync();
}

// KIND: which calls the kernel is for. The first has no masks and no addresses for what it does not do.
enum { HK_WHOLE = 0,        // rows of 8 * LPR channels whose addresses and strides take 16-byte accesses, turned whole or not at
                            // all, and one set of norm weights for all heads of a job
       HK_PART = 1,         // such accesses otherwise, a turn of halves over a multiple of 16 channels
       HK_ODD = 2,          // such accesses, a turn of halves over another number: pairs through LDS
       HK_ANY = 3 };        // rows of any width, address and stride, any turn, element by element (3,226 positions x 6 heads of 256
                            // turned over 232 channels: 25.7 us, 14.0 by HK_ODD)
// (HK_WHOLE: 16 wavefronts a CU, as launch_heads counts on, 128 registers; tq6_0 takes 120 to 128 of them)
template <typename T, int LPR, int MODE, int KIND>
__global__ __launch_bounds__(64 * HW, KIND == HK_WHOLE ? 4 : 1) void heads_kernel(const HeadBatch bt) {
    // Lanes behind the last row take the last row again, and lanes behind a row's channels its first ones, and write the same
    // values once more (both read in one instruction, so also where rows are written over themselves): loads and stores without
    // a branch around them, so that a wait for the next row's loads does not wait for this row's stores (on gfx9 one counter
    // holds both, and the compiler can count past the stores only where they are certain: 8,192 positions x 40 heads of
    // 128 turned in 39.5 us with branches, 36.1 without).
    constexpr bool ALL = KIND != HK_ANY;
    constexpr int RPW = 64 / LPR;                          // rows a wavefront holds
    constexpr int BS = 132;                                // floats from a 128-value block to the next (walks: other banks)
    constexpr int TB = MODE == HM_TQ6 ? TQ_BATCH : 1;      // heads staged together
    constexpr int WS = MODE == HM_TQ6 ? TB * 4 * BS : 512; // floats of a wavefront's LDS
    // reads in flight of a tq6_0 walk: 4 take 16 registers less and calls of few wavefronts 0.4 us more (64 positions 6.8 -> 7.3), so
    // only where 8 do not fit the bound above
    constexpr int UNROLL = KIND == HK_WHOLE && LPR == 16 && sizeof(T) == 4 ? 4 : 8;
    __shared__ alignas(16) float s_buf[HW * WS];
    __shared__ LevelCell s_cell[MODE == HM_TQ6 ? LV_CELLS : 1];
    __shared__ float s_cent[MODE == HM_TQ6 ? 64 : 1];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, sub = lane / LPR, D = KIND == HK_WHOLE ? 8 * LPR : bt.D;
    const bool again = ALL && KIND != HK_WHOLE && lane % LPR >= D / 8;    // a lane behind the row's channels
    // (rows of 32 channels and more take at least half of their lanes, narrower ones a quarter or an eighth)
    const int l = lane % LPR - (again ? LPR == 8 && D < 32 ? lane % LPR / (D / 8) * (D / 8) : D / 8 : 0), e0 = 8 * l;
    if (MODE == HM_TQ6) {
        if (threadIdx.x < LV_CELLS) s_cell[threadIdx.x] = c_levels.cell[threadIdx.x];
        if (threadIdx.x < 64) s_cent[threadIdx.x] = tq6_cent(threadIdx.x);
        __syncthreads();
    }
    // this wavefront's sequence, part, positions and heads (wave-uniform)
    int u = __builtin_amdgcn_readfirstlane((int) blockIdx.x * HW + wave);
    const int si = u / bt.units;
    if (si >= bt.n_seqs) return;
    u -= si * bt.units;
    int pi = bt.n_parts - 1;                               // keys and values first: staging them takes longest (last, 4,096
                                                           // positions to tq6_0 took 49 us for 39)
    while (pi > 0 && u >= bt.part[pi].n_units) u -= bt.part[pi--].n_units;
    const HeadPart & P = bt.part[pi];
    const HeadSeq & Q = bt.seq[si];
    if (bt.desc && bt.desc[SJK_DESC_QPOS0] < 0) return;
    const uint32_t pos0 = bt.desc ? (uint32_t) bt.desc[SJK_DESC_QPOS0] : Q.pos0;
    const int n_heads = P.n_heads, step = P.flags & HF_BY_HEAD ? RPW : 1;
    const bool rope = P.flags & HF_ROPE, rot = P.flags & HF_ROT;
    float * buf = s_buf + wave * WS;

    // the lane's rows: position cp, heads head_at(it, sub) of iterations it (ALL: of adjacent heads not past the last)
    const int block = u / P.n_chunks, run = u - block * P.n_chunks, h0 = run * P.n_iters * step;
    const int iters = min(P.n_iters, (n_heads - h0 + step - 1) / step);
    const bool by_head = P.flags & HF_BY_HEAD, uneven = ALL && by_head && n_heads % RPW;
    auto pos_at = [&](int r) {
        const int c = by_head ? block : block * RPW + r;
        return ALL ? min(c, bt.n_pos - 1) : c;
    };
    auto head_at = [&](int it, int r) {
        const int h = h0 + it * step + (by_head ? r : 0);
        return ALL && by_head ? min(h, n_heads - 1) : h;
    };
    const int cp = pos_at(sub);
    const bool here = cp < bt.n_pos;
    const int64_t x_head = P.x_head, x_step = step * x_head;
    const T * const x_base = (const T *) Q.x[pi] + (int64_t) cp * P.x_pos, * x_row = x_base + head_at(0, sub) * x_head;
    Raw<T> raw = {};
    if (ALL || (here && head_at(0, sub) < n_heads)) load_row<T, ALL>(raw, x_row, e0, D);

    const float * norm = P.w;
    const int64_t norm_head = P.w_head;
    float cs[8] = {}, sn[8] = {}, w[8];
    auto load_w = [&](int h) {
        const float * p = norm + h * norm_head;
#pragma unroll
        for (int m = 0; m < 8; ++m) w[m] = ALL || e0 + m < D ? p[e0 + m] : 0.0f;
#pragma unroll
        for (int m = 0; m < 8; ++m) asm volatile("" : "+v"(w[m]));         // waited for here, not where they are used
    };
    if (norm) load_w(norm_head && head_at(0, sub) < n_heads ? head_at(0, sub) : 0);
    const int n_rot = bt.n_rot, half = n_rot / 2;
    const bool pairs = bt.layout == SJK_ROPE_PAIRS, whole = KIND == HK_WHOLE || n_rot == 8 * LPR;
    // HK_PART: the lane of the other halves' channels; behind n_rot the lane itself
    const int pair_lane = sub * LPR + (e0 < half ? l + half / 8 : e0 < n_rot ? l - half / 8 : l);
    if (rope && here) {
        const double p = Q.pos ? (double) Q.pos[cp] : (double) (pos0 + (uint32_t) cp);
        double t[8];                                       // all of the table's loads before the first turn
        if (pairs) {
#pragma unroll
            for (int m = 0; m < 4; ++m) t[m] = whole || e0 + 2 * m < n_rot ? bt.turns[(e0 >> 1) + m] : 0.0;
#pragma unroll
            for (int m = 0; m < 4; ++m) {
                turn(p * t[m], bt.mscale, bt.sine, sn[2 * m + 1], cs[2 * m]);
                cs[2 * m + 1] = cs[2 * m];
                sn[2 * m] = -sn[2 * m + 1];
            }
        } else if (whole) {
            const bool up = l >= LPR / 2;                  // the pairs' second channels
            float s[4], c[4];
#pragma unroll
            for (int m = 0; m < 4; ++m) t[m] = bt.turns[(up ? e0 - half + 4 : e0) + m];
#pragma unroll
            for (int m = 0; m < 4; ++m) turn(p * t[m], bt.mscale, bt.sine, s[m], c[m]);
#pragma unroll
            for (int m = 0; m < 4; ++m) {
                const float so = lane_xor<LPR / 2>(s[m], lane), co = lane_xor<LPR / 2>(c[m], lane);
                cs[m] = up ? co : c[m];
                cs[m + 4] = up ? c[m] : co;
                sn[m] = up ? so : -s[m];
                sn[m + 4] = up ? s[m] : -so;
            }
        } else if (KIND == HK_PART) {                      // the same with the pair's lane half / 8 away
            const bool up = e0 >= half, in = e0 < n_rot;
            float s[4], c[4];
#pragma unroll
            for (int m = 0; m < 4; ++m) t[m] = in ? bt.turns[(up ? e0 - half + 4 : e0) + m] : 0.0;
#pragma unroll
            for (int m = 0; m < 4; ++m) turn(p * t[m], bt.mscale, bt.sine, s[m], c[m]);
#pragma unroll
            for (int m = 0; m < 4; ++m) {
                const float so = __shfl(s[m], pair_lane, 64), co = __shfl(c[m], pair_lane, 64);
                cs[m] = up ? co : c[m];
                cs[m + 4] = up ? c[m] : co;
                sn[m] = up ? so : -s[m];
                sn[m + 4] = up ? s[m] : -so;
            }
        } else {
#pragma unroll
            for (int m = 0; m < 8; ++m) {
                const int e = e0 + m;
                t[m] = e < n_rot ? bt.turns[e < half ? e : e - half] : 0.0;
            }
#pragma unroll
            for (int m = 0; m < 8; ++m) {
                turn(p * t[m], bt.mscale, bt.sine, sn[m], cs[m]);
                if (e0 + m < half) sn[m] = -sn[m];
            }
        }
    }

    // Where the rows go, d_head bytes from head to head. A cache's entry of the position: sink, or the ring's slot. Rows of fp32
    // with ALL: a lane's 32 bytes go through LDS, so that a store takes 1 KB on end (16 bytes a lane 32 apart reach 3.7 TB/s);
    // d_row and d_row2 are of the first and the second KB's rows then.
    uint8_t * d_row, * d_row2 = nullptr;
    int64_t d_head;
    bool f16_row = MODE == HM_F16;
    const bool rows_out = MODE == HM_ROWS || P.kind == HP_ROWS;
    const int o_type = P.o_type;
    const bool swapped = ALL && rows_out && (MODE != HM_ROWS || o_type == SJK_F32);
    const int cpr = D / 4;                                 // 16-byte pieces of a row of fp32
    const int g1 = min(lane, RPW * cpr - 1), g2 = min(64 + lane, RPW * cpr - 1);
    const int r1 = swapped ? g1 / cpr : sub, r2 = swapped ? g2 / cpr : sub;
    if (rows_out) {
        const int64_t size = o_type == SJK_F32 ? 4 : 2;
        uint8_t * o = (uint8_t *) Q.o[pi];
        d_row = o + size * (int64_t) pos_at(r1) * P.o_pos;
        d_head = size * P.o_head;
        if (swapped) {
            d_row += 16 * (g1 - r1 * cpr);
            d_row2 = o + size * (int64_t) pos_at(r2) * P.o_pos + 16 * (g2 - r2 * cpr);
        }
    } else {
        const uint32_t pos = pos0 + (uint32_t) cp;
        const bool in_sink = pos < Q.S, sink_f16 = in_sink && bt.sink_type == SJKVARN_SINK_F16;
        const size_t side = sink_f16 ? 2 * (size_t) D : bt.stage_bytes, at = in_sink ? pos : (pos - Q.S) % Q.cap;
        d_row = (uint8_t *) (in_sink ? Q.o[1] : Q.o[2]) + at * bt.H * 2 * side + (P.kind == HP_V ? side : 0);
        d_head = (int64_t) (2 * side);
        f16_row |= sink_f16;
    }
    uint8_t * const d_base = d_row, * const d_base2 = d_row2;
    d_row += head_at(0, r1) * d_head;
    d_row2 += head_at(0, r2) * d_head;
    const int64_t d_step = step * d_head;

    const float inv_D = bt.inv_D, eps = P.eps, rot_scale = bt.rot_scale;
    // what the rows become: fp32, halves, or the cache's entries (stores of one kind only, for the same reason as ALL)
    auto heads = [&](auto out) {
        constexpr int OUT = decltype(out)::value;
        constexpr bool TQ = OUT == HO_CACHE && MODE == HM_TQ6;
        uint64_t nf_batch = 0;                                 // tq6_0: the heads collected for a walk
        int xn_batch = 0;
        for (int it = 0; it < iters; ++it) {
            float * const tmp = TQ ? buf + it % TB * (4 * BS) : buf;
            const bool live = ALL || (here && head_at(it, sub) < n_heads);
            float x[8];
#pragma unroll
            for (int m = 0; m < 8; ++m) x[m] = raw_at<T>(raw, m);
            uint8_t * d1 = d_row, * d2 = d_row2;
            if (uneven) {                                      // (a last iteration with fewer heads than rows)
                x_row = x_base + head_at(min(it + 1, iters - 1), sub) * x_head;
                d_row = d_base + head_at(it + 1, r1) * d_head;
                d_row2 = d_base2 + head_at(it + 1, r2) * d_head;
            } else {
                if (it + 1 < iters) x_row += x_step;           // (the last iteration of ALL loads its own rows again)
                d_row += d_step;
                d_row2 += d_step;
            }
            if (ALL || (it + 1 < iters && here && head_at(it + 1, sub) < n_heads)) load_row<T, ALL>(raw, x_row, e0, D);

            if (norm) {
                if (KIND != HK_WHOLE && norm_head && it && live) load_w(head_at(it, sub));
                float ss = (__builtin_fmaf(x[1], x[1], x[0] * x[0]) + __builtin_fmaf(x[3], x[3], x[2] * x[2])) +
                           (__builtin_fmaf(x[5], x[5], x[4] * x[4]) + __builtin_fmaf(x[7], x[7], x[6] * x[6]));
                if (again) ss = 0.0f;
                ss += lane_xor<1>(ss, lane);
                ss += lane_xor<2>(ss, lane);
                ss += lane_xor<4>(ss, lane);
                if constexpr (LPR > 8) ss += lane_xor<8>(ss, lane);
                if constexpr (LPR > 16) ss += lane_xor<16>(ss, lane);
                if constexpr (LPR > 32) ss += lane_xor<32>(ss, lane);
                const float r = __builtin_amdgcn_rsqf(__builtin_fmaf(ss, inv_D, eps));      // within an ulp; eps keeps it normal
#pragma unroll
                for (int m = 0; m < 8; ++m) x[m] = x[m] * r * w[m];
            }

            if (rope) {
                float y[8];                                    // the other channel of each pair
                if (pairs) {
#pragma unroll
                    for (int m = 0; m < 8; ++m) y[m] = x[m ^ 1];
                } else if (whole) {
#pragma unroll
                    for (int m = 0; m < 8; ++m) y[m] = lane_xor<LPR / 2>(x[m], lane);
                } else if (KIND == HK_PART) {
#pragma unroll
                    for (int m = 0; m < 8; ++m) y[m] = __shfl(x[m], pair_lane, 64);
                } else {
                    // channel e in slot (e % 8) * 64 + sub * LPR + e / 8: both sides touch neighbouring words
                    wave_sync();
#pragma unroll
                    for (int m = 0; m < 8; ++m) tmp[m * 64 + lane] = x[m];
                    wave_sync();
#pragma unroll
                    for (int m = 0; m < 8; ++m) {
                        const int e = e0 + m, pe = e < half ? e + half : e < n_rot ? e - half : e;
                        y[m] = tmp[(pe & 7) * 64 + sub * LPR + (pe >> 3)];
                    }
                    wave_sync();
                }
                if (whole) {
#pragma unroll
                    for (int m = 0; m < 8; ++m) x[m] = __builtin_fmaf(x[m], cs[m], y[m] * sn[m]);
                } else {
#pragma unroll
                    for (int m = 0; m < 8; ++m)
                        if (e0 + m < n_rot) x[m] = __builtin_fmaf(x[m], cs[m], y[m] * sn[m]);
                }
            }

            // A row holding an infinity or a NaN takes the rotation and the tq6_0 sums with the host's NaN rule. Every value of
            // its rotation is an infinity or a NaN then, so a look at one of each lane's finds it. A row that overflows on the
            // way keeps the plain rotation, but where that makes NaNs their signs are hadamard_row's.
            uint64_t nf_rows = 0;
            bool xn = false;
            auto look = [&](const float (&v)[8]) {
                bool nf = false;
#pragma unroll
                for (int m = 0; m < 8; ++m) nf |= nonfinite(v[m]);
                nf_rows = __ballot(nf && live);
                xn = ((LPR == 64 ? nf_rows : nf_rows >> (sub * LPR)) & ((LPR == 64 ? 0 : 1ull << (LPR % 64)) - 1ull)) != 0;
            };
            bool nan = true;                                   // whether the rows may hold NaNs (wave-uniform)
            if (rot) {
                float y[8];
#pragma unroll
                for (int m = 0; m < 8; ++m) y[m] = x[m];
                hadamard_finite<8, LPR>(y, lane, rot_scale);
                uint64_t bad = __builtin_amdgcn_ballot_w64(nonfinite(y[0]));
#pragma unroll
                for (int m = 0; m < 8; m += 2) bad |= __builtin_amdgcn_ballot_w64(__builtin_isunordered(y[m], y[m + 1]));
                nan = (bad & (ALL ? ~0ull : __builtin_amdgcn_ballot_w64(live))) != 0;
                if (nan) {
                    look(x);
                    hadamard_rows_x<LPR>(x, tmp, lane, rot_scale, xn);
                } else {
#pragma unroll
                    for (int m = 0; m < 8; ++m) x[m] = y[m];
                }
            } else if (OUT == HO_CACHE && MODE == HM_TQ6) {
                look(x);
            }

            if constexpr (OUT == HO_F32) {
                if constexpr (ALL) {
                    float4 * t = (float4 *) buf;
                    wave_sync();
                    t[sub * cpr + 2 * l] = float4{x[0], x[1], x[2], x[3]};
                    t[sub * cpr + 2 * l + 1] = float4{x[4], x[5], x[6], x[7]};
                    wave_sync();
                    *(float4 *) d1 = t[g1];
                    *(float4 *) d2 = t[g2];
                } else if (live) {
#pragma unroll
                    for (int m = 0; m < 8; ++m) if (e0 + m < D) ((float *) d1)[e0 + m] = x[m];
                }
            } else {
                uint32_t h[4];
                if (OUT == HO_CACHE || o_type == SJK_F16) {
#pragma unroll
                    for (int m = 0; m < 4; ++m) h[m] = pack_f16(x[2 * m], x[2 * m + 1]);
                } else {
#pragma unroll
                    for (int m = 0; m < 4; ++m) h[m] = pack_bf16(x[2 * m], x[2 * m + 1]);
                }
                if (OUT == HO_CACHE && nan) {                  // a NaN is stored as its sign | 0x7E00 (f32_to_f16)
#pragma unroll
                    for (int m = 0; m < 4; ++m) h[m] = (uint32_t) f32_to_f16(x[2 * m]) | (uint32_t) f32_to_f16(x[2 * m + 1]) << 16;
                }
                if (live && (OUT == HO_HALF || f16_row)) store_halves<ALL>((uint16_t *) d1 + e0, h, e0, D);
                if constexpr (TQ) {
                    // sj_kvarn.h:1221-1247: two sums of 128 values in index order. The blocks of up to TQ_BATCH heads are
                    // collected in LDS and walked at once, 4 of a block's 16 lanes a head (4,096 positions of 32 + 8 heads of
                    // 128 take 36.9 us, 39.4 with a walk a head, whose 16 lanes did the same; 16 + 4 heads of 256 39.8 for 45.8).
                    if (!__any(!f16_row)) continue;
                    const int j = it % TB;
                    float * const blk = buf + (lane >> 4) * BS, * const own = blk + 8 * (lane & 15);
                    wave_sync();
                    *(float4 *) (own + j * (4 * BS)) = float4{x[0], x[1], x[2], x[3]};
                    *(float4 *) (own + j * (4 * BS) + 4) = float4{x[4], x[5], x[6], x[7]};
                    nf_batch |= nf_rows;
                    xn_batch |= (int) xn << j;
                    if (j < TB - 1 && it < iters - 1) continue;
                    wave_sync();
                    const int jw = min((lane & 15) / (16 / TB), j);            // the head this lane walks
                    const float * const row = blk + jw * (4 * BS);
                    const bool xnw = xn_batch >> jw & 1;
                    const float nsq = nf_batch ? walk<true, true>(row, xnw) : walk<false, true, UNROLL>(row);
                    const float norm = nsq != nsq ? nan_of(nsq) : __builtin_sqrtf(nsq);
                    const float inv = norm > 1e-10f ? 1.0f / norm : 0.0f;
                    wave_sync();
#pragma unroll 1
                    for (int i = 0; i <= j; ++i) {
                        float * const o4 = own + i * (4 * BS);
                        const float4 a = *(const float4 *) o4, b = *(const float4 *) (o4 + 4);
                        const float z[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
                        const int from = (lane & 48) + i * (16 / TB);
                        const float inv_i = __shfl(inv, from, 64);
                        const bool big = __shfl(norm, from, 64) > 1e-10f;
                        uint32_t qs = 0, qh = 0;               // low nibbles; high pairs
                        float c2[8];
#pragma unroll
                        for (int m = 0; m < 8; ++m) {
                            const float v = big ? z[m] * inv_i : 0.0f;
                            const int code = level_of(v, s_cell);
                            const float c = s_cent[code];
                            c2[m] = c * c;
                            qs |= (uint32_t) (code & 15) << (4 * m);
                            qh |= (uint32_t) ((code >> 4) & 3) << (2 * m);
                        }
                        *(float4 *) o4 = float4{c2[0], c2[1], c2[2], c2[3]};
                        *(float4 *) (o4 + 4) = float4{c2[4], c2[5], c2[6], c2[7]};
                        const int h = head_at(it - j + i, sub);
                        if (!f16_row && (ALL || (here && h < n_heads))) {
                            uint8_t * o = d_base + h * d_head + (size_t) (l >> 4) * SJKVARN_TQ6_BLOCK_BYTES;
                            const int i0 = 8 * (l & 15);
                            *(uint16_t *) (o + 2 + i0 / 2) = (uint16_t) qs;
                            *(uint16_t *) (o + 4 + i0 / 2) = (uint16_t) (qs >> 16);
                            *(uint16_t *) (o + 66 + i0 / 4) = (uint16_t) qh;
                        }
                    }
                    wave_sync();
                    const float rn = __builtin_sqrtf(walk<false, false, UNROLL>(row));
                    const int h = head_at(it - j + jw, sub);
                    if (!f16_row && (lane & 15) % (16 / TB) == 0 && (ALL || (here && h < n_heads)))
                        *(uint16_t *) (d_base + h * d_head + (size_t) (l >> 4) * SJKVARN_TQ6_BLOCK_BYTES) =
                            f32_to_f16(rn > 1e-10f ? xdiv(norm, rn) : norm);
                    nf_batch = 0;
                    xn_batch = 0;
                }
            }
        }
    };
    if (!rows_out) heads(Int<MODE == HM_ROWS ? HO_F32 : HO_CACHE>());
    else if (MODE != HM_ROWS || o_type == SJK_F32) heads(Int<HO_F32>());
    else heads(Int<HO_HALF>());
}

static size_t elem_size(int type) { return type == SJK_F32 ? 4 : 2; }
static bool type_ok(int type) { return type == SJK_F32 || type == SJK_F16 || type == SJK_BF16; }
// rows at p with strides in elements of `size` bytes can be read and written 16 bytes at a time
static bool wide_rows(const void * p, int64_t pos, int64_t head, size_t size, int D) {
    return D % 8 == 0 && !((uintptr_t) p & 15u) && !((uint64_t) pos * size & 15u) && !((uint64_t) head * size & 15u);
}

static int rope_ok(const sjk_hip_rope & r, int D) {
    if (r.n_rot == 0) return 0;
    if ((r.layout != SJK_ROPE_HALVES && r.layout != SJK_ROPE_PAIRS) || r.n_rot < 0 || r.n_rot > D || r.n_rot % 2)
        return refuse("rotary positions: a layout of SJK_ROPE_HALVES or _PAIRS and an even n_rot up to the head's width");
    if (!r.d_turns || (uintptr_t) r.d_turns % 8 || !__builtin_isfinite(r.mscale))
        return refuse("rotary positions: a table of turns (device, 8-byte aligned) and a finite mscale");
    return 0;
}

static int norm_ok(const float * w, float eps) {
    if (!w) return 0;
    if ((uintptr_t) w % 4 || !(eps >= 1.17549435e-38f) || !__builtin_isfinite(eps))
        return refuse("head norms: fp32 weights and a finite, normal eps > 0");
    return 0;
}

static void set_rope(HeadBatch & bt, const sjk_hip_rope & r) {
    bt.layout = r.layout;
    bt.n_rot = r.n_rot;
    bt.turns = r.d_turns;
    bt.mscale = r.mscale;
    bt.sine = r.inverse ? -1.0f : 1.0f;
}

template <typename T, int KIND>
static int launch_kind(const HeadBatch & bt, int lpr, int mode, unsigned grid, hipStream_t st) {
    const dim3 g(grid), b(64 * HW);
#define SJK_HEADS(L, M) hipLaunchKernelGGL((heads_kernel<T, L, M, KIND>), g, b, 0, st, bt)
    if (mode == HM_ROWS) {
        if (lpr == 8) SJK_HEADS(8, HM_ROWS);
        else if (lpr == 16) SJK_HEADS(16, HM_ROWS);
        else if (lpr == 32) SJK_HEADS(32, HM_ROWS);
        else SJK_HEADS(64, HM_ROWS);
    } else if (mode == HM_F16) {
        if (lpr == 16) SJK_HEADS(16, HM_F16);
        else SJK_HEADS(32, HM_F16);
    } else {
        if (lpr == 16) SJK_HEADS(16, HM_TQ6);
        else SJK_HEADS(32, HM_TQ6);
    }
#undef SJK_HEADS
    return SJK_CHECK_LAUNCH();
}

template <typename T>
static int launch_typed(const HeadBatch & bt, int lpr, int mode, bool wide, unsigned grid, hipStream_t st) {
    bool turned = false, weights = false;
    for (int p = 0; p < bt.n_parts; ++p) {
        turned |= (bt.part[p].flags & HF_ROPE) != 0;
        weights |= bt.part[p].w && bt.part[p].w_head;
    }
    if (!wide) return launch_kind<T, HK_ANY>(bt, lpr, mode, grid, st);
    if (turned && bt.layout == SJK_ROPE_HALVES && bt.n_rot % 16) return launch_kind<T, HK_ODD>(bt, lpr, mode, grid, st);
    if (bt.D != 8 * lpr || weights || (turned && bt.n_rot != 8 * lpr)) return launch_kind<T, HK_PART>(bt, lpr, mode, grid, st);
    return launch_kind<T, HK_WHOLE>(bt, lpr, mode, grid, st);
}

// the table from position n on
static void skip_positions(HeadBatch & bt, int n, size_t size) {
    bt.n_pos -= n;
    for (int k = 0; k < bt.n_seqs; ++k) {
        HeadSeq & Q = bt.seq[k];
        for (int p = 0; p < bt.n_parts; ++p) {
            const HeadPart & P = bt.part[p];
            if (!P.n_heads) continue;
            Q.x[p] = (const uint8_t *) Q.x[p] + n * P.x_pos * (int64_t) size;
            if (P.kind == HP_ROWS) Q.o[p] = (uint8_t *) Q.o[p] + n * P.o_pos * (int64_t) elem_size(P.o_type);
        }
        Q.pos0 += (uint32_t) n;
        if (Q.pos) Q.pos += n;
    }
}

// wavefronts of a launch, which has fewer than 2^32 threads
constexpr int64_t MAX_WAVES = 0xffffffffll / (64 * HW) * HW;

// The launch's shape. A wavefront goes through as many heads, up to HEAD_ITERS, as it takes for all wavefronts to be on the
// device at once (the sines and cosines of a position serve its heads): a second, partly filled round of them costs a
// 512-position append 7.1 -> 8.5 us, 1,237 positions x 64 heads of 80 10.8 -> 12.1. 16 wavefronts a CU are counted on, which the
// kernels for whole turns are bound to. 24 of the others have the registers for 12 (most HK_ODD ones from fp32 and fp16 rows; to
// tq6_0 HK_ODD, HK_ANY, and HK_PART but for 16-bit rows of 128; HK_ODD of fp32 rows of 256 for 8): their calls of 12 to 16 a CU
// take a second round all the same.
// A wavefront's rows are adjacent positions, except in calls of fewer positions than that, and where rows of fp32 go out: those of
// one position lie on end, and stores of 2 KB reach 5.0 TB/s where four of 512 bytes reach 4.6. (Rows of 16 bits: 4.5 by head,
// 4.9 by position, whose sines also serve more heads.)
static int launch_heads(HeadBatch & bt, int type, int mode, bool wide, hipStream_t st) {
    const int lpr = bt.D <= 64 ? 8 : bt.D <= 128 ? 16 : bt.D <= 256 ? 32 : 64, rpw = 64 / lpr;
    int64_t blocks[HEAD_PARTS];
    int step[HEAD_PARTS];
    for (int p = 0; p < bt.n_parts; ++p) {
        HeadPart & P = bt.part[p];
        const bool by_head = bt.n_pos < rpw || (P.kind == HP_ROWS && P.o_type == SJK_F32 && P.n_heads % rpw == 0);
        P.flags = by_head ? P.flags | HF_BY_HEAD : P.flags & ~HF_BY_HEAD;
        step[p] = by_head ? rpw : 1;                                       // heads an iteration takes on
        blocks[p] = by_head ? bt.n_pos : (bt.n_pos + rpw - 1) / rpw;
    }
    // staging tq6_0 rows takes longer than a query: half as many of them a wavefront, where all are on the device at once
    // (512 positions of 32 + 8 heads 9.7 -> 9.3 us, 2,048 21.0 -> 18.8; 4,096, in several rounds, 37.4 -> 37.9)
    int64_t waves = 0;
    auto shape = [&](int most, int most_tq) {
        bt.units = 0;
        for (int p = 0; p < bt.n_parts; ++p) {
            HeadPart & P = bt.part[p];
            const int steps = (P.n_heads + step[p] - 1) / step[p], run = mode == HM_TQ6 && P.kind != HP_ROWS ? most_tq : most;
            P.n_chunks = (steps + run - 1) / run;
            P.n_iters = P.n_chunks ? (steps + P.n_chunks - 1) / P.n_chunks : 0;
            P.n_units = (int) (blocks[p] * P.n_chunks);
            bt.units += P.n_units;
        }
        waves = (int64_t) bt.units * bt.n_seqs;
        return waves <= (int64_t) n_cus() * 4 * HW;
    };
    int most = 1;
    while (most <= HEAD_ITERS && !shape(most, (most + 1) / 2)) ++most;
    if (most > HEAD_ITERS) shape(HEAD_ITERS, HEAD_ITERS);
    if (!waves) return 0;
    if (waves > MAX_WAVES) {                               // (8 channels of one head: from 2^29 positions on)
        // a descriptor's position is the launch's first: with an offset of its own the kernels take 3 to 6% more (8 positions x
        // 40 heads 4.6 -> 4.8 us, 2,048 positions appended with a part turned 16.0 -> 17.0)
        if (bt.desc || bt.n_pos <= 8) return refuse("head rows: more rows than a launch holds");
        const int n = (bt.n_pos / 2 + 7) & ~7;
        HeadBatch first = bt;
        first.n_pos = n;
        const int rc = launch_heads(first, type, mode, wide, st);
        if (rc) return rc;
        skip_positions(bt, n, elem_size(type));
        return launch_heads(bt, type, mode, wide, st);
    }
    bt.inv_D = 1.0f / (float) bt.D;
    bt.rot_scale = rot_scale(bt.D);
    const unsigned grid = (unsigned) ((waves + HW - 1) / HW);
    if (type == SJK_F32) return launch_typed<float>(bt, lpr, mode, wide, grid, st);
    if (type == SJK_F16) return launch_typed<_Float16>(bt, lpr, mode, wide, grid, st);
    return launch_typed<__bf16>(bt, lpr, mode, wide, grid, st);
}

// rows of a sequence are counted in 32 bits
static bool rows_fit(uint64_t n_pos, uint64_t heads) { return n_pos <= 0x7fffffffu && n_pos * heads < 0x7fffff00u; }

}  // namespace sjk

using namespace sjk;

extern "C" int sjk_hip_head_rows(const sjk_hip_head_job * jobs, int n_jobs, uint32_t n_pos, int D, const sjk_hip_rope * rope,
                                 uint32_t pos0, const int32_t * d_pos, void * stream) {
    if (n_jobs < 0 || (n_jobs > 0 && !jobs)) return SJKVARN_ERR_ARG;
    if (D < 1 || D > 512) return refuse("sjk_hip_head_rows: head widths 1 to 512");
    if (d_pos && (uintptr_t) d_pos % 4) return SJKVARN_ERR_ARG;
    uint64_t heads = 0;
    bool turned = false;
    for (int k = 0; k < n_jobs; ++k) {
        const sjk_hip_head_job & J = jobs[k];
        if (!J.d_x || !J.d_out || J.n_heads < 0 || !type_ok(J.x_type) || !type_ok(J.out_type)) return SJKVARN_ERR_ARG;
        if ((uintptr_t) J.d_x % elem_size(J.x_type) || (uintptr_t) J.d_out % elem_size(J.out_type)) return SJKVARN_ERR_ARG;
        int rc = norm_ok(J.d_norm, J.eps);
        if (!rc && J.rope) rc = rope ? rope_ok(*rope, D) : refuse("sjk_hip_head_rows: a job turns its rows and rope is NULL");
        if (rc) return rc;
        if (J.rotate && D != 64 && D != 128 && D != 256 && D != 512) {
            set_error("sjk_hip_head_rows: the rotation needs a head width of 64, 128, 256 or 512");
            return SJK_ERR_UNSUPPORTED;
        }
        heads += (uint64_t) J.n_heads;
        turned |= J.rope && rope->n_rot;
    }
    if (!rows_fit(n_pos, heads)) return refuse("sjk_hip_head_rows: 2^31 rows or more");
    if (turned && !d_pos && (uint64_t) pos0 + n_pos > 0xffffffffull) return refuse("sjk_hip_head_rows: positions past 2^32 - 2");
    for (int k0 = 0; k0 < n_jobs;) {
        HeadBatch bt = {};
        bt.n_pos = (int) n_pos;
        bt.D = D;
        bt.n_seqs = 1;
        bt.seq[0].pos = d_pos;
        bt.seq[0].pos0 = pos0;
        if (rope) set_rope(bt, *rope);
        int k = k0;
        bool wide = true;
        for (; k < n_jobs && k - k0 < HEAD_PARTS && jobs[k].x_type == jobs[k0].x_type; ++k) {
            const sjk_hip_head_job & J = jobs[k];
            HeadPart & P = bt.part[bt.n_parts];
            P.x_pos = J.x_pos; P.x_head = J.x_head; P.o_pos = J.out_pos; P.o_head = J.out_head;
            P.w = J.d_norm; P.w_head = J.norm_head; P.eps = J.eps;
            P.n_heads = J.n_heads; P.kind = HP_ROWS; P.o_type = J.out_type;
            P.flags = (J.rope && rope->n_rot ? HF_ROPE : 0) | (J.rotate ? HF_ROT : 0);
            if (J.n_heads)
                wide = wide && wide_rows(J.d_x, J.x_pos, J.x_head, elem_size(J.x_type), D) &&
                       wide_rows(J.d_out, J.out_pos, J.out_head, elem_size(J.out_type), D);
            bt.seq[0].x[bt.n_parts] = J.d_x;
            bt.seq[0].o[bt.n_parts] = J.d_out;
            if (J.n_heads) ++bt.n_parts;
        }
        const int rc = n_pos && bt.n_parts ? launch_heads(bt, jobs[k0].x_type, HM_ROWS, wide, (hipStream_t) stream) : 0;
        if (rc) return rc;
        k0 = k;
    }
    return 0;
}

namespace sjk {

int qkv_ok(const sjk_hip_view & v, const sjk_hip_qkv & m, uint32_t pos0, uint32_t n_pos, const int32_t * d_pos, const void * d_q,
           const void * d_k, const void * d_v, const float * d_q_out) {
    const int D = v.lay.D, H = v.n_head_kv;
    if (!d_k || !d_v || !v.sink || !v.ring || v.cap == 0 || H <= 0 || m.n_head < 0 || !type_ok(m.type)) return SJKVARN_ERR_ARG;
    if (m.n_head && (!d_q || !d_q_out)) return SJKVARN_ERR_ARG;
    if (D != 128 && D != 256) {
        set_error("sjk_hip_store_qkv: head_dim 128 or 256");
        return SJK_ERR_UNSUPPORTED;
    }
    if ((v.staging != SJKVARN_STAGING_TQ6_0 && v.staging != SJKVARN_STAGING_F16) ||
        v.stage_bytes != sj_kvarn_stage_row_bytes(v.staging, D) || (v.sink_type != SJKVARN_SINK_F16 && v.sink_type != SJKVARN_SINK_INHERIT))
        return SJKVARN_ERR_ARG;
    const size_t size = elem_size(m.type);
    if (((uintptr_t) d_k | (uintptr_t) d_v | (m.n_head ? (uintptr_t) d_q : 0)) % size || (uintptr_t) d_q_out % 4 ||
        (uintptr_t) d_pos % 4 || (((uintptr_t) v.sink | (uintptr_t) v.ring) & 1u))
        return SJKVARN_ERR_ARG;
    if ((uint64_t) pos0 + n_pos > 0xffffffffull) return refuse("sjk_hip_store_qkv: positions past 2^32 - 2");
    const uint64_t room = (uint64_t) v.cap + (pos0 < v.S ? v.S - pos0 : 0);
    if (n_pos > room) {
        set_error("sjk_hip_store_qkv: more positions than sink and ring hold at once");
        return SJKVARN_ERR_CAPACITY;
    }
    if (!rows_fit(n_pos, (uint64_t) m.n_head + 2u * (uint64_t) H)) return refuse("sjk_hip_store_qkv: 2^31 rows or more");
    int rc = norm_ok(m.n_head ? m.d_q_norm : nullptr, m.eps);
    if (!rc) rc = norm_ok(m.d_k_norm, m.eps);
    if (!rc) rc = rope_ok(m.rope, D);
    return rc;
}

// the launch's table without its sequences
static void qkv_table(HeadBatch & bt, const sjk_hip_view & v, const sjk_hip_qkv & m, uint32_t n_pos) {
    const int D = v.lay.D;
    bt.n_pos = (int) n_pos;
    bt.D = D;
    bt.n_parts = HEAD_PARTS;
    bt.H = v.n_head_kv;
    bt.sink_type = v.sink_type;
    bt.stage_bytes = v.stage_bytes;
    set_rope(bt, m.rope);
    const int qk = (m.rope.n_rot ? HF_ROPE : 0) | (m.rotate_qk ? HF_ROT : 0);
    const int64_t pos[3] = {m.q_pos, m.k_pos, m.v_pos}, head[3] = {m.q_head, m.k_head, m.v_head};
    const float * w[3] = {m.d_q_norm, m.d_k_norm, nullptr};
    for (int p = 0; p < HEAD_PARTS; ++p) {
        HeadPart & P = bt.part[p];
        P.x_pos = pos[p]; P.x_head = head[p];
        P.o_pos = (int64_t) m.n_head * D; P.o_head = D;
        P.w = w[p]; P.w_head = m.norm_head; P.eps = m.eps;
        P.n_heads = p ? v.n_head_kv : m.n_head;
        P.kind = p; P.o_type = SJK_F32;
        P.flags = p < 2 ? qk : m.rotate_v ? HF_ROT : 0;
    }
}

// one more sequence; whether its rows and its cache take 16-byte accesses
static bool qkv_seq(HeadBatch & bt, const sjk_hip_view & v, const sjk_hip_qkv & m, uint32_t pos0, const int32_t * d_pos, const void * d_q,
                    const void * d_k, const void * d_v, float * d_q_out) {
    HeadSeq & Q = bt.seq[bt.n_seqs++];
    const void * x[3] = {d_q, d_k, d_v};
    bool wide = !(((uintptr_t) v.sink | (uintptr_t) v.ring) & 15u) && wide_rows(d_q_out, 0, 0, 4, bt.D);
    for (int p = 0; p < HEAD_PARTS; ++p) {
        const HeadPart & P = bt.part[p];
        Q.x[p] = x[p];
        wide = wide && (P.n_heads == 0 || wide_rows(x[p], P.x_pos, P.x_head, elem_size(m.type), bt.D));
    }
    Q.o[0] = d_q_out; Q.o[1] = v.sink; Q.o[2] = v.ring;
    Q.pos = d_pos; Q.pos0 = pos0; Q.S = v.S; Q.cap = v.cap;
    return wide;
}

static int qkv_launch(HeadBatch & bt, const sjk_hip_view & v, int type, bool wide, hipStream_t st) {
    if (!bt.n_pos) return 0;
    return launch_heads(bt, type, v.staging == SJKVARN_STAGING_F16 ? HM_F16 : HM_TQ6, wide, st);
}

}  // namespace sjk

extern "C" int sjk_hip_store_qkv(const sjk_hip_view * v, uint32_t pos0, uint32_t n_pos, const sjk_hip_qkv * m, const int32_t * d_pos,
                                 const void * d_q, const void * d_k, const void * d_v, float * d_q_out, void * stream) {
    if (!v || !m) return SJKVARN_ERR_ARG;
    const int rc = qkv_ok(*v, *m, pos0, n_pos, d_pos, d_q, d_k, d_v, d_q_out);
    if (rc) return rc;
    HeadBatch bt = {};
    qkv_table(bt, *v, *m, n_pos);
    const bool wide = qkv_seq(bt, *v, *m, pos0, d_pos, d_q, d_k, d_v, d_q_out);
    return qkv_launch(bt, *v, m->type, wide, (hipStream_t) stream);
}

extern "C" int sjk_hip_store_qkv_dyn(const sjk_hip_view * v, const int32_t * d_desc, uint32_t n_pos, const sjk_hip_qkv * m,
                                     const int32_t * d_pos, const void * d_q, const void * d_k, const void * d_v, float * d_q_out,
                                     void * stream) {
    if (!v || !m || !d_desc) return SJKVARN_ERR_ARG;
    // the positions are not known here: as for one that starts behind the sink
    const int rc = qkv_ok(*v, *m, v->S, n_pos, d_pos, d_q, d_k, d_v, d_q_out);
    if (rc) return rc;
    HeadBatch bt = {};
    qkv_table(bt, *v, *m, n_pos);
    const bool wide = qkv_seq(bt, *v, *m, 0, d_pos, d_q, d_k, d_v, d_q_out);
    bt.desc = d_desc;
    return qkv_launch(bt, *v, m->type, wide, (hipStream_t) stream);
}

extern "C" int sjk_hip_store_qkv_batch(const sjk_hip_qkv_job * jobs, int n_jobs, uint32_t n_pos, const sjk_hip_qkv * m, void * stream) {
    if (n_jobs < 0 || (n_jobs > 0 && !jobs) || !m) return SJKVARN_ERR_ARG;
    for (int k = 0; k < n_jobs; ++k) {
        const sjk_hip_qkv_job & J = jobs[k];
        const int rc = J.v.lay.D != jobs[0].v.lay.D ? SJKVARN_ERR_ARG
                                                    : qkv_ok(J.v, *m, J.pos0, n_pos, J.d_pos, J.d_q, J.d_k, J.d_v, J.d_q_out);
        if (rc) return rc;
    }
    // two jobs on one ring could write one slot
    for (int k = 1; k < n_jobs; ++k)
        for (int i = 0; i < k; ++i)
            if (jobs[i].v.ring == jobs[k].v.ring) return refuse("sjk_hip_store_qkv_batch: two jobs on one ring");
    for (int k = 0; k < n_jobs;) {
        const sjk_hip_view & v = jobs[k].v;
        HeadBatch bt = {};
        bool wide = true;
        qkv_table(bt, v, *m, n_pos);
        for (; k < n_jobs && bt.n_seqs < HEAD_SEQS; ++k) {
            const sjk_hip_qkv_job & J = jobs[k];
            if (J.v.n_head_kv != v.n_head_kv || J.v.staging != v.staging || J.v.sink_type != v.sink_type) break;
            wide = qkv_seq(bt, J.v, *m, J.pos0, J.d_pos, J.d_q, J.d_k, J.d_v, J.d_q_out) && wide;
        }
        const int rc = qkv_launch(bt, v, m->type, wide, (hipStream_t) stream);
        if (rc) return rc;
    }
    return 0;
}
