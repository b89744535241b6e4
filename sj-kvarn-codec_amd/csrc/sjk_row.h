// sjk_row.h - what the row kernels share (sjk_rows.hip, sjk_heads.hip): a row of V * LPR values lies V consecutive
// values a lane in LPR adjacent lanes (a power of two), several rows in a wavefront where LPR < 64.
#pragma once
#include "sjk_dev.h"

namespace sjk {

// v of the lane that the DPP control names, in an arithmetic instruction's own operand where the compiler can put it there
// (every lane of these controls has a source, so nothing stands in for a missing one)
template <int CTRL> SJK_DEV float dpp_in(float v) {
    return __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), CTRL, 0xF, 0xF, true));
}

// v of lane l ^ LM. Inside a 16-lane row by DPP, across rows by row swaps: none of a lane shuffle's LDS round trips.
template <int LM> SJK_DEV float lane_xor(float v, int lane) {
    if constexpr (LM == 1) return dpp_in<0xB1>(v);                    // quad_perm 1 0 3 2
    else if constexpr (LM == 2) return dpp_in<0x4E>(v);               // quad_perm 2 3 0 1
    else if constexpr (LM == 4) return dpp_in<0x1B>(dpp_in<0x141>(v));// 7 - l (row_half_mirror), then quad_perm 3 2 1 0
    else if constexpr (LM == 8) return dpp_in<0x128>(v);              // row_ror 8
    else {
        uint32_t lo = f_bits(v), hi = lo;                             // the lower and the upper partner's value
        if constexpr (LM == 16) swap16(lo, hi);
        else swap32(lo, hi);
        return bits_f(lane & LM ? lo : hi);
    }
}

// Hadamard of one row of 64 V values (sj_kvarn.h:735-752): stages h < V inside the lane, stages h >= V between lanes l and
// l ^ (h / V) (the lower partner keeps a + b, the upper a - b, a = the lower value), then one multiply by 1/sqrt(64 V). XN: the
// host's NaN rule (a row holding an infinity or a NaN).
template <int V, bool XN>
SJK_DEV void hadamard_row(float (&x)[V], int lane, float scale) {
    auto add = [&](float a, float b) { return XN ? xadd(a, b) : a + b; };
    auto sub = [&](float a, float b) { return XN ? xsub(a, b) : a - b; };
#pragma unroll
    for (int h = 1; h < V; h *= 2)
#pragma unroll
        for (int m = 0; m < V; ++m)
            if (!(m & h)) {
                const float a = x[m], b = x[m + h];
                x[m] = add(a, b);
                x[m + h] = sub(a, b);
            }
    if (XN) {
#pragma unroll
        for (int lm = 1; lm < 64; lm *= 2) {
            const bool upper = (lane & lm) != 0;
#pragma unroll
            for (int m = 0; m < V; ++m) {
                const float o = __shfl_xor(x[m], lm, 64);
                x[m] = upper ? sub(o, x[m]) : add(x[m], o);
            }
        }
    } else {
        // appends of 8 rows at D = 256 4.5 -> 4.3 us, of 8,192 9.2 -> 8.7, fp16 rows 2.85 -> 2.63 and 5.1 -> 4.95, against
        // lane shuffles (six LDS round trips one after the other)
        auto stage = [&](int lm, auto && partner) {
            const bool upper = (lane & lm) != 0;
#pragma unroll
            for (int m = 0; m < V; ++m) {
                const float o = partner(x[m]);
                x[m] = upper ? o - x[m] : x[m] + o;
            }
        };
        stage(1, [&](float v) { return lane_xor<1>(v, lane); });
        stage(2, [&](float v) { return lane_xor<2>(v, lane); });
        stage(4, [&](float v) { return lane_xor<4>(v, lane); });
        stage(8, [&](float v) { return lane_xor<8>(v, lane); });
#pragma unroll
        for (int lm = 16; lm < 64; lm *= 2) {
            const bool upper = (lane & lm) != 0;
#pragma unroll
            for (int m = 0; m < V; ++m) {
                uint32_t lo = f_bits(x[m]), hi = lo;                    // the lower and the upper partner's value
                if (lm == 16) swap16(lo, hi);
                else swap32(lo, hi);
                const float p = bits_f(lo), q = bits_f(hi);
                x[m] = upper ? p - q : p + q;
            }
        }
    }
#pragma unroll
    for (int m = 0; m < V; ++m) x[m] = XN ? xmul(x[m], scale) : x[m] * scale;
}

// The same of a row of V * LPR values in LPR lanes, for rows whose result is finite: a stage across lanes is the lane's own value
// with its sign turned in the upper partner, added to the partner's value as the addition's DPP operand (two instructions a value
// for four).
// A NaN on the way may come out with another sign.
template <int V, int LPR> SJK_DEV void hadamard_finite(float (&x)[V], int lane, float scale) {
#pragma unroll
    for (int h = 1; h < V; h *= 2)
#pragma unroll
        for (int m = 0; m < V; ++m)
            if (!(m & h)) {
                const float a = x[m], b = x[m + h];
                x[m] = a + b;
                x[m + h] = a - b;
            }
    auto stage = [&](int lm, auto && partner) {
        const uint32_t flip = lane & lm ? 0x80000000u : 0u;
#pragma unroll
        for (int m = 0; m < V; ++m) x[m] = partner(x[m]) + bits_f(f_bits(x[m]) ^ flip);
    };
    if constexpr (LPR > 1) stage(1, [&](float v) { return lane_xor<1>(v, lane); });
    if constexpr (LPR > 2) stage(2, [&](float v) { return lane_xor<2>(v, lane); });
    if constexpr (LPR > 4) stage(4, [&](float v) { return lane_xor<4>(v, lane); });
    if constexpr (LPR > 8) stage(8, [&](float v) { return lane_xor<8>(v, lane); });
#pragma unroll
    for (int lm = 16; lm < LPR; lm *= 2) {
        const uint32_t flip = lane & lm ? 0x80000000u : 0u;
#pragma unroll
        for (int m = 0; m < V; ++m) {
            uint32_t lo = f_bits(x[m]), hi = lo;                        // the lower and the upper partner's value
            if (lm == 16) swap16(lo, hi);
            else swap32(lo, hi);
            x[m] = bits_f(lo) + bits_f(hi ^ flip);
        }
    }
#pragma unroll
    for (int m = 0; m < V; ++m) x[m] = x[m] * scale;
}

// the sum of 128 values (SQUARED: of their squares) in index order, UNROLL reads of four in flight; XN: the host's NaN rule where
// xn is set
template <bool XN, bool SQUARED = false, int UNROLL = 8> SJK_DEV float walk(const float * sq, bool xn = true) {
    const float4 * p = (const float4 *) sq;
    float s = 0.0f;
    if (XN) {
        auto add = [&](float a, float v) {
            const float b = SQUARED ? xn ? xmul(v, v) : v * v : v;
            return xn ? xadd(a, b) : a + b;
        };
        for (int i = 0; i < 32; ++i) {
            const float4 q = p[i];
            s = add(s, q.x); s = add(s, q.y); s = add(s, q.z); s = add(s, q.w);
        }
    } else {
        auto sq1 = [](float v) { return SQUARED ? v * v : v; };
#pragma unroll UNROLL
        for (int i = 0; i < 32; ++i) {
            const float4 q = p[i];
            s = s + sq1(q.x); s = s + sq1(q.y); s = s + sq1(q.z); s = s + sq1(q.w);
        }
    }
    return s;
}

inline float rot_scale(int D) { return 1.0f / __builtin_sqrtf((float) D); }

}  // namespace sjk
