// Kernels of the 8-bit KV cache's attention (include/rk_npu_attention_q8.h).
//
// Layout in HBM. Codes lie in the order in which the matrix cores take them, so
// that a wave's loads are whole lines and go from memory to operands without a
// transposition: a unit is 32 tokens of one KV head, 32 D bytes of K and of V,
//   K: [16-key half cb][64-dim step s][lane][16 B]: key 16 cb + lane % 16, dims
//      64 s + 8 (lane / 16)..+7, then the 8 dims 32 further on;
//   V: [32-dim step s][lane][16 B]: dim 32 s + lane % 16, then the dim 16 further
//      on, 8 keys each: 4 h..4 h + 3 and 16 + 4 h..+3 with h = lane / 16.
// i8 codes are stored plus 128. The scales are one float4 per block and head:
// K's scale, and V's as m 2^e with 1 <= m < 2: m, e (an int) and 1 / scale. A
// block of zeros has the smallest scale, of fp16's least value; a poisoned one (an
// infinity or NaN came) has NaN. The tail's fp16 rows lie in the same order with 8 values a lane and step.
//
// Operands of v_mfma_f32_16x16x32_f16: A lane l = row l % 16, k-slots
// 8 (l / 16)..+7; B lane l = column l % 16, the same slots; C lane l = rows
// 4 (l / 16)..+3 of column l % 16. S^T = K Q^T leaves lane l the scores of query
// row l % 16 for keys 4 (l / 16)..+3 of each 16, which is what B of
// O^T += V^T P^T wants once V's slots name the same keys, as above.
#pragma once

#include <hip/hip_fp16.h>
#include <hip/hip_runtime.h>

#include "../../include/rk_npu_attention_q8.h"
#include "kernels.hpp"

namespace hm {

constexpr int Q8_SLOTS = 3;  // fp16 blocks kept
constexpr int Q8_MAX_SPLITS = 256;  // key splits that a row's join takes

struct AttnQ8Params {
    const void* q;
    int q_f32;
    long long q_head, q_row;  // strides, elements
    void* out;
    int out_f16;
    long long o_head, o_row;
    const uint8_t* k;    // codes [kh][cap * D]
    const uint8_t* v;
    const float4* sc;    // [kh][cap / block]
    const __half* kt;    // the open block's fp16 rows [kh][block * D]
    const __half* vt;
    float* part;         // accumulators [kh][rows_pad][splits][D], then (max, sum) pairs
    int qh, kh, m, len, pos, causal;
    float scale;
    size_t head_bytes;   // cap * D
    int blocks;          // cap / block
    int unit_shift;      // log2(block / 32)
    int block_values;    // block * D
    int coded;           // keys below this are read as codes
    int units;           // 32-key units that some row sees
    int splits, units_per_split, row_tiles, rows_pad;
};

typedef _Float16 q8_h8 __attribute__((ext_vector_type(8)));
typedef _Float16 q8_h2 __attribute__((ext_vector_type(2)));
typedef float q8_f4 __attribute__((ext_vector_type(4)));

// 8 codes (two words) to 8 fp16, exactly. i8: a byte u = code + 128 under 0x64
// is the fp16 1024 + u. e4m3: the conversion instruction. (i8 without the subtraction, a
// byte under 0x00 as the fp16 u 2^-24 and 128 times the weights' sum taken off at the
// end: 512 rows of 8 heads over 8000 keys of 128 28.7 us instead of 30.9, but beside that
// offset the values of light keys are lost. With a key of no value 10 above the others'
// scores, outputs were 3 % off.)
template <int FMT>
__device__ __forceinline__ q8_h8 q8_halves(unsigned lo, unsigned hi) {
    unsigned w[4];
    if constexpr (FMT == RK_NPU_HIP_KV_I8) {
        const unsigned src[2] = {lo, hi};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const q8_h2 x = __builtin_bit_cast(
                q8_h2, __builtin_amdgcn_perm(0x64646464u, src[i >> 1], (i & 1) ? 0x04030402u : 0x04010400u));
            w[i] = __builtin_bit_cast(unsigned, x - q8_h2{(_Float16)1152.0f, (_Float16)1152.0f});
        }
    } else {
        w[0] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.0f, false));
        w[1] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.0f, true));
        w[2] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.0f, false));
        w[3] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.0f, true));
    }
    return __builtin_bit_cast(q8_h8, v4u{w[0], w[1], w[2], w[3]});
}

// Two f32 to fp16, once: without the empty asm the compiler folds the product
// before a rounding into it in one of the rounding's uses (a single rounding there,
// two in the others), and the remainder is then that of another value.
__device__ __forceinline__ q8_h2 q8_round2(float a, float b) {
    unsigned w = __builtin_bit_cast(unsigned, q8_h2{(_Float16)a, (_Float16)b});
    asm("" : "+v"(w));
    return __builtin_bit_cast(q8_h2, w);
}

// Max / sum over the 4 lanes of a query row (l % 16 + 16 j), in each of them: the
// swaps exchange odd with even 16-lane rows, then the wave's halves.
__device__ __forceinline__ float q8_rows4_max(float v) {
    const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
    const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ float q8_rows4_sum(float v) {
    const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(a[0]) + __uint_as_float(a[1]);
    const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}
// Min over each 16 lanes, in each of them.
__device__ __forceinline__ int q8_row_min(int v) {
    v = min(v, dpp_move<DPP_QUAD_XOR1>(v));
    v = min(v, dpp_move<DPP_QUAD_XOR2>(v));
    v = min(v, dpp_move<DPP_ROW_HALF_MIRROR>(v));
    return min(v, dpp_move<DPP_ROW_MIRROR>(v));
}

// 4 consecutive outputs of any alignment.
__device__ __forceinline__ void q8_store4(const AttnQ8Params& P, long long at, q8_f4 y) {
    typedef unsigned u8 __attribute__((ext_vector_type(2), aligned(2)));
    typedef float f16 __attribute__((ext_vector_type(4), aligned(4)));
    if (P.out_f16) {
        const unsigned short b0 = __half_as_ushort(__float2half_rn(y[0])), b1 = __half_as_ushort(__float2half_rn(y[1]));
        const unsigned short b2 = __half_as_ushort(__float2half_rn(y[2])), b3 = __half_as_ushort(__float2half_rn(y[3]));
        *reinterpret_cast<u8*>(static_cast<__half*>(P.out) + at) =
            u8{b0 | ((unsigned)b1 << 16), b2 | ((unsigned)b3 << 16)};
    } else {
        *reinterpret_cast<f16*>(static_cast<float*>(P.out) + at) = f16{y[0], y[1], y[2], y[3]};
    }
}

// A row's maximum before it has seen a key: finite, so that differences are no NaN.
constexpr float Q8_NONE = -1e30f;
// The weight 2^d of a partial result whose maximum lies d <= 0 below the row's:
// never 0, so that an infinite accumulator stays one (0 times it is NaN). A finite sum
// gains by that 2^-72 a key at most (2^15 the weight, 2^33 for the least V scale),
// where the row's is above 2^-5.
__device__ __forceinline__ float q8_weight(float m, float top) {
    return fmaxf(__builtin_amdgcn_exp2f(m - top), 0x1p-120f);
}

// A row's maximum moves when a score passes it by LAZY (powers of 2), to SHIFT below
// the score: weights lie below 2^15, the row's largest above 2^(SHIFT - 1) (SPLIT) or
// 2^SHIFT. More of fp16's range for the small ones costs more moves, which show where
// waves do not wait for memory: 1024 rows of 8 heads of 128 over 32768 keys, SPLIT with
// LAZY 8 198 us, with 4 207; one fp16 a weight with 8 145, with 6 146, with 4 153.
constexpr float q8_lazy(bool split, bool few) { return few ? 4.0f : split ? 8.0f : 6.0f; }
constexpr float q8_shift(bool split, bool few) { return (split ? 14.0f : 15.0f) - q8_lazy(split, few); }

// A wave's query rows, RW groups of 16 (lane l: row l % 16 of each): their key
// limits, queries, running maxima (less SHIFT), sums and accumulators (lane l:
// dims 16 n + 4 (l / 16)..+3).
//
// With c = scale log2(e) and a block's scales ks and vs = mu 2^e, a key's weight
// is kept as p = 2^(c ks s + e - m): e in the exponent gives the products p mu code
// of different blocks one unit, which fp16 operands need. The row's accumulators add
// p mu code, its sum p 2^-e; m is the running maximum, a whole number with SPLIT so
// that e - m is exact.
//
// p follows V's scale, not only the softmax weight, so a key of small values may be
// among the row's smallest p and hold the row's largest softmax weight: the sum takes
// p in f32, before any rounding. (The sum of the fp16 weights lost such keys: 17 % off
// where half of the weight had 2^-24 of the other half's scale.)
//
// SPLIT: p mu goes into the products as two fp16, 22 bits. Otherwise p mu goes in as
// one, mu in the exponent. fp16 has fewer bits below 2^-14, and 2^-25 is lost: a weight
// times scale is off by 2^-30 (FEW, or one fp16: 2^-34) of the row's largest at most.
template <int D, int RW, bool SPLIT, bool FEW = false>
struct Q8Wave {
    static constexpr int KS = D / 32, NB = D / 16;
    static constexpr float LAZY = q8_lazy(SPLIT, FEW), SHIFT = q8_shift(SPLIT, FEW);
    int lim[RW];
    int open, seen;  // keys below `open` every row sees, from `seen` on none
    q8_h8 qf[RW][KS];
    float mrun[RW], lsum[RW];
    q8_f4 o[RW][NB];

    // Rows r0 + 16 w + lane % 16 of KV head g. Rows from R on are computed as the
    // head's first row and not written. Every load of the queries comes before the
    // first use (one memory round trip).
    __device__ __forceinline__ void start(const AttnQ8Params& P, int g, int r0, int lo, int hi) {
        typedef unsigned u16 __attribute__((ext_vector_type(4), aligned(2)));
        typedef float f16 __attribute__((ext_vector_type(4), aligned(4)));
        const int G = P.qh / P.kh, R = G * P.m;
        open = 0x7fffffff;
        seen = 0;
        long long at[RW];
#pragma unroll
        for (int w = 0; w < RW; ++w) {
            const int rr = r0 + 16 * w + lo;
            const bool ok = rr < R;
            const int h = ok ? rr / P.m : 0, r = ok ? rr - h * P.m : 0;
            at[w] = (long long)(g * G + h) * P.q_head + r * P.q_row + 8 * hi;
            lim[w] = ok ? (P.causal ? min(P.len, P.pos + r + 1) : P.len) : 0;
            if (ok) {
                open = min(open, lim[w]);
                seen = max(seen, lim[w]);
            }
            mrun[w] = Q8_NONE;
            lsum[w] = 0.0f;
        }
        if (!P.q_f32) {
#pragma unroll
            for (int w = 0; w < RW; ++w)
#pragma unroll
                for (int s = 0; s < KS; ++s)
                    qf[w][s] = __builtin_bit_cast(
                        q8_h8, v4u(*reinterpret_cast<const u16*>(static_cast<const __half*>(P.q) + at[w] + 32 * s)));
        } else {
#pragma unroll
            for (int w = 0; w < RW; ++w) {
                f16 x[KS][2];
#pragma unroll
                for (int s = 0; s < KS; ++s)
#pragma unroll
                    for (int i = 0; i < 2; ++i)
                        x[s][i] = *reinterpret_cast<const f16*>(static_cast<const float*>(P.q) + at[w] + 32 * s + 4 * i);
#pragma unroll
                for (int s = 0; s < KS; ++s)
#pragma unroll
                    for (int i = 0; i < 8; ++i) qf[w][s][i] = (_Float16)x[s][i >> 2][i & 3];
            }
        }
        open = __builtin_amdgcn_readfirstlane(q8_row_min(open));
        seen = -__builtin_amdgcn_readfirstlane(q8_row_min(-seen));
    }

    // The accumulators: after start(), or by tail<FIRST>.
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int w = 0; w < RW; ++w)
#pragma unroll
            for (int n = 0; n < NB; ++n) o[w][n] = q8_f4{0.0f, 0.0f, 0.0f, 0.0f};
    }

    // What a unit's weights take from its scales. Without SPLIT, e + log2(mu) goes
    // into the exponent whole: what its rounding takes is far below fp16's. A NaN
    // scale (poison) makes cks NaN, so every weight of the block is.
    struct Unit {
        float cks, lg, mu, part;  // part: what a weight's sum is multiplied with
    };
    static __device__ __forceinline__ Unit unit(float c, float ks, float mu, int e, float inv) {
        const bool poison = ks != ks || mu != mu;
        Unit x;
        x.cks = poison ? NAN : fmaxf(c * ks, 0x1p-120f);
        x.mu = poison ? 1.0f : mu;
        x.lg = SPLIT ? (float)e : (float)e + __builtin_amdgcn_logf(x.mu);
        x.part = SPLIT ? __int_as_float((127 - e) << 23) : poison ? 1.0f : inv;  // 2^-e, 1 / (mu 2^e)
        return x;
    }
    // Masked scores become -inf; where there are some, those of a poisoned block
    // become NaN here. (`none`: every key is)
    __device__ __forceinline__ bool masked(int key0, bool none) const { return key0 + 32 > open || none; }
    __device__ __forceinline__ void mask(Unit& x, int key0, bool none, int hi, q8_f4 (&s)[RW][2]) const {
        const bool poison = x.cks != x.cks;
        x.cks = poison ? 1.0f : x.cks;
#pragma unroll
        for (int w = 0; w < RW; ++w)
#pragma unroll
            for (int cb = 0; cb < 2; ++cb)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const float y = poison ? NAN : s[w][cb][r];
                    s[w][cb][r] = none || key0 + 16 * cb + 4 * hi + r >= lim[w] ? -INFINITY : y;
                }
    }
    // The rows' largest scores of a unit, in the maxima's units, and whether one
    // passes its row's maximum by more than LAZY.
    __device__ __forceinline__ bool over(const Unit& x, const q8_f4 (&s)[RW][2], float (&top)[RW]) const {
        bool any = false;
#pragma unroll
        for (int w = 0; w < RW; ++w) {
            top[w] = __builtin_elementwise_maximum(
                __builtin_elementwise_maximum(__builtin_elementwise_maximum(s[w][0][0], s[w][0][1]),
                                              __builtin_elementwise_maximum(s[w][0][2], s[w][0][3])),
                __builtin_elementwise_maximum(__builtin_elementwise_maximum(s[w][1][0], s[w][1][1]),
                                              __builtin_elementwise_maximum(s[w][1][2], s[w][1][3])));
            top[w] = __builtin_fmaf(top[w], x.cks, x.lg);
            any |= top[w] > mrun[w] + (LAZY + SHIFT);
        }
        return any;
    }
    template <bool FIRST = false>
    __device__ __forceinline__ void raise(const float (&top)[RW]) {
#pragma unroll
        for (int w = 0; w < RW; ++w) {
            float tm = q8_rows4_max(top[w]);
            tm = (SPLIT ? __builtin_ceilf(tm) : tm) - SHIFT;
            float alpha = 1.0f;
            if (tm > mrun[w] + LAZY) {
                alpha = __builtin_amdgcn_exp2f(mrun[w] - tm);
                mrun[w] = tm;
            }
            if constexpr (FIRST) continue;
            lsum[w] *= alpha;
#pragma unroll
            for (int n = 0; n < NB; ++n) o[w][n] *= alpha;
        }
    }
    // Scores to weights ph (and pl), and the rows' sums.
    __device__ __forceinline__ void weigh(const Unit& x, const q8_f4 (&s)[RW][2], q8_h8 (&ph)[RW], q8_h8 (&pl)[RW]) {
#pragma unroll
        for (int w = 0; w < RW; ++w) {
            const float b = x.lg - mrun[w];
            float l[2] = {0.0f, 0.0f};
#pragma unroll
            for (int cb = 0; cb < 2; ++cb)
#pragma unroll
                for (int r = 0; r < 4; r += 2) {
                    const float p0 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[w][cb][r], x.cks, b));
                    const float p1 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[w][cb][r + 1], x.cks, b));
                    if constexpr (SPLIT) {
                        const float x0 = p0 * x.mu, x1 = p1 * x.mu;
                        const q8_h2 h = q8_round2(x0, x1);
                        const q8_h2 d = {(_Float16)(x0 - (float)h[0]), (_Float16)(x1 - (float)h[1])};
                        ph[w][4 * cb + r] = h[0];
                        ph[w][4 * cb + r + 1] = h[1];
                        pl[w][4 * cb + r] = d[0];
                        pl[w][4 * cb + r + 1] = d[1];
                    } else {
                        const q8_h2 h = q8_round2(p0, p1);
                        ph[w][4 * cb + r] = h[0];
                        ph[w][4 * cb + r + 1] = h[1];
                    }
                    l[cb] += p0 + p1;
                }
            lsum[w] = __builtin_fmaf(l[0] + l[1], x.part, lsum[w]);
        }
    }
    __device__ __forceinline__ void product(int n, q8_h8 a, const q8_h8 (&ph)[RW], const q8_h8 (&pl)[RW]) {
#pragma unroll
        for (int w = 0; w < RW; ++w) {
            o[w][n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, ph[w], o[w][n], 0, 0, 0);
            if constexpr (SPLIT) o[w][n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, pl[w], o[w][n], 0, 0, 0);
        }
    }

    // Unit u, one of the tail: fp16 rows in the codes' order. What is not finite in V
    // stays out of the products (0 times it is NaN, so masked keys would show); V's
    // exponents move so that its largest magnitude lies near the codes'. Returns
    // whether there is such a value: wild() then adds them to the rows that see them,
    // after the last change of a maximum (whatever the weights, which are positive).
    // FIRST: nothing came before, not clear() either. KEEP: one memory round trip for
    // all of K and V; heads of 256 whose accumulators are in use have no registers for
    // it and take V twice, a part at a time, for its magnitude and for the products.
    template <bool FIRST, bool KEEP>
    __device__ __forceinline__ bool tail(const AttnQ8Params& P, float c, int g, int u, int lane) {
        const int hi = lane >> 4;
        unsigned wild = 0;
        const size_t at = (size_t)g * P.block_values + (size_t)(u - (P.coded >> 5)) * (32 * D) + lane * 8;
        v4u k[2 * KS], v[KEEP ? NB : 1];
        auto v_at = [&](int n) { return *reinterpret_cast<const v4u*>(P.vt + at + n * 512); };
#pragma unroll
        for (int i = 0; i < 2 * KS; ++i) k[i] = *reinterpret_cast<const v4u*>(P.kt + at + i * 512);
        if constexpr (KEEP) {
#pragma unroll
            for (int n = 0; n < NB; ++n) v[n] = v_at(n);
        }
        q8_f4 s[RW][2];
#pragma unroll
        for (int w = 0; w < RW; ++w) s[w][0] = s[w][1] = q8_f4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int i = 0; i < 2 * KS; ++i)
#pragma unroll
            for (int w = 0; w < RW; ++w)
                s[w][i / KS] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(q8_h8, k[i]), qf[w][i % KS],
                                                                      s[w][i / KS], 0, 0, 0);
        // (what lies behind the last row is not the cache's)
        v4u held;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int key = (u << 5) + (i >> 1) * 16 + 4 * hi + (i & 1) * 2;
            held[i] = (key < P.len ? 0xFFFFu : 0u) | (key + 1 < P.len ? 0xFFFF0000u : 0u);
        }
        auto clean = [&](v4u x) {
            x &= held;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const unsigned wild0 = (x[i] & 0x7C00u) == 0x7C00u ? 0xFFFFu : 0u;
                const unsigned wild1 = (x[i] & 0x7C000000u) == 0x7C000000u ? 0xFFFF0000u : 0u;
                wild |= wild0 | wild1;
                x[i] &= ~(wild0 | wild1);
            }
            return x;
        };
        unsigned big = 0;
#pragma unroll(KEEP ? NB : 4)
        for (int n = 0; n < NB; ++n) {
            const v4u x = clean(KEEP ? v[KEEP ? n : 0] : v_at(n));
            if constexpr (KEEP) v[n] = x;
#pragma unroll
            for (int i = 0; i < 4; ++i) big = max(big, max(x[i] & 0x7FFFu, (x[i] >> 16) & 0x7FFFu));
        }
        const float top = wave_max(__half2float(__ushort_as_half((unsigned short)big)));
        const int e = top > 0.0f ? ((__float_as_int(top) >> 23) & 255) - 127 - 6 : -30;
        const float up = __int_as_float((127 - e) << 23);
        q8_h8 ph[RW], pl[RW];
        Unit x = unit(c, 1.0f, 1.0f, e, up);
        if (masked(u << 5, false)) mask(x, u << 5, false, hi, s);  // (uniform)
        float top1[RW];
        if (__builtin_amdgcn_ballot_w64(over(x, s, top1)) != 0) raise<FIRST>(top1);
        weigh(x, s, ph, pl);
        if constexpr (FIRST) clear();
#pragma unroll
        for (int n = 0; n < NB; ++n) {
            q8_h8 a = __builtin_bit_cast(q8_h8, KEEP ? v[KEEP ? n : 0] : clean(v_at(n)));
#pragma unroll
            for (int i = 0; i < 8; ++i) a[i] = (_Float16)((float)a[i] * up);
            product(n, a, ph, pl);
        }
        return __builtin_amdgcn_ballot_w64(wild != 0) != 0;
    }
    // The sums of a row's 4 lanes.
    __device__ __forceinline__ void sums() {
#pragma unroll
        for (int w = 0; w < RW; ++w) lsum[w] = q8_rows4_sum(lsum[w]);
    }
    __device__ __forceinline__ void wild(const AttnQ8Params& P, int g, int u, int u_end, int lane) {
        const int hi = lane >> 4, coded_units = P.coded >> 5;
#pragma unroll 1
        for (; u < u_end; ++u) {
            const __half* vt = P.vt + (size_t)g * P.block_values + (size_t)(u - coded_units) * (32 * D);
#pragma unroll 1
            for (int j = 0; j < 32; ++j) {
                const __half* at = vt + ((j >> 2) & 3) * 128 + (j >> 4) * 4 + (j & 3);  // (uniform)
#pragma unroll
                for (int n = 0; n < NB; ++n)
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const float x = __half2float((at + n * 512 + r * 8)[(unsigned)hi * 32]);
                        const float y = fabsf(x) < INFINITY ? 0.0f : x;
#pragma unroll
                        for (int w = 0; w < RW; ++w) o[w][n][r] += (u << 5) + j < lim[w] ? y : 0.0f;
                    }
            }
        }
    }
};

// Row rr of KV head g, dims 16 (n0 + n) + 4 hi..+3 for n < NB, one of PARTS calls
// for the row: divided by l and stored, or, with several splits, left as a partial.
template <int NB, int PARTS>
__device__ __forceinline__ void q8_finish(const AttnQ8Params& P, int g, int rr, int split, int hi, int n0, float m,
                                          float l, const q8_f4 (&o)[NB]) {
    constexpr int D = 16 * NB * PARTS;
    const int G = P.qh / P.kh;
    if (P.splits == 1) {
        const float il = 1.0f / l;
        const int h = rr / P.m;
        const long long at = (long long)(g * G + h) * P.o_head + (rr - h * P.m) * P.o_row + 16 * n0 + 4 * hi;
#pragma unroll
        for (int n = 0; n < NB; ++n) q8_store4(P, at + 16 * n, o[n] * il);
        return;
    }
    const size_t row = ((size_t)g * P.rows_pad + rr) * P.splits + split;
    float* acc = P.part + row * D + 16 * n0 + 4 * hi;
    float* ml = P.part + (size_t)P.kh * P.rows_pad * P.splits * D + row * 2;
#pragma unroll
    for (int n = 0; n < NB; ++n) *reinterpret_cast<q8_f4*>(acc + 16 * n) = o[n];
    if (hi == 0 && n0 == 0) *reinterpret_cast<float2*>(ml) = float2{m, l};
}

// The NW waves of a row tile meet: each leaves its accumulators in LDS (NW RW NB KiB)
// and its rows' (max, sum), and takes an NW-th of the tile's (row group, dims) pairs.
template <int D, int NW, int RW, class Wave>
__device__ __forceinline__ void q8_meet(const AttnQ8Params& P, const Wave& W, int g, int rt, int split,
                                        int wave, int lane, uint8_t* smem, float (&ml)[NW][RW][2][16]) {
    constexpr int NB = D / 16;
    const int lo = lane & 15, hi = lane >> 4, R = P.qh / P.kh * P.m;
#pragma unroll
    for (int w = 0; w < RW; ++w) {
#pragma unroll
        for (int n = 0; n < NB; ++n)
            *reinterpret_cast<q8_f4*>(smem + ((w * NB + n) * NW + wave) * 1024 + lane * 16) = W.o[w][n];
        if (hi == 0) {
            ml[wave][w][0][lo] = W.mrun[w];
            ml[wave][w][1][lo] = W.lsum[w];
        }
    }
    __syncthreads();
    // pairs of a wave, all of one row group (more waves than pairs: the first ones')
    constexpr int MINE = RW * NB >= NW ? RW * NB / NW : 1;
    static_assert(RW * NB % MINE == 0 && NB % MINE == 0, "pairs per wave");
    if (wave * MINE >= RW * NB) return;
    const int w = wave * MINE / NB, n0 = wave * MINE % NB;
    float top = Q8_NONE, l = 0.0f, m1[NW];
#pragma unroll
    for (int i = 0; i < NW; ++i) {
        m1[i] = ml[i][w][0][lo];
        top = fmaxf(top, m1[i]);
    }
    q8_f4 sum[MINE];
#pragma unroll
    for (int n = 0; n < MINE; ++n) sum[n] = q8_f4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int i = 0; i < NW; ++i) {
        // (a wave that saw no key holds zeros, one that saw NaN scores a NaN sum)
        const float b = q8_weight(m1[i], top), l1 = ml[i][w][1][lo];
        l += l1 != l1 ? l1 : l1 * b;
#pragma unroll
        for (int n = 0; n < MINE; ++n)
            sum[n] += *reinterpret_cast<const q8_f4*>(smem + ((w * NB + n0 + n) * NW + i) * 1024 + lane * 16) * b;
    }
    const int rr = (rt * RW + w) * 16 + lo;
    if (rr < R) q8_finish<MINE, NB / MINE>(P, g, rr, split, hi, n0, top, l, sum);
}

// Few rows. Block: NW waves over one tile of 16 RW query rows of one KV head; wave w
// takes units w, w + NW, .. of its split, so nothing is shared until the waves'
// partial (max, sum, accumulators) meet in LDS. A unit's codes go from memory into
// operand registers; the loads of the next unit are issued as soon as this one's are
// converted.
//
// Measured, the join included: one row of 32 heads over 8 of 128 and 131072 keys
// (268 MB) e4m3 45.8 us, i8 45.3: 5.9 TB/s (a large copy reads and writes 4.9). Over
// 3968 keys (8 MB) 7.5: there it is latency, a unit's load to its products, the waves'
// meeting and the join's launch. 512 rows of 8 heads over 4096 keys, fp16 output, 21.1:
// conversion and softmax, vector instructions that every 32 rows repeat, take a SIMD 64 %
// of its time and the products 24 %, mostly one after the other; 1024 rows of 2 heads of
// 256 over 2048 keys 16.6: 37 and 22 %, one wave a SIMD waits for its loads. The tail
// after the coded units, its loads a round trip of their own: one row of 16 heads over
// 2 of 256, 1000 keys 12.2 us instead of 11.0. The splits joined by their last block,
// in the same launch, lost to a launch of their own (8.6): 10.0 with the partials
// through atomics of agent scope, 30 behind a fence, which writes the L2 back. Blocks
// of 2 or 4 groups of waves with keys of their own and more rows each: 27 to 31 for the
// 512 rows.
template <int D, int NW, int RW, int FMT, bool SPLIT>
__global__ __launch_bounds__(64 * NW) void attn_q8_kernel(AttnQ8Params P) {
    constexpr int KP = D / 32;  // 16-byte pieces per lane, of K (and V)
    constexpr int RT = 16 * RW;
    __shared__ __attribute__((aligned(16))) uint8_t smem[NW * RW * (D / 16) * 1024];
    __shared__ float ml[NW][RW][2][16];
    const int g = blockIdx.x, rt = blockIdx.y, split = blockIdx.z;
    const int lane = threadIdx.x & 63, lo = lane & 15, hi = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const float c = fminf(P.scale * 1.4426950408889634f, 0x1.fffffep127f);
    const uint8_t* kbase = P.k + (size_t)g * P.head_bytes + lane * 16;
    const uint8_t* vbase = P.v + (size_t)g * P.head_bytes + lane * 16;
    const float4* sc = P.sc + (size_t)g * P.blocks;
    const int coded_units = P.coded >> 5;
    const int u_begin = split * P.units_per_split + wave;

    v4u kr[KP], vr[KP];
    auto load_k = [&](int u) {
        const uint8_t* p = kbase + (size_t)u * (32 * D);
#pragma unroll
        for (int i = 0; i < KP; ++i) kr[i] = *reinterpret_cast<const v4u*>(p + i * 1024);
    };
    auto load_v = [&](int u) {
        const uint8_t* p = vbase + (size_t)u * (32 * D);
#pragma unroll
        for (int i = 0; i < KP; ++i) vr[i] = *reinterpret_cast<const v4u*>(p + i * 1024);
    };
    float4 next = float4{1.0f, 1.0f, 0.0f, 1.0f};  // the next unit's scales
    auto first = [&] {
        if (u_begin >= coded_units) return;
        next = sc[u_begin >> P.unit_shift];
        load_k(u_begin);
        load_v(u_begin);
    };
    // A wave has one unit of the tail at most (4 units, NW waves). It comes first: its
    // loads and those of the first coded unit are one memory round trip, for which
    // heads of 256 have no registers.
    const int u_tail = u_begin + (max(coded_units - u_begin, 0) + NW - 1) / NW * NW;
    const bool late = D == 256 && u_tail < min((split + 1) * P.units_per_split, P.units);
    if (!late) first();
    Q8Wave<D, RW, SPLIT, RW == 1> W;
    W.start(P, g, rt * RT, lo, hi);
    const int u_end = min(min((split + 1) * P.units_per_split, P.units), (W.seen + 31) >> 5);
    const int coded_end = min(u_end, coded_units);
    bool wild = false;
    if (u_tail < u_end)
        wild = W.template tail<true, true>(P, c, g, u_tail, lane);
    else
        W.clear();
    if (late) first();
    for (int u = u_begin; u < coded_end; u += NW) {
        q8_f4 s[RW][2];
#pragma unroll
        for (int w = 0; w < RW; ++w) s[w][0] = s[w][1] = q8_f4{0.0f, 0.0f, 0.0f, 0.0f};
        const float4 x = next;
        const bool more = u + NW < coded_end;
        if (more) next = sc[(u + NW) >> P.unit_shift];
#pragma unroll
        for (int i = 0; i < KP; ++i) {
            const int cb = i / (D / 64), st = i % (D / 64);
            const q8_h8 a0 = q8_halves<FMT>(kr[i][0], kr[i][1]);
            const q8_h8 a1 = q8_halves<FMT>(kr[i][2], kr[i][3]);
#pragma unroll
            for (int w = 0; w < RW; ++w) {
                s[w][cb] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a0, W.qf[w][2 * st], s[w][cb], 0, 0, 0);
                s[w][cb] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a1, W.qf[w][2 * st + 1], s[w][cb], 0, 0, 0);
            }
        }
        if (more) load_k(u + NW);
        q8_h8 ph[RW], pl[RW];
        auto un = W.unit(c, x.x, x.y, __float_as_int(x.z), x.w);
        if (__builtin_expect(W.masked(u << 5, false), 0)) W.mask(un, u << 5, false, hi, s);  // (uniform)
        float top[RW];
        if (__builtin_expect(__builtin_amdgcn_ballot_w64(W.over(un, s, top)) != 0, 0)) W.raise(top);
        W.weigh(un, s, ph, pl);
#pragma unroll
        for (int i = 0; i < KP; ++i) {
            W.product(2 * i, q8_halves<FMT>(vr[i][0], vr[i][1]), ph, pl);
            W.product(2 * i + 1, q8_halves<FMT>(vr[i][2], vr[i][3]), ph, pl);
        }
        if (more) load_v(u + NW);
    }
    W.sums();
    if (wild) W.wild(P, g, u_tail, u_tail + 1, lane);
    q8_meet<D, NW, RW>(P, W, g, rt, split, wave, lane, smem, ml);
}

// Much work. Block: NW waves with RW groups of 16 rows each over one split; the codes
// of a stage of U units are converted once, by all threads, into fp16 fragments in
// LDS that every wave multiplies with its own rows (attn_q8_kernel converts a unit
// in every wave: 128 of some 250 vector instructions a unit of 32 rows).
//
// In step j a wave turns the scores of unit j into weights, computes those of unit
// j + 1 and multiplies V of unit j - 1: one straight piece of code in which matrix
// and vector instructions do not depend on each other. In stage t K of stage t + 2
// and V of stage t + U - 1 (codes in registers since U = 2: stage t - 1, U = 1:
// t - 2) are converted meanwhile; U + 1 stages of each are in LDS, with one barrier
// per stage.
//
// Measured: 1024 rows of 8 heads of 128 over 32768 keys 148 us with f16 output, 0.92
// PFLOP/s of a large matrix product's 1.29, 196 with f32 (half as many products more:
// V's with two fp16 for a weight). Matrix cores 43 % busy (f32 48), vector instructions
// 57 % of the time (59): the softmax of 16 scores a lane and unit holds back the products,
// whose operands come from LDS once for 32 rows. U = 1: 151 to 157. Matrix and vector
// instructions interleaved by scheduling groups: 162.
template <int D, int NW, int U, int RW, int FMT, bool SPLIT>
__global__ __launch_bounds__(64 * NW) void attn_q8_tile_kernel(AttnQ8Params P) {
    constexpr int KS = D / 32, NB = D / 16, NT = 64 * NW;
    constexpr int BUFS = U + 1;  // stages in LDS
    constexpr int UNIT = 64 * D, HALF = UNIT * U;  // bytes of a unit's, a stage's K (or V) fragments
    constexpr int PIECES = 2 * D * U;       // 16-byte code pieces of a stage's K (and V)
    constexpr int PT = (2 * PIECES + NT - 1) / NT;  // of both, per thread
    constexpr bool DEEP = U == 1;  // (codes two stages ahead)
    static_assert((U == 1 || U == 2) && PIECES % 64 == 0 && 2 * BUFS * HALF <= 144 * 1024, "stage shape");
    __shared__ __attribute__((aligned(16))) uint8_t smem[2 * BUFS * HALF];
    __shared__ float4 units[3][U];
    const int g = blockIdx.x, rt = blockIdx.y, split = blockIdx.z;
    const int R = P.qh / P.kh * P.m;
    const int tid = threadIdx.x, lane = tid & 63, lo = lane & 15, hi = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const float c = fminf(P.scale * 1.4426950408889634f, 0x1.fffffep127f);
    const uint8_t* kbase = P.k + (size_t)g * P.head_bytes;
    const uint8_t* vbase = P.v + (size_t)g * P.head_bytes;
    const float4* sc = P.sc + (size_t)g * P.blocks;
    const int coded_units = P.coded >> 5;
    const int u_begin = split * P.units_per_split;
    const int u_last = min((split + 1) * P.units_per_split, P.units);
    const int u_coded = min(u_last, coded_units);
    const int stages = (u_coded - u_begin + U - 1) / U;  // (0 or less: only the tail)

    // Pieces 0..PIECES - 1 of a thread's count are K of stage tk, the others V of
    // stage tv. (a unit past the split's coded ones: the last of these again, not
    // used)
    v4u raw[PT], raw1[PT];
    auto load = [&](v4u (&raw)[PT], int tk, int tv) {
#pragma unroll
        for (int i = 0; i < PT; ++i) {
            const int p = i * NT + tid, q = p % PIECES;
            const bool k = p < PIECES;  // (whole waves)
            const int unit = min(u_begin + (k ? tk : tv) * U + q / (2 * D), u_coded - 1);
            if (2 * PIECES % NT == 0 || p < 2 * PIECES)
                raw[i] = *reinterpret_cast<const v4u*>((k ? kbase : vbase) + (size_t)unit * (32 * D) + (q % (2 * D)) * 16);
        }
    };
    auto load_scale = [&](int t) {
        return tid < U ? sc[min(u_begin + t * U + tid, u_coded - 1) >> P.unit_shift] : float4{1.0f, 1.0f, 0.0f, 1.0f};
    };
    auto kbuf = [&](int t) { return smem + t % BUFS * HALF; };
    auto vbuf = [&](int t) { return smem + (BUFS + t % BUFS) * HALF; };
    // (piece p of 64 lanes: fragments 2 (p / 64) and the next)
    auto store = [&](const v4u (&raw)[PT], int tk, int tv) {
#pragma unroll
        for (int i = 0; i < PT; ++i) {
            const int p = i * NT + tid, q = p % PIECES;
            uint8_t* at = (p < PIECES ? kbuf(tk) : vbuf(tv)) + (q >> 6) * 2048 + (q & 63) * 16;
            if (2 * PIECES % NT == 0 || p < 2 * PIECES) {
                *reinterpret_cast<q8_h8*>(at) = q8_halves<FMT>(raw[i][0], raw[i][1]);
                *reinterpret_cast<q8_h8*>(at + 1024) = q8_halves<FMT>(raw[i][2], raw[i][3]);
            }
        }
    };

    typedef Q8Wave<D, RW, SPLIT> Wave;
    auto store_unit = [&](int t, const float4& s) {
        const typename Wave::Unit x = Wave::unit(c, s.x, s.y, __float_as_int(s.z), s.w);
        units[t % 3][tid] = float4{x.cks, x.lg, x.mu, x.part};
    };
    Wave W;
    float4 s0, s1;
    if (stages > 0) {
        load(raw, 0, 0);
        load(raw1, 1, 0);
        s0 = load_scale(0);
        s1 = load_scale(1);
    }
    W.start(P, g, (rt * NW + wave) * 16 * RW, lo, hi);
    W.clear();
    if (stages > 0) {
        // (V of stage 0 into the place of stage -1 too: finite, its weights are 0)
        store(raw, 0, BUFS - 1);
        store(raw1, 1, 0);
        if (tid < U) {
            store_unit(0, s0);
            store_unit(1, s1);
        }
        // In stage t: K of t + 2, and V of the first stage not there.
        constexpr int VA = U - 1;
        load(raw, 2, VA);
        s0 = load_scale(2);
        if constexpr (DEEP) {
            load(raw1, 3, 1);
            s1 = load_scale(3);
        }
        __syncthreads();
        // (unit j: j % U of stage j / U)
        auto scores = [&](q8_f4 (&s)[RW][2], int j) {
            const uint8_t* k = kbuf(j / U) + j % U * UNIT + lane * 16;
#pragma unroll
            for (int w = 0; w < RW; ++w) s[w][0] = s[w][1] = q8_f4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int i = 0; i < KS; ++i)
#pragma unroll
                for (int cb = 0; cb < 2; ++cb) {
                    const q8_h8 a = *reinterpret_cast<const q8_h8*>(k + (cb * KS + i) * 1024);
#pragma unroll
                    for (int w = 0; w < RW; ++w)
                        s[w][cb] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, W.qf[w][i], s[w][cb], 0, 0, 0);
                }
        };
        auto products = [&](int j, const q8_h8 (&ph)[RW], const q8_h8 (&pl)[RW]) {
            const uint8_t* v = (j < 0 ? vbuf(BUFS - 1) : vbuf(j / U) + j % U * UNIT) + lane * 16;
#pragma unroll
            for (int n = 0; n < NB; ++n) W.product(n, *reinterpret_cast<const q8_h8*>(v + n * 1024), ph, pl);
        };
        auto unit_of = [&](int j) {
            const float4 x = units[j / U % 3][j % U];
            return typename Wave::Unit{x.x, x.y, x.z, x.w};
        };
        // What a unit's scores need before they are weighed: masks, and whether a
        // maximum moves.
        auto look = [&](int j, typename Wave::Unit& x, q8_f4 (&s)[RW][2], float (&top)[RW]) {
            bool any = W.over(x, s, top);
            const int u = u_begin + j;
            if (__builtin_expect(W.masked(u << 5, u >= u_coded), 0)) {  // (uniform)
                W.mask(x, u << 5, u >= u_coded, hi, s);
                any = W.over(x, s, top);
            }
            return __builtin_amdgcn_ballot_w64(any) != 0;
        };
        typename Wave::Unit now = unit_of(0);
        float top[RW];
        q8_f4 sa[RW][2], sb[RW][2];
        q8_h8 pha[RW], pla[RW], phb[RW], plb[RW];
#pragma unroll
        for (int w = 0; w < RW; ++w) pha[w] = pla[w] = phb[w] = plb[w] = q8_h8{};
        scores(sa, 0);
        bool moves = look(0, now, sa, top);
        // One unit: s and (ph0, pl0) in, of this unit and the one before; sn and
        // (ph1, pl1) out, of the next and this one. A stage's first unit waits for
        // the stage and fills the next one.
        auto step = [&](int j, bool begins, v4u (&raw)[PT], float4& s0, q8_f4 (&s)[RW][2], q8_h8 (&ph0)[RW],
                        q8_h8 (&pl0)[RW], q8_f4 (&sn)[RW][2], q8_h8 (&ph1)[RW], q8_h8 (&pl1)[RW]) {
            if (begins) __syncthreads();
            if (__builtin_expect(moves, 0)) {  // (uniform)
                // (what waits to be added has the old maximum)
                products(j - 1, ph0, pl0);
#pragma unroll
                for (int w = 0; w < RW; ++w) ph0[w] = pl0[w] = q8_h8{};
                W.raise(top);
            }
            if (begins) {
                const int t = j / U;
                constexpr int AHEAD = DEEP ? 2 : 1;
                store(raw, t + 2, t + VA);
                if (tid < U) store_unit(t + 2, s0);
                load(raw, t + 2 + AHEAD, t + VA + AHEAD);
                s0 = load_scale(t + 2 + AHEAD);
            }
            typename Wave::Unit then = unit_of(j + 1);
            scores(sn, j + 1);
            W.weigh(now, s, ph1, pl1);
            products(j - 1, ph0, pl0);
            moves = look(j + 1, then, sn, top);
            now = then;
        };
        const int count = stages * U;
        for (int j = 0; j < count; j += 2) {
            step(j, true, raw, s0, sa, pha, pla, sb, phb, plb);
            if (U == 2 || j + 1 < count) {
                if constexpr (DEEP)
                    step(j + 1, true, raw1, s1, sb, phb, plb, sa, pha, pla);
                else
                    step(j + 1, U == 1, raw, s0, sb, phb, plb, sa, pha, pla);
            } else {
#pragma unroll
                for (int w = 0; w < RW; ++w) {
                    pha[w] = phb[w];
                    pla[w] = plb[w];
                }
            }
        }
        __syncthreads();
        products(count - 1, pha, pla);
    }
    const int t_begin = max(u_begin, coded_units), t_end = min(u_last, (W.seen + 31) >> 5);
    bool wild = false;
#pragma unroll 1
    for (int u = t_begin; u < t_end; ++u) wild |= W.template tail<false, (D < 256)>(P, c, g, u, lane);
    W.sums();
    if (wild) W.wild(P, g, t_begin, t_end, lane);
#pragma unroll
    for (int w = 0; w < RW; ++w) {
        const int rr = ((rt * NW + wave) * RW + w) * 16 + lo;
        if (rr < R) q8_finish<NB, 1>(P, g, rr, split, hi, 0, W.mrun[w], W.lsum[w], W.o[w]);
    }
}

// The splits' partials of one row: out = sum_s w_s acc_s / sum_s w_s l_s with
// w_s = 2^(m_s - max m). Block: DB dims (part blockIdx.z of D) of RPB rows, T = 256 / RPB
// threads each, thread t with 4 dims of every GS-th split (GS = 4 T / DB); their loads, 8
// at a time, do not wait for the weights, which the row's threads find meanwhile; sums
// over the GS groups meet in LDS.
template <int D, int RPB, int DB>
__global__ __launch_bounds__(256) void attn_q8_combine_kernel(AttnQ8Params P) {
    constexpr int T = 256 / RPB, LD = DB / 4, GS = T / LD, B = 8, W = Q8_MAX_SPLITS / T;
    static_assert(GS >= 1 && T % LD == 0, "threads per row");
    __shared__ float weight[RPB][Q8_MAX_SPLITS];
    __shared__ float red[RPB][2][T / 32];
    __shared__ q8_f4 part[RPB][GS][LD];
    const int row = threadIdx.x / T, t = threadIdx.x % T, d4 = t % LD, gs = t / LD, g = blockIdx.y;
    const int rr0 = blockIdx.x * RPB + row;
    const int G = P.qh / P.kh, R = G * P.m, S = P.splits;
    const int rr = min(rr0, R - 1);  // (threads past the last row: that row again, not written)
    const size_t at = ((size_t)g * P.rows_pad + rr) * S;
    const q8_f4* acc = reinterpret_cast<const q8_f4*>(P.part + at * D) + blockIdx.z * LD + d4;
    q8_f4 v[B];
#pragma unroll
    for (int i = 0; i < B; ++i) v[i] = acc[(size_t)min(gs + i * GS, S - 1) * (D / 4)];
    // weights and denominator, over the row's threads (whole half waves)
    const float2* ml = reinterpret_cast<const float2*>(P.part + (size_t)P.kh * P.rows_pad * S * D) + at;
    float2 x[W];
    float top = -INFINITY;
#pragma unroll
    for (int i = 0; i < W; ++i) {
        x[i] = t + i * T < S ? ml[t + i * T] : float2{-INFINITY, 0.0f};
        top = fmaxf(top, x[i].x);
    }
#pragma unroll
    for (int i = 1; i < 32; i <<= 1) top = fmaxf(top, __shfl_xor(top, i));
    if (t % 32 == 0) red[row][0][t / 32] = top;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < T / 32; ++i) top = fmaxf(top, red[row][0][i]);
    float den = 0.0f;
#pragma unroll
    for (int i = 0; i < W; ++i) {
        const float w = q8_weight(x[i].x, top);
        weight[row][t + i * T] = w;
        // (a split that saw NaN scores has a NaN sum)
        den += x[i].y != x[i].y ? x[i].y : w * x[i].y;
    }
#pragma unroll
    for (int i = 1; i < 32; i <<= 1) den += __shfl_xor(den, i);
    if (t % 32 == 0) red[row][1][t / 32] = den;
    __syncthreads();
    q8_f4 num = q8_f4{0.0f, 0.0f, 0.0f, 0.0f};
    for (int s = gs; s < S; s += B * GS) {
#pragma unroll
        for (int i = 0; i < B; ++i) {
            if (s + i * GS < S) num += v[i] * weight[row][s + i * GS];
            v[i] = acc[(size_t)min(s + (B + i) * GS, S - 1) * (D / 4)];
        }
    }
    if constexpr (GS > 1) {
        part[row][gs][d4] = num;
        __syncthreads();
        if (gs) return;
#pragma unroll
        for (int i = 1; i < GS; ++i) num += part[row][i][d4];
    }
    if (rr0 >= R) return;
    den = red[row][1][0];
#pragma unroll
    for (int i = 1; i < T / 32; ++i) den += red[row][1][i];
    const int h = rr / P.m;
    q8_store4(P, (long long)(g * G + h) * P.o_head + (rr - h * P.m) * P.o_row + DB * blockIdx.z + 4 * d4,
              num * (1.0f / den));
}

// The kernel of a run: attn_q8_tile_kernel (8 waves with row groups of their own, 2,
// or 1 of heads of 256) or attn_q8_kernel (waves that share `groups` row groups of 16).
struct Q8Plan {
    bool tile;
    int groups, waves;
    int rows() const { return 16 * groups * (tile ? waves : 1); }  // of a block
};

void launch_attn_q8_i8(const AttnQ8Params& P, int head_dim, const Q8Plan& plan, bool two, hipStream_t s);
void launch_attn_q8_e4m3(const AttnQ8Params& P, int head_dim, const Q8Plan& plan, bool two, hipStream_t s);

template <int D, int FMT, bool SPLIT>
static void launch_attn_q8_rows(const AttnQ8Params& P, const Q8Plan& plan, hipStream_t s) {
    // (a row tile's blocks of one KV head are 8 apart where there are 8 heads: the
    // XCDs take blocks in turn, so each keeps one head's codes in its L2)
    const dim3 grid(P.kh, P.row_tiles, P.splits), block(64 * plan.waves);
    constexpr int G = D == 256 ? 1 : 2;
    if (plan.tile)
        hipLaunchKernelGGL((attn_q8_tile_kernel<D, 8, G, G, FMT, SPLIT>), grid, block, 0, s, P);
    else if (plan.groups == 1)  // (narrow heads: up to 16 rows, whose weights are two fp16)
        hipLaunchKernelGGL((attn_q8_kernel<D, 4, 1, FMT, SPLIT || D != 256>), grid, block, 0, s, P);
    else
        hipLaunchKernelGGL((attn_q8_kernel<D, D == 256 ? 4 : 8, 2, FMT, SPLIT>), grid, block, 0, s, P);
}

template <int FMT>
static void launch_attn_q8(const AttnQ8Params& P, int head_dim, const Q8Plan& plan, bool two, hipStream_t s) {
#define HM_Q8_ROWS(DD)                                     \
    if (two)                                               \
        launch_attn_q8_rows<DD, FMT, true>(P, plan, s); \
    else                                                   \
        launch_attn_q8_rows<DD, FMT, false>(P, plan, s)
    if (head_dim == 64) {
        HM_Q8_ROWS(64);
    } else if (head_dim == 128) {
        HM_Q8_ROWS(128);
    } else {
        HM_Q8_ROWS(256);
    }
#undef HM_Q8_ROWS
}

}  // namespace hm
