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
// block of zeros has scale 1 here; a poisoned one (an infinity or NaN came) has
// NaN. The tail's fp16 rows lie in the same order with 8 values a lane and step.
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
// is the fp16 1024 + u. e4m3: the conversion instruction.
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

// Max / sum over the 4 lanes of a query row (l % 16 + 16 j), in each of them.
__device__ __forceinline__ float q8_rows4_max(float v) {
    v = fmaxf(v, __shfl_xor(v, 16));
    return fmaxf(v, __shfl_xor(v, 32));
}
__device__ __forceinline__ float q8_rows4_sum(float v) {
    v += __shfl_xor(v, 16);
    return v + __shfl_xor(v, 32);
}

// 8 consecutive q values of any alignment, as fp16.
__device__ __forceinline__ q8_h8 q8_load_q(const AttnQ8Params& P, long long at) {
    typedef unsigned u16 __attribute__((ext_vector_type(4), aligned(2)));
    typedef float f16 __attribute__((ext_vector_type(4), aligned(4)));
    if (!P.q_f32)
        return __builtin_bit_cast(q8_h8, v4u(*reinterpret_cast<const u16*>(static_cast<const __half*>(P.q) + at)));
    const float* p = static_cast<const float*>(P.q) + at;
    const f16 a = *reinterpret_cast<const f16*>(p), b = *reinterpret_cast<const f16*>(p + 4);
    q8_h8 r;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        r[i] = (_Float16)a[i];
        r[4 + i] = (_Float16)b[i];
    }
    return r;
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

// The weight 2^d of a partial result whose maximum lies d <= 0 below the row's:
// never 0, so that an infinite accumulator stays one (0 times it is NaN). What a
// finite one gains by that is below 2^-100 of the result.
__device__ __forceinline__ float q8_weight(float m, float top) {
    return m == -INFINITY ? 0.0f : fmaxf(__builtin_amdgcn_exp2f(m - top), 0x1p-120f);
}

constexpr float Q8_LAZY = 8.0f;   // a row's maximum moves when a score passes it by this much (powers of 2)
constexpr float Q8_SHIFT = 6.0f;  // SPLIT: the weights lie this much higher (p below 2^14, p mu below 2^15)

// Attention over codes and tail. Block: 4 waves over one tile of 16 RW query
// rows of one KV head; wave w takes units w, w + 4, .. of its split, so nothing
// is shared until the waves' partial (max, sum, accumulators) meet in LDS. A
// unit's codes go from memory into operand registers; the loads of the next
// unit are issued as soon as this one's are converted.
//
// With c = scale log2(e) and a block's scales ks and vs = mu 2^e, a key's weight
// is kept as p = 2^(c ks s + e - m): e in the exponent keeps the products p mu
// code of different blocks in one range, whatever their scales, so fp16 holds
// them. The row's sum adds p 2^-e, its accumulators p mu code; m is the running
// maximum, a whole number with SPLIT so that e - m is exact.
//
// SPLIT (f32 output): p mu goes into the products as two fp16, 22 bits.
// Otherwise (fp16 output) as one, and the sum adds the rounded weights (p mu
// times 1 / vs), so that a row whose weight is all on one key is not off.
//
// `poison`: a NaN scale makes every score of its block NaN, before the mask.
template <int D, int RW, int FMT, bool SPLIT>
__global__ __launch_bounds__(256) void attn_q8_kernel(AttnQ8Params P) {
    constexpr int KS = D / 32, NB = D / 16, KP = D / 32;  // KP: 16-byte pieces per lane, of K (and V)
    constexpr int RT = 16 * RW;
    constexpr float SHIFT = SPLIT ? Q8_SHIFT : 0.0f;
    __shared__ __attribute__((aligned(16))) float merge[3 * NB * 256];
    __shared__ float merge_ml[3][2][64];
    const int split = blockIdx.x, rt = blockIdx.y, g = blockIdx.z;
    const int G = P.qh / P.kh, R = G * P.m;
    const int lane = threadIdx.x & 63, lo = lane & 15, hi = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const float c = fminf(P.scale * 1.4426950408889634f, 0x1.fffffep127f);
    const uint8_t* kbase = P.k + (size_t)g * P.head_bytes + lane * 16;
    const uint8_t* vbase = P.v + (size_t)g * P.head_bytes + lane * 16;
    const float4* sc = P.sc + (size_t)g * P.blocks;
    const int coded_units = P.coded >> 5;

    // this lane's query rows: their key limits and fragments
    int lim[RW];
    q8_h8 qf[RW][KS];
    int open = 0x7fffffff, seen = 0;  // keys below `open` every row sees, from `seen` on none
#pragma unroll
    for (int w = 0; w < RW; ++w) {
        const int rr = rt * RT + 16 * w + lo;
        const bool ok = rr < R;
        const int h = g * G + (ok ? rr / P.m : 0), r = ok ? rr % P.m : 0;
        lim[w] = ok ? (P.causal ? min(P.len, P.pos + r + 1) : P.len) : 0;
        if (ok) {
            open = min(open, lim[w]);
            seen = max(seen, lim[w]);
        }
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            qf[w][s] = q8_load_q(P, h * P.q_head + r * P.q_row + 32 * s + 8 * hi);
            if (!ok) qf[w][s] = q8_h8{};
        }
    }
#pragma unroll
    for (int i = 1; i < 16; i <<= 1) {
        open = min(open, __shfl_xor(open, i));
        seen = max(seen, __shfl_xor(seen, i));
    }
    open = __builtin_amdgcn_readfirstlane(open);
    seen = __builtin_amdgcn_readfirstlane(seen);
    const int u_end = min(min((split + 1) * P.units_per_split, P.units), (seen + 31) >> 5);
    const int u_begin = split * P.units_per_split + wave;

    q8_f4 o[RW][NB];
    float mrun[RW], lsum[RW];  // (mrun: the row's maximum less SHIFT)
#pragma unroll
    for (int w = 0; w < RW; ++w) {
        mrun[w] = -INFINITY;
        lsum[w] = 0.0f;
#pragma unroll
        for (int n = 0; n < NB; ++n) o[w][n] = q8_f4{0.0f, 0.0f, 0.0f, 0.0f};
    }

    v4u kr[KP], vr[KP];
    // (the last coded unit's own codes again where there is no further one)
    auto load_k = [&](int u) {
        const uint8_t* p = kbase + (size_t)min(u, coded_units - 1) * (32 * D);
#pragma unroll
        for (int i = 0; i < KP; ++i) kr[i] = *reinterpret_cast<const v4u*>(p + i * 1024);
    };
    auto load_v = [&](int u) {
        const uint8_t* p = vbase + (size_t)min(u, coded_units - 1) * (32 * D);
#pragma unroll
        for (int i = 0; i < KP; ++i) vr[i] = *reinterpret_cast<const v4u*>(p + i * 1024);
    };
    if (u_begin < u_end && coded_units > 0) {
        load_k(u_begin);
        load_v(u_begin);
    }
    // A unit's scores to weights: s in, ph (and pl) out, the row's sum and, when
    // its maximum moves, its accumulators updated. `mu` 2^e: V's scale; `inv`: one
    // over it.
    auto weigh = [&](int key0, float ks, float mu, float inv, int e, q8_f4 (&s)[RW][2], q8_h8 (&ph)[RW],
                     q8_h8 (&pl)[RW]) {
        const bool poison = ks != ks || mu != mu;  // (uniform)
        const float ef = (float)e, down = __int_as_float((127 - e) << 23);  // 2^-e
        const float cks = fmaxf(c * ks, 0x1p-120f);
        if (__builtin_expect(poison, 0)) {
            mu = inv = 1.0f;
#pragma unroll
            for (int w = 0; w < RW; ++w)
#pragma unroll
                for (int cb = 0; cb < 2; ++cb) s[w][cb] = q8_f4{NAN, NAN, NAN, NAN};
        }
#pragma unroll
        for (int w = 0; w < RW; ++w) {
            if (__builtin_expect(key0 + 32 > open, 0)) {  // (uniform) the unit crosses a mask
#pragma unroll
                for (int cb = 0; cb < 2; ++cb)
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        if (key0 + 16 * cb + 4 * hi + r >= lim[w]) s[w][cb][r] = -INFINITY;
            }
            float top = __builtin_elementwise_maximum(
                __builtin_elementwise_maximum(__builtin_elementwise_maximum(s[w][0][0], s[w][0][1]),
                                              __builtin_elementwise_maximum(s[w][0][2], s[w][0][3])),
                __builtin_elementwise_maximum(__builtin_elementwise_maximum(s[w][1][0], s[w][1][1]),
                                              __builtin_elementwise_maximum(s[w][1][2], s[w][1][3])));
            top = __builtin_fmaf(top, cks, ef);
            if (__builtin_expect(__builtin_amdgcn_ballot_w64(top > mrun[w] + (Q8_LAZY + SHIFT)) != 0, 0)) {
                float tm = q8_rows4_max(top);
                if constexpr (SPLIT) tm = __builtin_ceilf(tm) - SHIFT;
                float alpha = 1.0f;
                if (tm > mrun[w] + Q8_LAZY) {
                    alpha = __builtin_amdgcn_exp2f(mrun[w] - tm);  // (0 from -inf)
                    mrun[w] = tm;
                }
                lsum[w] *= alpha;
#pragma unroll
                for (int n = 0; n < NB; ++n) o[w][n] *= alpha;
            }
            // (no key seen yet: every score is -inf)
            const float b = ef - (mrun[w] == -INFINITY ? 0.0f : mrun[w]);
            float l = 0.0f;
#pragma unroll
            for (int cb = 0; cb < 2; ++cb)
#pragma unroll
                for (int r = 0; r < 4; r += 2) {
                    const float p0 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[w][cb][r], cks, b));
                    const float p1 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[w][cb][r + 1], cks, b));
                    const float x0 = p0 * mu, x1 = p1 * mu;
                    const q8_h2 h = q8_round2(x0, x1);
                    ph[w][4 * cb + r] = h[0];
                    ph[w][4 * cb + r + 1] = h[1];
                    if constexpr (SPLIT) {
                        const q8_h2 d = {(_Float16)(x0 - (float)h[0]), (_Float16)(x1 - (float)h[1])};
                        pl[w][4 * cb + r] = d[0];
                        pl[w][4 * cb + r + 1] = d[1];
                        l += p0 + p1;
                    } else {
                        l = __builtin_amdgcn_fdot2(h, q8_h2{(_Float16)1.0f, (_Float16)1.0f}, l, false);
                    }
                }
            lsum[w] = __builtin_fmaf(l, SPLIT ? down : inv, lsum[w]);
        }
    };
    auto product = [&](int n, q8_h8 a, const q8_h8 (&ph)[RW], const q8_h8 (&pl)[RW]) {
#pragma unroll
        for (int w = 0; w < RW; ++w) {
            o[w][n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, ph[w], o[w][n], 0, 0, 0);
            if constexpr (SPLIT) o[w][n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, pl[w], o[w][n], 0, 0, 0);
        }
    };

    int u = u_begin;
    for (; u < min(u_end, coded_units); u += 4) {
        q8_f4 s[RW][2];
#pragma unroll
        for (int w = 0; w < RW; ++w) s[w][0] = s[w][1] = q8_f4{0.0f, 0.0f, 0.0f, 0.0f};
        const float4 x = sc[u >> P.unit_shift];
#pragma unroll
        for (int i = 0; i < KP; ++i) {
            const int cb = i / (D / 64), st = i % (D / 64);
            const q8_h8 a0 = q8_halves<FMT>(kr[i][0], kr[i][1]), a1 = q8_halves<FMT>(kr[i][2], kr[i][3]);
#pragma unroll
            for (int w = 0; w < RW; ++w) {
                s[w][cb] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a0, qf[w][2 * st], s[w][cb], 0, 0, 0);
                s[w][cb] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a1, qf[w][2 * st + 1], s[w][cb], 0, 0, 0);
            }
        }
        load_k(u + 4);
        q8_h8 ph[RW], pl[RW];
        weigh(u << 5, x.x, x.y, x.w, __float_as_int(x.z), s, ph, pl);
#pragma unroll
        for (int i = 0; i < KP; ++i) {
            product(2 * i, q8_halves<FMT>(vr[i][0], vr[i][1]), ph, pl);
            product(2 * i + 1, q8_halves<FMT>(vr[i][2], vr[i][3]), ph, pl);
        }
        load_v(u + 4);
    }

    // The tail: fp16 rows in the same order. What is not finite in V stays out of
    // the products (0 times it is NaN, so masked keys would show); V's exponents
    // move so that its largest magnitude lies near the codes'.
    const int u_tail = u;
    unsigned wild = 0;
    for (; u < u_end; u += 4) {
        const size_t at = (size_t)g * P.block_values + (size_t)(u - coded_units) * (32 * D) + lane * 8;
        q8_f4 s[RW][2];
#pragma unroll
        for (int w = 0; w < RW; ++w) s[w][0] = s[w][1] = q8_f4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int i = 0; i < 2 * KS; ++i) {
            const q8_h8 a = __builtin_bit_cast(q8_h8, *reinterpret_cast<const v4u*>(P.kt + at + i * 512));
#pragma unroll
            for (int w = 0; w < RW; ++w)
                s[w][i / KS] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, qf[w][i % KS], s[w][i / KS], 0, 0, 0);
        }
        // (what lies behind the last row is not the cache's)
        unsigned held[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int key = (u << 5) + (i >> 1) * 16 + 4 * hi + (i & 1) * 2;
            held[i] = (key < P.len ? 0xFFFFu : 0u) | (key + 1 < P.len ? 0xFFFF0000u : 0u);
        }
        unsigned big = 0;
#pragma unroll 2
        for (int n = 0; n < NB; ++n) {
            const v4u x = *reinterpret_cast<const v4u*>(P.vt + at + n * 512);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const unsigned y0 = x[i] & held[i] & 0x7FFFu, y1 = ((x[i] & held[i]) >> 16) & 0x7FFFu;
                wild |= (y0 >= 0x7C00u) | (y1 >= 0x7C00u);
                big = max(big, max(y0 >= 0x7C00u ? 0u : y0, y1 >= 0x7C00u ? 0u : y1));
            }
        }
#pragma unroll
        for (int i = 1; i < 64; i <<= 1) big = max(big, (unsigned)__shfl_xor((int)big, i));
        const float top = __half2float(__ushort_as_half((unsigned short)__builtin_amdgcn_readfirstlane((int)big)));
        const int e = top > 0.0f ? ((__float_as_int(top) >> 23) & 255) - 127 - 6 : -30;
        const float up = __int_as_float((127 - e) << 23);
        q8_h8 ph[RW], pl[RW];
        weigh(u << 5, 1.0f, 1.0f, up, e, s, ph, pl);
#pragma unroll
        for (int n = 0; n < NB; ++n) {
            const v4u x = *reinterpret_cast<const v4u*>(P.vt + at + n * 512);
            q8_h8 a = __builtin_bit_cast(q8_h8, x & v4u{held[0], held[1], held[2], held[3]});
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float y = (float)a[i];
                a[i] = (_Float16)(fabsf(y) < INFINITY ? y * up : 0.0f);
            }
            product(n, a, ph, pl);
        }
    }
#pragma unroll
    for (int w = 0; w < RW; ++w) lsum[w] = q8_rows4_sum(lsum[w]);

    // The infinite and NaN values of the tail that a row sees: its outputs take
    // their sum (whatever the weights, which are positive).
    if (__builtin_amdgcn_ballot_w64(wild != 0) != 0) {
#pragma unroll 1
        for (u = u_tail; u < u_end; u += 4) {
            const __half* vt = P.vt + (size_t)g * P.block_values + (size_t)(u - coded_units) * (32 * D);
#pragma unroll 1
            for (int j = 0; j < 32; ++j) {
                const __half* at = vt + ((j >> 2) & 3) * 128 + hi * 32 + (j >> 4) * 4 + (j & 3);
#pragma unroll
                for (int n = 0; n < NB; ++n)
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const float x = __half2float(at[n * 512 + r * 8]);
                        const float y = fabsf(x) < INFINITY ? 0.0f : x;
#pragma unroll
                        for (int w = 0; w < RW; ++w) o[w][n][r] += (u << 5) + j < lim[w] ? y : 0.0f;
                    }
            }
        }
    }

    // The waves' partials meet: wave w % 4 gathers row group w.
#pragma unroll
    for (int w = 0; w < RW; ++w) {
        const int owner = w & 3;
        if (w) __syncthreads();  // (the previous group's reads are done)
        if (wave != owner) {
            const int at = wave < owner ? wave : wave - 1;
#pragma unroll
            for (int n = 0; n < NB; ++n) *reinterpret_cast<q8_f4*>(&merge[((at * NB + n) * 64 + lane) * 4]) = o[w][n];
            merge_ml[at][0][lane] = mrun[w];
            merge_ml[at][1][lane] = lsum[w];
        }
        __syncthreads();
        if (wave != owner) continue;
        float mx[3], top = mrun[w];
#pragma unroll
        for (int at = 0; at < 3; ++at) {
            mx[at] = merge_ml[at][0][lane];
            top = fmaxf(top, mx[at]);
        }
        const float a = q8_weight(mrun[w], top);
        float l = lsum[w] * a;
#pragma unroll
        for (int n = 0; n < NB; ++n) o[w][n] *= a;
#pragma unroll
        for (int at = 0; at < 3; ++at) {
            // (a wave that saw no key holds zeros; one that saw NaN scores has
            // maximum -inf and NaN sums)
            const float b = q8_weight(mx[at], top), l1 = merge_ml[at][1][lane];
            l += l1 != l1 ? l1 : l1 * b;
#pragma unroll
            for (int n = 0; n < NB; ++n)
                o[w][n] += *reinterpret_cast<const q8_f4*>(&merge[((at * NB + n) * 64 + lane) * 4]) * b;
        }
        if (lsum[w] != lsum[w]) l = lsum[w];
        const int rr = rt * RT + 16 * w + lo;
        if (rr >= R) continue;
        if (P.splits == 1) {
            const float il = 1.0f / l;
            const long long at = (g * G + rr / P.m) * P.o_head + rr % P.m * P.o_row + 4 * hi;
#pragma unroll
            for (int n = 0; n < NB; ++n) q8_store4(P, at + 16 * n, o[w][n] * il);
        } else {
            const size_t row = ((size_t)g * P.rows_pad + rr) * P.splits + split;
#pragma unroll
            for (int n = 0; n < NB; ++n)
                *reinterpret_cast<q8_f4*>(P.part + row * D + 16 * n + 4 * hi) = o[w][n];
            if (hi == 0) {
                float* ml = P.part + (size_t)P.kh * P.rows_pad * P.splits * D + row * 2;
                ml[0] = top;
                ml[1] = l;
            }
        }
    }
}

// The splits' partials of one row: out = sum_s w_s acc_s / sum_s w_s l_s with
// w_s = 2^(m_s - max m). One wave per row, 4 rows a block; lane s holds the
// weights of splits s, s + 64, ..; the accumulators of 8 splits are in flight.
template <int D>
__global__ __launch_bounds__(256) void attn_q8_combine_kernel(AttnQ8Params P) {
    constexpr int ND = D / 64, B = 8;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, g = blockIdx.y;
    const int rr = blockIdx.x * 4 + wave;
    const int G = P.qh / P.kh, R = G * P.m, S = P.splits;
    if (rr >= R) return;  // (wave-uniform; no barrier below)
    const size_t row = ((size_t)g * P.rows_pad + rr) * S;
    const float2* ml = reinterpret_cast<const float2*>(P.part + (size_t)P.kh * P.rows_pad * S * D) + row;
    float top = -INFINITY;
    for (int s = lane; s < S; s += 64) top = fmaxf(top, ml[s].x);
#pragma unroll
    for (int i = 1; i < 64; i <<= 1) top = fmaxf(top, __shfl_xor(top, i));
    float den = 0.0f, num[ND];
#pragma unroll
    for (int d = 0; d < ND; ++d) num[d] = 0.0f;
    for (int s0 = 0; s0 < S; s0 += 64) {
        const int mine = s0 + lane;
        const float2 x = mine < S ? ml[mine] : float2{-INFINITY, 0.0f};
        const float w = q8_weight(x.x, top);
        den += x.y != x.y ? x.y : w * x.y;
        const int count = min(64, S - s0);
        for (int b = 0; b < count; b += B) {
            float v[B][ND];
#pragma unroll
            for (int i = 0; i < B; ++i)
#pragma unroll
                for (int d = 0; d < ND; ++d)
                    v[i][d] = P.part[(row + s0 + min(b + i, count - 1)) * D + lane + 64 * d];
#pragma unroll
            for (int i = 0; i < B; ++i) {
                const float wi = __shfl(w, min(b + i, count - 1));
#pragma unroll
                for (int d = 0; d < ND; ++d)
                    num[d] = b + i < count ? __builtin_fmaf(wi, v[i][d], num[d]) : num[d];
            }
        }
    }
#pragma unroll
    for (int i = 1; i < 64; i <<= 1) den += __shfl_xor(den, i);
    const float il = 1.0f / den;
    const long long at = (g * G + rr / P.m) * P.o_head + rr % P.m * P.o_row + lane;
#pragma unroll
    for (int d = 0; d < ND; ++d) {
        const float y = num[d] * il;
        if (P.out_f16)
            static_cast<__half*>(P.out)[at + 64 * d] = __float2half_rn(y);
        else
            static_cast<float*>(P.out)[at + 64 * d] = y;
    }
}

// Row groups (16 rows) per tile for R rows of a KV head.
inline int q8_row_groups(int head_dim, int R) { return R <= 16 ? 1 : R <= 32 || head_dim == 256 ? 2 : 4; }

void launch_attn_q8_i8(const AttnQ8Params& P, int head_dim, int row_groups, bool f32_weights, hipStream_t s);
void launch_attn_q8_e4m3(const AttnQ8Params& P, int head_dim, int row_groups, bool f32_weights, hipStream_t s);

template <int D, int FMT, bool SPLIT>
static void launch_attn_q8_rows(const AttnQ8Params& P, int row_groups, hipStream_t s) {
    const dim3 grid(P.splits, P.row_tiles, P.kh);
    if (row_groups == 1)
        hipLaunchKernelGGL((attn_q8_kernel<D, 1, FMT, SPLIT>), grid, dim3(256), 0, s, P);
    else if (row_groups == 2)
        hipLaunchKernelGGL((attn_q8_kernel<D, 2, FMT, SPLIT>), grid, dim3(256), 0, s, P);
    else if constexpr (D < 256)
        hipLaunchKernelGGL((attn_q8_kernel<D, 4, FMT, SPLIT>), grid, dim3(256), 0, s, P);
}

template <int FMT>
static void launch_attn_q8(const AttnQ8Params& P, int head_dim, int row_groups, bool f32_weights, hipStream_t s) {
#define HM_Q8_ROWS(DD)                                       \
    if (f32_weights)                                         \
        launch_attn_q8_rows<DD, FMT, true>(P, row_groups, s); \
    else                                                     \
        launch_attn_q8_rows<DD, FMT, false>(P, row_groups, s)
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
