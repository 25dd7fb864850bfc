// Kernels of the paged KV cache's attention (include/rk_npu_attention_paged.h).
//
// Layout in HBM, per page and KV head, `page` tokens in tiles of 16:
//   K: [4-key group][D / 8 pieces][4 keys][8 dims]; piece p of group n lies at
//      place p ^ (n & 3). A lane of a matrix operand takes one piece, lanes of
//      4 keys a 64-byte line;
//   V: [key][D / 8 pieces][8 dims], piece p of key j at place p ^ v_turn(j).
// The turned places keep 16 keys' pieces out of each other's LDS banks when a
// tile lies there as it does in HBM.
//
// Operands of v_mfma_f32_16x16x32_f16: A lane l = row l % 16, k-slots
// 8 (l / 16)..+7; B lane l = column l % 16, the same slots; C lane l = rows
// 4 (l / 16)..+3 of column l % 16. S^T = K Q^T leaves lane l the scores of query
// row l % 16 for keys 4 (l / 16)..+3 of each 16, which is what B of
// O^T += V^T P^T wants once V's slots name the same keys.
#pragma once

#include <hip/hip_fp16.h>
#include <hip/hip_runtime.h>

#include "../../include/rk_npu_attention_paged.h"
#include "kernels.hpp"

namespace hm {

constexpr int PAGED_MAX_SPLITS = 256;  // key splits that a row's join takes

typedef _Float16 pg_h8 __attribute__((ext_vector_type(8)));
typedef _Float16 pg_h2 __attribute__((ext_vector_type(2)));
typedef float pg_f4 __attribute__((ext_vector_type(4)));
typedef unsigned pg_u4a2 __attribute__((ext_vector_type(4), aligned(2)));
typedef unsigned pg_u2a2 __attribute__((ext_vector_type(2), aligned(2)));
typedef float pg_f4a4 __attribute__((ext_vector_type(4), aligned(4)));

// The batch and the pool in a kernel's arguments.
struct PagedBatch {
    const int* lengths;
    const int* offsets;  // nullptr: a row each
    const int* table;
    int* flaw;           // set where the batch is wrong
    __half* k;           // [page][kv head][page tokens * D]
    __half* v;
    int sequences, rows, max_rows, max_tokens, table_stride;
    int kh, pages, page_shift;
};

__device__ __forceinline__ int pg_k_place(int D, int j, int piece) {  // of piece `piece` of key j, in 8 halves
    return (j >> 2) * (D >> 1) + (piece ^ ((j >> 2) & 3)) * 4 + (j & 3);
}
// (heads of 64: two keys fill the 256 bytes of the banks)
__device__ __forceinline__ constexpr int pg_v_turn(int D, int j) { return D == 64 ? 2 * ((j >> 1) & 3) : 2 * (j & 7); }
__device__ __forceinline__ int pg_v_place(int D, int j, int piece) { return j * (D >> 3) + (piece ^ pg_v_turn(D, j)); }

__device__ __forceinline__ void pg_flaw(const PagedBatch& B) { atomicOr(B.flaw, 1); }

// Sequence s: its rows and length, none of what the batch has wrong.
struct PagedSeq {
    int row, n, len;
};
__device__ __forceinline__ PagedSeq pg_seq(const PagedBatch& B, int s) {
    PagedSeq q{s, 1, B.lengths[s]};
    if (B.offsets) {
        const int a = B.offsets[s], b = B.offsets[s + 1];
        const bool ok = a >= 0 && b >= a && b <= B.rows && b - a <= B.max_rows;
        q.row = ok ? a : 0;
        q.n = ok ? b - a : 0;
        if (!ok) pg_flaw(B);
    }
    if (q.len < 0 || q.len > B.max_tokens) {
        q.len = 0;
        pg_flaw(B);
    }
    return q;
}
// The page of a token of sequence s (below its length), or -1.
__device__ __forceinline__ int pg_page(const PagedBatch& B, int s, int token) {
    const int p = B.table[(size_t)s * B.table_stride + (token >> B.page_shift)];
    if ((unsigned)p < (unsigned)B.pages) return p;
    pg_flaw(B);
    return -1;
}

struct AttnPagedParams {
    PagedBatch b;
    const void* q;
    int q_f32;
    long long q_head, q_row;  // strides, elements
    void* out;
    int out_f16;
    long long o_head, o_row;
    float* part;     // accumulators [item][kh][tile rows][D], then (max, sum) pairs
    int qh, causal;
    float scale;
    int items;       // blocks per KV head
    int target;      // blocks per KV head that splits aim at; 0: no splits
    int least;       // units of a split, at least
    int tile_rows;   // query rows of a block
    int tiles;       // row tiles of the whole batch, at most
};

__device__ __forceinline__ int pg_scan(int v) {  // inclusive, over the wave
    v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, false);  // row_shr:1, 2, 4, 8
    v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, DPP_ROW_BCAST15, 0xa, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, DPP_ROW_BCAST31, 0xc, 0xf, false);
    return v;
}

// One block's work: row tile `tile` of a sequence, split `split` of `splits` of its
// keys; `item`: the sequence's first block of that tile.
struct PagedItem {
    int s, row, n, len, tile, split, splits, item;
    bool any;
};

// The schedule, made by every wave from the lengths alone: a sequence has ceil(rows /
// tile_rows) tiles, each split into as many pieces of at least `per` units of 32 keys
// as it has; per is the batch's units over `target`, so that splits of short and long
// sequences take the same time. Blocks of a sequence lie in the order of their tiles,
// then splits. Counted by tiles alone (`joins`), index `at` is the tile of a join.
// Lane l has sequences l C..l C + C - 1.
__device__ __forceinline__ PagedItem pg_item(const AttnPagedParams& P, int at, int lane, bool joins) {
    const PagedBatch& B = P.b;
    const int G = P.qh / B.kh, C = (B.sequences + 63) >> 6;
    auto tiles_of = [&](const PagedSeq& q) { return (int)(((long long)q.n * G + P.tile_rows - 1) / P.tile_rows); };
    int per = 0x7fffffff;
    if (P.target > 0) {
        int units = 0;
        for (int i = 0; i < C; ++i) {
            const int s = lane * C + i;
            if (s >= B.sequences) break;
            const PagedSeq q = pg_seq(B, s);
            units += tiles_of(q) * ((q.len + 31) >> 5);
        }
        const int total = __builtin_amdgcn_readlane(pg_scan(units), 63);
        per = max(P.least, (total + P.target - 1) / P.target);
    }
    auto splits_of = [&](const PagedSeq& q) {
        return min(PAGED_MAX_SPLITS, max(1, (int)(((q.len + 31) >> 5) + (long long)per - 1) / per));
    };
    int items = 0, tiles = 0;
    for (int i = 0; i < C; ++i) {
        const int s = lane * C + i;
        if (s >= B.sequences) break;
        const PagedSeq q = pg_seq(B, s);
        items += tiles_of(q) * splits_of(q);
        tiles += tiles_of(q);
    }
    const int item_end = pg_scan(items), tile_end = pg_scan(tiles);
    const int end = joins ? tile_end : item_end;
    const unsigned long long over = __builtin_amdgcn_ballot_w64(end > at);
    PagedItem x{};
    x.any = over != 0;
    if (!x.any) return x;
    const int owner = __builtin_ctzll(over);
    int first = __builtin_amdgcn_readlane(item_end - items, owner);
    int before = __builtin_amdgcn_readlane(end - (joins ? tiles : items), owner);
    for (int i = 0; i < C; ++i) {
        x.s = min(owner * C + i, B.sequences - 1);
        const PagedSeq q = pg_seq(B, x.s);
        const int t = tiles_of(q), p = splits_of(q), count = joins ? t : t * p;
        if (at < before + count) {
            const int in = at - before;
            x.row = q.row;
            x.n = q.n;
            x.len = q.len;
            x.splits = p;
            x.tile = joins ? in : in / p;
            x.split = joins ? 0 : in - x.tile * p;
            x.item = first + x.tile * p;
            return x;
        }
        before += count;
        first += t * p;
    }
    x.any = false;
    return x;
}

// Two f32 to fp16, once: without the empty asm the compiler folds the product
// before a rounding into it in one of the rounding's uses (a single rounding there,
// two in the others), and the remainder is then that of another value.
__device__ __forceinline__ pg_h2 pg_round2(float a, float b) {
    unsigned w = __builtin_bit_cast(unsigned, pg_h2{(_Float16)a, (_Float16)b});
    asm("" : "+v"(w));
    return __builtin_bit_cast(pg_h2, w);
}

// Max / sum over the 4 lanes of a query row (l % 16 + 16 j), in each of them.
__device__ __forceinline__ float pg_rows4_max(float v) {
    const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
    const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ float pg_rows4_sum(float v) {
    const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(a[0]) + __uint_as_float(a[1]);
    const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}
// Min over each 16 lanes, in each of them.
__device__ __forceinline__ int pg_row_min(int v) {
    v = min(v, dpp_move<DPP_QUAD_XOR1>(v));
    v = min(v, dpp_move<DPP_QUAD_XOR2>(v));
    v = min(v, dpp_move<DPP_ROW_HALF_MIRROR>(v));
    return min(v, dpp_move<DPP_ROW_MIRROR>(v));
}

// A row's maximum before it has seen a key: finite, so that differences are no NaN.
constexpr float PG_NONE = -1e30f;
// The weight 2^d of a partial result whose maximum lies d <= 0 below the row's:
// never 0, so that an infinite accumulator stays one (0 times it is NaN). A finite sum
// gains by that 2^-106 of the row's at most (weights lie below 2^14).
__device__ __forceinline__ float pg_weight(float m, float top) {
    return fmaxf(__builtin_amdgcn_exp2f(m - top), 0x1p-120f);
}

// 8 consecutive outputs of any alignment.
__device__ __forceinline__ void pg_store8(const AttnPagedParams& P, long long at, const float (&y)[8]) {
    if (P.out_f16) {
        v4u w;
#pragma unroll
        for (int i = 0; i < 4; ++i)
            w[i] = __half_as_ushort(__float2half_rn(y[2 * i])) |
                   ((unsigned)__half_as_ushort(__float2half_rn(y[2 * i + 1])) << 16);
        *reinterpret_cast<pg_u4a2*>(static_cast<__half*>(P.out) + at) = pg_u4a2(w);
    } else {
        float* p = static_cast<float*>(P.out) + at;
        *reinterpret_cast<pg_f4a4*>(p) = pg_f4a4{y[0], y[1], y[2], y[3]};
        *reinterpret_cast<pg_f4a4*>(p + 4) = pg_f4a4{y[4], y[5], y[6], y[7]};
    }
}

// 8 query values as fp16.
__device__ __forceinline__ pg_h8 pg_load_q(const AttnPagedParams& P, long long at) {
    if (!P.q_f32) return __builtin_bit_cast(pg_h8, v4u(*reinterpret_cast<const pg_u4a2*>(static_cast<const __half*>(P.q) + at)));
    const float* p = static_cast<const float*>(P.q) + at;
    const pg_f4a4 a = *reinterpret_cast<const pg_f4a4*>(p), b = *reinterpret_cast<const pg_f4a4*>(p + 4);
    pg_h8 h;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        h[i] = (_Float16)a[i];
        h[4 + i] = (_Float16)b[i];
    }
    return h;
}

// A row's maximum moves when a score passes it by LAZY (powers of 2), to SHIFT below
// the score: weights lie below 2^14, the row's largest above 2^10, so that the second
// fp16 of a weight, of 2^-11 of the first, keeps its bits down to weights of 2^-13.
constexpr float PG_LAZY = 4.0f, PG_SHIFT = 10.0f;

// Few rows. Block: NW waves over one tile of 16 query rows (8 where PACK) of one KV
// head of a sequence; wave w takes units w, w + NW, .. of 32 keys of its split, so
// nothing is shared until the waves' partial (max, sum, accumulators) meet in LDS.
// K comes from memory in operand order; V comes as rows, 8 keys of 8 dims a lane, and
// is transposed there, two keys' halves a v_perm_b32. Weights go into the products
// with V as two fp16. PACK: columns 8..15 are columns 0..7 again and take the second
// fp16, so that both cost one product.
template <int D, int NW, bool PACK>
__global__ __launch_bounds__(64 * NW) void attn_paged_rows_kernel(AttnPagedParams P) {
    constexpr int KS = D / 32;                  // 32-dim steps of a score
    constexpr int DW = D == 64 ? 4 : 8;         // dims of V a lane takes of a key, H times
    constexpr int H = D / (16 * DW), NB = H * DW;
    constexpr int COLS = PACK ? 8 : 16, PITCH = D + 4;
    __shared__ __attribute__((aligned(16))) float acc[NW][COLS][PITCH];
    __shared__ float ml[NW][2][16];
    const PagedBatch& B = P.b;
    const int g = blockIdx.x % B.kh, at = blockIdx.x / B.kh;
    const int lane = threadIdx.x & 63, lo = lane & 15, hi = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const PagedItem I = pg_item(P, at, lane, false);
    if (!I.any) return;  // (block-uniform)
    const int G = P.qh / B.kh, R = G * I.n, col = PACK ? lo & 7 : lo;
    const int rr = I.tile * COLS + col;
    const bool live = rr < R;
    const int r = live ? rr / G : 0, h = live ? rr - r * G : 0;
    const int lim = !live ? 0 : P.causal ? max(0, min(I.len, I.len - I.n + r + 1)) : I.len;
    // keys below `open` every row sees, from `seen` on none
    const int open = __builtin_amdgcn_readfirstlane(pg_row_min(live ? lim : 0x7fffffff));
    const int seen = -__builtin_amdgcn_readfirstlane(pg_row_min(-lim));
    const int units = (seen + 31) >> 5, each = (units + I.splits - 1) / I.splits;
    const int u_begin = I.split * each, u_end = min(units, u_begin + each);

    pg_h8 qf[KS];
    const long long q_at = (long long)(g * G + h) * P.q_head + (long long)(I.row + r) * P.q_row + 8 * hi;
#pragma unroll
    for (int i = 0; i < KS; ++i) qf[i] = pg_load_q(P, q_at + 32 * i);

    const float c = fminf(P.scale * 1.4426950408889634f, 0x1.fffffep127f);
    // Lane l's place in the table of the wave's next 32 units: unit l / 2, half l % 2,
    // as 16-key tiles of the pool (-1: no token there).
    const int page_tiles = 1 << (B.page_shift - 4);
    auto places = [&](int u) {
        const int token = (u + NW * (lane >> 1)) * 32 + (lane & 1) * 16;
        if (token >= min(seen, u_end * 32)) return -1;
        const int page = pg_page(B, I.s, token);
        return page < 0 ? -1 : (page * B.kh + g) * page_tiles + ((token >> 4) & (page_tiles - 1));
    };
    int place = -1, place_at = -64 * NW;
    v4u kr[2][KS];
    v4u vr[2][4][H];
    int tile[2];
    auto load = [&](int u) {
        if (u - place_at >= 32 * NW) {
            place = places(u);
            place_at = u;
        }
        const int i = (u - place_at) / NW * 2;
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            tile[t] = __builtin_amdgcn_readlane(place, i + t);
            const size_t at = (size_t)max(tile[t], 0) * (16 * D);
            const __half* kp = B.k + at;
            const __half* vp = B.v + at;
#pragma unroll
            for (int s = 0; s < KS; ++s) kr[t][s] = *reinterpret_cast<const v4u*>(kp + pg_k_place(D, lo, 4 * s + hi) * 8);
#pragma unroll
            for (int k = 0; k < 4; ++k)
#pragma unroll
                for (int w = 0; w < H; ++w) {
                    const int j = 4 * hi + k;
                    if constexpr (D == 64) {
                        const uint2 x = *reinterpret_cast<const uint2*>(vp + pg_v_place(D, j, lo >> 1) * 8 + (lo & 1) * 4);
                        vr[t][k][w] = v4u{x.x, x.y, 0u, 0u};
                    } else {
                        vr[t][k][w] = *reinterpret_cast<const v4u*>(vp + pg_v_place(D, j, 16 * w + lo) * 8);
                    }
                }
        }
    };

    float mrun = PG_NONE, lsum = 0.0f;
    pg_f4 o[NB];
#pragma unroll
    for (int n = 0; n < NB; ++n) o[n] = pg_f4{0.0f, 0.0f, 0.0f, 0.0f};
    bool wild = false;
    const float second = PACK && lo >= 8 ? 1.0f : 0.0f;
    for (int u = u_begin + wave; u < u_end; u += NW) {
        load(u);
        pg_f4 s[2];
        s[0] = s[1] = pg_f4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int i = 0; i < KS; ++i)
                s[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(pg_h8, kr[t][i]), qf[i], s[t], 0, 0, 0);
        const bool part = u * 32 + 32 > open || tile[0] < 0 || tile[1] < 0;
        if (part) {  // (uniform)
            unsigned odd = 0;
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const int key = u * 32 + 16 * t + 4 * hi + k;
                    if (key >= lim || tile[t] < 0) s[t][k] = -INFINITY;
                    // (0 times what is not finite is NaN: such a value of a key that not
                    // every row sees is added after the last one)
                    const bool none = key >= seen || tile[t] < 0;
#pragma unroll
                    for (int w = 0; w < H; ++w)
#pragma unroll
                        for (int i = 0; i < DW / 2; ++i) {
                            unsigned x = vr[t][k][w][i];
                            unsigned drop = (x & 0x7C00u) == 0x7C00u ? 0xFFFFu : 0u;
                            drop |= (x & 0x7C000000u) == 0x7C000000u ? 0xFFFF0000u : 0u;
                            if (key < open) drop = 0u;
                            if (!none) odd |= drop;
                            vr[t][k][w][i] = none ? 0u : x & ~drop;
                        }
                }
            wild |= odd != 0;
        }
        float top = __builtin_elementwise_maximum(
            __builtin_elementwise_maximum(__builtin_elementwise_maximum(s[0][0], s[0][1]),
                                          __builtin_elementwise_maximum(s[0][2], s[0][3])),
            __builtin_elementwise_maximum(__builtin_elementwise_maximum(s[1][0], s[1][1]),
                                          __builtin_elementwise_maximum(s[1][2], s[1][3])));
        top *= c;
        if (__builtin_amdgcn_ballot_w64(top > mrun + (PG_LAZY + PG_SHIFT)) != 0) {
            const float tm = pg_rows4_max(top) - PG_SHIFT;
            if (tm > mrun + PG_LAZY) {
                const float alpha = __builtin_amdgcn_exp2f(mrun - tm);
                mrun = tm;
                lsum *= alpha;
#pragma unroll
                for (int n = 0; n < NB; ++n) o[n] *= alpha;
            }
        }
        pg_h8 ph, pl;
        float l[2] = {0.0f, 0.0f};
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int k = 0; k < 4; k += 2) {
                const float p0 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[t][k], c, -mrun));
                const float p1 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[t][k + 1], c, -mrun));
                const pg_h2 x = pg_round2(p0, p1);
                if constexpr (PACK) {
                    ph[4 * t + k] = (_Float16)__builtin_fmaf((float)x[0], -second, p0);
                    ph[4 * t + k + 1] = (_Float16)__builtin_fmaf((float)x[1], -second, p1);
                } else {
                    ph[4 * t + k] = x[0];
                    ph[4 * t + k + 1] = x[1];
                    pl[4 * t + k] = (_Float16)(p0 - (float)x[0]);
                    pl[4 * t + k + 1] = (_Float16)(p1 - (float)x[1]);
                }
                l[t] += p0 + p1;
            }
        lsum += l[0] + l[1];
#pragma unroll
        for (int w = 0; w < H; ++w)
#pragma unroll
            for (int d = 0; d < DW; ++d) {
                v4u a;
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    a[i] = __builtin_amdgcn_perm(vr[i >> 1][2 * (i & 1) + 1][w][d >> 1], vr[i >> 1][2 * (i & 1)][w][d >> 1],
                                                 d & 1 ? 0x07060302u : 0x05040100u);
                const pg_h8 av = __builtin_bit_cast(pg_h8, a);
                o[w * DW + d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(av, ph, o[w * DW + d], 0, 0, 0);
                if constexpr (!PACK)
                    o[w * DW + d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(av, pl, o[w * DW + d], 0, 0, 0);
            }
    }
    lsum = pg_rows4_sum(lsum);
    // Infinities and NaN among the values: the products leave NaN of them (0, or a
    // negative second fp16, times an infinity). A result that they reach is their sum,
    // whatever the weights, which are positive.
#pragma unroll
    for (int n = 0; n < NB; ++n)
#pragma unroll
        for (int k = 0; k < 4; ++k) wild |= !(fabsf(o[n][k]) < INFINITY);
    if (__builtin_amdgcn_ballot_w64(wild) != 0) {
        float sum[NB][4];
#pragma unroll
        for (int n = 0; n < NB; ++n)
#pragma unroll
            for (int k = 0; k < 4; ++k) sum[n][k] = 0.0f;
#pragma unroll 1
        for (int u = u_begin + wave; u < u_end; u += NW) {
#pragma unroll 1
            for (int key = u * 32; key < min(u * 32 + 32, seen); ++key) {
                const int page = pg_page(B, I.s, key), j = key & 15;
                if (page < 0) continue;
                const __half* vp = B.v + ((size_t)(page * B.kh + g) * page_tiles + ((key >> 4) & (page_tiles - 1))) * (16 * D);
#pragma unroll
                for (int w = 0; w < H; ++w)
#pragma unroll
                    for (int k = 0; k < 4; ++k)
#pragma unroll
                        for (int d = 0; d < DW; ++d) {
                            const int dim = 128 * w + (4 * hi + k) * DW + d;
                            const float x = __half2float(vp[pg_v_place(D, j, dim >> 3) * 8 + (dim & 7)]);
                            sum[w * DW + d][k] += key < lim && !(fabsf(x) < INFINITY) ? x : 0.0f;
                        }
            }
        }
#pragma unroll
        for (int n = 0; n < NB; ++n)
#pragma unroll
            for (int k = 0; k < 4; ++k) o[n][k] = fabsf(sum[n][k]) < INFINITY ? float(o[n][k]) : sum[n][k];
    }
    // The waves meet. Lane (lo, hi) has dims 128 w + (4 hi + k) DW + d of its row.
    if constexpr (PACK) {
#pragma unroll
        for (int n = 0; n < NB; ++n)
#pragma unroll
            for (int k = 0; k < 4; ++k) o[n][k] += dpp_move<0x128>(float(o[n][k]));  // row_ror:8
    }
    if (lo < COLS) {
#pragma unroll
        for (int w = 0; w < H; ++w)
#pragma unroll
            for (int k = 0; k < 4; ++k)
#pragma unroll
                for (int d = 0; d < DW; d += 4)
                    *reinterpret_cast<pg_f4*>(&acc[wave][lo][128 * w + (4 * hi + k) * DW + d]) =
                        pg_f4{o[w * DW + d][k], o[w * DW + d + 1][k], o[w * DW + d + 2][k], o[w * DW + d + 3][k]};
        if (hi == 0) {
            ml[wave][0][lo] = mrun;
            ml[wave][1][lo] = lsum;
        }
    }
    __syncthreads();
    constexpr int PIECES = COLS * D / 8;
    for (int i = threadIdx.x; i < PIECES; i += 64 * NW) {
        const int row = i / (D / 8), d = i % (D / 8) * 8, rr = I.tile * COLS + row;
        if (rr >= R) continue;
        float top = PG_NONE, m1[NW], l = 0.0f, y[8];
#pragma unroll
        for (int w = 0; w < NW; ++w) {
            m1[w] = ml[w][0][row];
            top = fmaxf(top, m1[w]);
        }
#pragma unroll
        for (int k = 0; k < 8; ++k) y[k] = 0.0f;
#pragma unroll
        for (int w = 0; w < NW; ++w) {
            // (a wave that saw no key holds zeros, one that saw NaN scores a NaN sum)
            const float b = pg_weight(m1[w], top), l1 = ml[w][1][row];
            l += l1 != l1 ? l1 : l1 * b;
            const pg_f4 x0 = *reinterpret_cast<const pg_f4*>(&acc[w][row][d]);
            const pg_f4 x1 = *reinterpret_cast<const pg_f4*>(&acc[w][row][d + 4]);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                y[k] += x0[k] * b;
                y[4 + k] += x1[k] * b;
            }
        }
        if (I.splits == 1) {
            const int r = rr / G, h = rr - r * G;
            const bool empty = P.causal ? I.len - I.n + r + 1 <= 0 : I.len == 0;
            const float il = empty ? 0.0f : 1.0f / l;
#pragma unroll
            for (int k = 0; k < 8; ++k) y[k] *= il;
            pg_store8(P, (long long)(g * G + h) * P.o_head + (long long)(I.row + r) * P.o_row + d, y);
        } else {
            const size_t row_at = ((size_t)at * B.kh + g) * COLS + row;
            float* p = P.part + row_at * D + d;
            *reinterpret_cast<pg_f4*>(p) = pg_f4{y[0], y[1], y[2], y[3]};
            *reinterpret_cast<pg_f4*>(p + 4) = pg_f4{y[4], y[5], y[6], y[7]};
            if (d == 0)
                *reinterpret_cast<float2*>(P.part + (size_t)P.items * B.kh * COLS * D + row_at * 2) = float2{top, l};
        }
    }
}

// The splits' partials of one row: out = sum_s w_s acc_s / sum_s w_s l_s with
// w_s = 2^(m_s - max m). Block: one row of one row tile (blockIdx.y) and KV head; 256
// threads, 8 dims of every 2048 / D-th split each.
template <int D>
__global__ __launch_bounds__(256) void attn_paged_join_kernel(AttnPagedParams P) {
    constexpr int LD = D / 8, GS = 256 / LD;
    __shared__ float weight[PAGED_MAX_SPLITS];
    __shared__ float red[2][4];
    __shared__ __attribute__((aligned(16))) float part[GS][D];
    const PagedBatch& B = P.b;
    const int g = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const PagedItem I = pg_item(P, blockIdx.y, lane, true);
    // (a block past the grid of the batch's wrong offsets has written nothing)
    if (!I.any || I.splits == 1 || I.item + I.splits > P.items) return;
    const int G = P.qh / B.kh, row = blockIdx.z, rr = I.tile * P.tile_rows + row;
    if (rr >= G * I.n) return;
    const size_t step = (size_t)B.kh * P.tile_rows, at = ((size_t)I.item * B.kh + g) * P.tile_rows + row;
    const float2* ml = reinterpret_cast<const float2*>(P.part + (size_t)P.items * step * D) + at;
    const float2 x = tid < I.splits ? ml[tid * step] : float2{PG_NONE, 0.0f};
    float top = wave_max(x.x);
    if (lane == 0) red[0][wave] = top;
    __syncthreads();
    top = fmaxf(fmaxf(red[0][0], red[0][1]), fmaxf(red[0][2], red[0][3]));
    const float w = pg_weight(x.x, top);
    weight[tid] = w;
    // (a split that saw NaN scores has a NaN sum)
    float den = x.y != x.y ? x.y : w * x.y;
#pragma unroll
    for (int i = 1; i < 64; i <<= 1) den += __shfl_xor(den, i);
    if (lane == 0) red[1][wave] = den;
    __syncthreads();
    const int d = tid % LD * 8, gs = tid / LD;
    float y[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) y[k] = 0.0f;
    for (int s = gs; s < I.splits; s += GS) {
        const float* p = P.part + (at + s * step) * D + d;
        const pg_f4 x0 = *reinterpret_cast<const pg_f4*>(p), x1 = *reinterpret_cast<const pg_f4*>(p + 4);
        const float b = weight[s];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            y[k] += x0[k] * b;
            y[4 + k] += x1[k] * b;
        }
    }
    *reinterpret_cast<pg_f4*>(&part[gs][d]) = pg_f4{y[0], y[1], y[2], y[3]};
    *reinterpret_cast<pg_f4*>(&part[gs][d + 4]) = pg_f4{y[4], y[5], y[6], y[7]};
    __syncthreads();
    if (gs) return;
    for (int i = 1; i < min(GS, I.splits); ++i)
#pragma unroll
        for (int k = 0; k < 8; ++k) y[k] += part[i][d + k];
    den = red[1][0] + red[1][1] + red[1][2] + red[1][3];
    const int r = rr / G, h = rr - r * G;
    const bool empty = P.causal ? I.len - I.n + r + 1 <= 0 : I.len == 0;
    const float il = empty ? 0.0f : 1.0f / den;
#pragma unroll
    for (int k = 0; k < 8; ++k) y[k] *= il;
    pg_store8(P, (long long)(g * G + h) * P.o_head + (long long)(I.row + r) * P.o_row + d, y);
}

}  // namespace hm
