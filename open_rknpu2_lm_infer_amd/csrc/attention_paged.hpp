// Kernels of the paged KV cache's attention (include/rk_npu_attention_paged.h).
//
// Layout in HBM, per page and KV head, `page` tokens in tiles of 16:
//   K: [4-key group][D / 8 pieces][4 keys][8 dims]; piece p of group n lies at
//      place p ^ k_turn(n). A lane of a matrix operand takes one piece, lanes of
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

// (0, 2, 3, 1: a 16-byte LDS read takes lanes 0..3, 12..15, 20..27 at a time, in operands
// of 16 keys groups 0 and 3 of one piece with 1 and 2 of the next)
__device__ __forceinline__ constexpr int pg_k_turn(int n) { return (0x78 >> (2 * (n & 3))) & 3; }
__device__ __forceinline__ int pg_k_place(int D, int j, int piece) {  // of piece `piece` of key j, in 8 halves
    return (j >> 2) * (D >> 1) + (piece ^ pg_k_turn(j >> 2)) * 4 + (j & 3);
}
// (heads of 64: two keys fill the 256 bytes of the banks; of 256: operands of 16 dims,
// of 8 keys for 32 lanes at a time)
__device__ __forceinline__ constexpr int pg_v_turn(int D, int j) {
    return D == 64 ? 4 * ((j >> 1) & 1) : D == 128 ? 4 * (j & 3) : 2 * (j & 7);
}
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

// The 16-key tile of the pool that holds KV head g of such a token (of a wrong page:
// tile 0, whose values have no meaning there).
__device__ __forceinline__ int pg_tile(const PagedBatch& B, int s, int g, int token) {
    const int page = pg_page(B, s, token), tiles = 1 << (B.page_shift - 4);
    return page < 0 ? 0 : (page * B.kh + g) * tiles + ((token >> 4) & (tiles - 1));
}

struct AttnPagedParams {
    PagedBatch b;
    const void* q;
    int q_f32;
    long long q_head, q_row;  // strides, elements
    void* out;
    int out_f16;
    long long o_head, o_row;
    float* part;     // accumulators [slot][kh][tile rows][D], then (max, sum) pairs
    int qh, causal;
    float scale;
    int items;       // blocks per KV head
    int slots;       // of partials per KV head
    int target;      // blocks per KV head that splits aim at; 0: no splits
    int least;       // units of a split, at least
    int tile_rows;   // query rows of a block
    int tiles;       // row tiles of the whole batch, at most
    int wave;        // blocks per KV head that a block for each CU are, where long tiles come first; 0: they do not
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
// keys. Partials of split 0 of that tile lie in slot `first`, of split i > 0 in `more` + i.
struct PagedItem {
    int s, row, n, len, tile, split, splits, first, more;
    bool any;
};

// The schedule where sequences of few rows are more than the blocks that splits aim at:
// block s has sequence s, or its first split, blocks from B.sequences on have the further
// splits of long ones: more than P.least units, and more than the batch's units over
// P.target. Who has P.least at most looks at no other sequence. Slots: further splits in
// their order, then, P.target behind each sequence's second one, the first ones. (A join's
// tile is a sequence.)
__device__ __forceinline__ PagedItem pg_item_behind(const AttnPagedParams& P, int at, int lane) {
    const PagedBatch& B = P.b;
    auto units_of = [](const PagedSeq& q) { return q.n > 0 ? (q.len + 31) >> 5 : 0; };
    PagedItem x{};
    PagedSeq own{0, 0, 0};
    if (at < B.sequences) {
        own = pg_seq(B, at);
        x.s = at;
        x.row = own.row;
        x.n = own.n;
        x.len = own.len;
        x.splits = 1;
        x.any = own.n > 0;
        if (units_of(own) <= P.least) return x;
    }
    const int C = (B.sequences + 63) >> 6, end = min(lane * C + C, B.sequences);
    int units = 0;
#pragma unroll 4
    for (int s = lane * C; s < end; ++s) units += units_of(pg_seq(B, s));
    const unsigned total = __builtin_amdgcn_readlane(pg_scan(units), 63);
    const unsigned per = max((unsigned)P.least, (total + P.target - 1) / (unsigned)P.target);
    auto more_of = [&](const PagedSeq& q) {
        return min(PAGED_MAX_SPLITS, max(1, (int)(((unsigned)units_of(q) + per - 1) / per))) - 1;
    };
    int more = 0;
#pragma unroll 4
    for (int s = lane * C; s < end; ++s) more += more_of(pg_seq(B, s));
    const int more_end = pg_scan(more);
    int k = 0, owner, before;
    if (at < B.sequences) {
        owner = at / C;
        before = __builtin_amdgcn_readlane(more_end - more, owner);
        for (int s = owner * C; s < at; ++s) before += more_of(pg_seq(B, s));
    } else {
        k = at - B.sequences;
        const unsigned long long over = __builtin_amdgcn_ballot_w64(more_end > k);
        if (over == 0) return x;
        owner = __builtin_ctzll(over);
        before = __builtin_amdgcn_readlane(more_end - more, owner);
        for (x.s = owner * C; x.s < B.sequences; ++x.s) {
            own = pg_seq(B, x.s);
            if (k < before + more_of(own)) break;
            before += more_of(own);
        }
        x.split = 1 + k - before;
        x.row = own.row;
        x.n = own.n;
        x.len = own.len;
    }
    x.splits = 1 + more_of(own);
    x.first = P.target + before;
    x.more = before - 1;
    // (not so if the lengths changed meanwhile)
    x.any = x.s < B.sequences && x.splits > x.split && before < P.target && x.more + x.splits <= P.target;
    if (x.splits == 1) x.any = at < B.sequences;
    return x;
}

// The schedule, made by every wave from the lengths alone: a sequence has ceil(rows /
// tile_rows) tiles, each split into as many pieces of at least `per` units of 32 keys
// as it has; per is the batch's units over `target`, so that splits of short and long
// sequences take the same time. Blocks of a sequence lie in the order of their tiles,
// the last first (causal ones see the most keys), then splits. Counted by tiles alone
// (`joins`), index `at` is the tile of a join. Lane l has sequences l C..l C + C - 1.
__device__ __forceinline__ PagedItem pg_item(const AttnPagedParams& P, int at, int lane, bool joins) {
    const PagedBatch& B = P.b;
    const int G = P.qh / B.kh, C = (B.sequences + 63) >> 6;
    auto tiles_of = [&](const PagedSeq& q) { return (int)(((unsigned)q.n * (unsigned)G + P.tile_rows - 1) / (unsigned)P.tile_rows); };
    const PagedSeq none{0, 0, 0};
    if (!P.target && !B.offsets && G <= P.tile_rows) {
        // (one row each, not split: block `at` has sequence `at`)
        PagedItem x{};
        x.s = at;
        x.any = at < B.sequences;
        if (!x.any) return x;
        const PagedSeq q = pg_seq(B, at);
        x.row = q.row;
        x.n = q.n;
        x.len = q.len;
        x.splits = 1;
        return x;
    }
    PagedSeq mine = lane * C < B.sequences ? pg_seq(B, lane * C) : none;
    // (one sequence a lane: the one in registers)
    if (!P.target && P.wave > 0 && C == 1) {
        // By tiles' places in their sequences, the last places first: above(k) blocks have
        // places from k on. Where two blocks a CU hold them all, the second ones come in
        // reverse, a short one beside a long one.
        const int t = tiles_of(mine), total = wave_sum(t);
        PagedItem x{};
        x.any = at < total;
        if (!x.any) return x;
        if (total > P.wave) {
            const int i = at >= P.wave && total <= 2 * P.wave ? total - 1 - (at - P.wave) : at;
            auto above = [&](int k) { return wave_sum(max(0, t - k)); };
            int k = 0, end = (int)wave_max((float)t) + 1;
            while (end - k > 1) {
                const int mid = (k + end) >> 1;
                if (above(mid) > i)
                    k = mid;
                else
                    end = mid;
            }
            const unsigned long long has = __builtin_amdgcn_ballot_w64(t > k);
            const int nth = i - above(k + 1);
            const int rank = __builtin_amdgcn_mbcnt_hi((unsigned)(has >> 32), __builtin_amdgcn_mbcnt_lo((unsigned)has, 0));
            x.s = __builtin_ctzll(__builtin_amdgcn_ballot_w64(t > k && rank == nth) | 1ull << 63);
            x.row = __builtin_amdgcn_readlane(mine.row, x.s);
            x.n = __builtin_amdgcn_readlane(mine.n, x.s);
            x.len = __builtin_amdgcn_readlane(mine.len, x.s);
            x.tile = k;
            x.splits = 1;
            return x;
        }
    }
    auto seq = [&](int i) { return C == 1 ? mine : lane * C + i < B.sequences ? pg_seq(B, lane * C + i) : none; };
    unsigned per = 0x7fffffff;
    if (P.target > 0) {
        int units = 0;
#pragma unroll 4
        for (int i = 0; i < C; ++i) {
            const PagedSeq q = seq(i);
            units += tiles_of(q) * ((q.len + 31) >> 5);
        }
        const unsigned total = __builtin_amdgcn_readlane(pg_scan(units), 63);
        per = max((unsigned)P.least, (total + P.target - 1) / (unsigned)P.target);
    }
    auto splits_of = [&](const PagedSeq& q) {
        const unsigned units = (unsigned)(q.len + 31) >> 5;
        return P.target > 0 ? min(PAGED_MAX_SPLITS, max(1, (int)((units + per - 1) / per))) : 1;
    };
    int items = 0, tiles = 0;
#pragma unroll 4
    for (int i = 0; i < C; ++i) {
        const PagedSeq q = seq(i);
        const int t = tiles_of(q);
        items += t * splits_of(q);
        tiles += t;
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
        PagedSeq q;
        if (C == 1) {
            q.row = __builtin_amdgcn_readlane(mine.row, owner);
            q.n = __builtin_amdgcn_readlane(mine.n, owner);
            q.len = __builtin_amdgcn_readlane(mine.len, owner);
        } else {
            q = pg_seq(B, x.s);
        }
        const int t = tiles_of(q), p = splits_of(q), count = joins ? t : t * p;
        if (at < before + count) {
            const int in = at - before;
            x.row = q.row;
            x.n = q.n;
            x.len = q.len;
            x.splits = p;
            const int k = joins ? in : in / p;
            x.tile = t - 1 - k;
            x.split = joins ? 0 : in - k * p;
            x.first = x.more = first + k * p;
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

// The same over each 32, in every lane (both halves hold the same).
__device__ __forceinline__ int pg_lo_min(int v) {
    v = pg_row_min(v);
    const auto a = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    return __builtin_amdgcn_readfirstlane(min((int)a[0], (int)a[1]));
}

// A row's maximum before it has seen a key: finite, so that differences are no NaN.
constexpr float PG_NONE = -1e30f;
// The weight 2^d of a partial result whose maximum lies d <= 0 below the row's:
// never 0, so that an infinite accumulator stays one (0 times it is NaN). A finite sum
// gains by that 2^-105 of a key's value at most (weights lie below 2^15), where the row's
// own sum is above 2^5.
__device__ __forceinline__ float pg_weight(float m, float top) {
    return fmaxf(__builtin_amdgcn_exp2f(m - top), 0x1p-120f);
}

// A mean of fp16 values lies in their range. One whose weights are rounded to one fp16
// after they are summed may pass its end by 2^-11, where fp16 has infinities: it is that end.
__device__ __forceinline__ float pg_in_range(float y) {
    return fabsf(y) < INFINITY ? __builtin_amdgcn_fmed3f(y, -65504.0f, 65504.0f) : y;
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

__device__ __forceinline__ void pg_store4(const AttnPagedParams& P, long long at, float a, float b, float c, float d) {
    if (P.out_f16) {
        const unsigned short h0 = __half_as_ushort(__float2half_rn(a)), h1 = __half_as_ushort(__float2half_rn(b));
        const unsigned short h2 = __half_as_ushort(__float2half_rn(c)), h3 = __half_as_ushort(__float2half_rn(d));
        *reinterpret_cast<pg_u2a2*>(static_cast<__half*>(P.out) + at) =
            pg_u2a2{h0 | ((unsigned)h1 << 16), h2 | ((unsigned)h3 << 16)};
    } else {
        *reinterpret_cast<pg_f4a4*>(static_cast<float*>(P.out) + at) = pg_f4a4{a, b, c, d};
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

// Few rows. Block: NW waves over one tile of RW groups of 16 query rows (one of 8 where
// PACK) of one KV head of a sequence; wave w takes units w, w + NW, .. of 32 keys of its
// split, so nothing is shared until the waves' partial (max, sum, accumulators) meet in
// LDS. K comes from memory in operand order; V comes as rows, 8 keys of 8 dims a lane,
// and is transposed there, two keys' halves a v_perm_b32. Weights go into the products
// with V as two fp16. PACK: columns 8..15 are columns 0..7 again and take the second
// fp16, so that both cost one product. A tile holds all rows of a sequence, so pages
// are read once, by loads that leave nothing in the caches.
//
// Measured with the join, contexts not in the last-level cache: one row of 32 heads over 8
// of 128 and 64 sequences of 60 to 8100 tokens (1.08 GB) 182 us, 5.9 TB/s; 2 of 131072 162,
// 6.6 (large reads alone reach 6.7, a copy reads and writes 5.1); cached loads 202 and 214.
// 256 sequences of up to 700 tokens of 8 heads of 64 33 (42). 16 sequences of 2 heads of 256
// 57: 4.6 TB/s, 220 registers leave two blocks a CU. One of 4000 tokens 12.4, latency: launch,
// table, one unit's loads and products, the waves' meeting (8.0), the join (4.4). The next unit's
// loads before this one's products changed nothing with 128 dims and lost with 256 (51 to
// 57: registers).
template <int D, int NW, int RW, bool PACK, bool BEHIND>
__global__ __launch_bounds__(64 * NW) void attn_paged_rows_kernel(AttnPagedParams P) {
    constexpr int KS = D / 32;                  // 32-dim steps of a score
    constexpr int DW = D == 64 ? 4 : 8;         // dims of V a lane takes of a key, H times
    constexpr int H = D / (16 * DW), NB = H * DW;
    constexpr int COLS = PACK ? 8 : 16 * RW, PITCH = D + 4;
    static_assert(RW == 1 || !PACK, "packed columns");
    typedef unsigned u2 __attribute__((ext_vector_type(2)));
    __shared__ __attribute__((aligned(16))) float acc[NW][COLS][PITCH];
    __shared__ float ml[NW][2][COLS];
    const PagedBatch& B = P.b;
    const int g = blockIdx.x % B.kh, at = blockIdx.x / B.kh;
    const int lane = threadIdx.x & 63, lo = lane & 15, hi = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const PagedItem I = BEHIND ? pg_item_behind(P, at, lane) : pg_item(P, at, lane, false);
    if (!I.any) return;  // (block-uniform)
    const int G = P.qh / B.kh, R = G * I.n;
    int lim[RW];
    int open = 0x7fffffff, seen = 0;  // keys below `open` every row sees, from `seen` on none
    pg_h8 qf[RW][KS];
#pragma unroll
    for (int x = 0; x < RW; ++x) {
        const int rr = I.tile * COLS + 16 * x + (PACK ? lo & 7 : lo);
        const bool live = rr < R;
        const int r = live ? rr / G : 0, h = live ? rr - r * G : 0;
        lim[x] = !live ? 0 : P.causal ? max(0, min(I.len, I.len - I.n + r + 1)) : I.len;
        open = min(open, live ? lim[x] : 0x7fffffff);
        seen = max(seen, lim[x]);
        const long long q_at = (long long)(g * G + h) * P.q_head + (long long)(I.row + r) * P.q_row + 8 * hi;
#pragma unroll
        for (int i = 0; i < KS; ++i) qf[x][i] = pg_load_q(P, q_at + 32 * i);
    }
    open = __builtin_amdgcn_readfirstlane(pg_row_min(open));
    seen = -__builtin_amdgcn_readfirstlane(pg_row_min(-seen));
    const int units = (seen + 31) >> 5, each = (units + I.splits - 1) / I.splits;
    const int u_begin = I.split * each, u_end = min(units, u_begin + each);

    const float c = fminf(P.scale * 1.4426950408889634f, 0x1.fffffep127f);
    // Lane l's place in the table of the wave's next 32 units: unit l / 2, half l % 2,
    // as 16-key tiles of the pool.
    auto places = [&](int u) {
        const int token = (u + NW * (lane >> 1)) * 32 + (lane & 1) * 16;
        return token < min(seen, u_end * 32) ? pg_tile(B, I.s, g, token) : 0;
    };
    int place = 0, place_at = -64 * NW;
    v4u kr[2][KS];
    v4u vr[2][4][H];
    auto get = [](const auto* p) __attribute__((always_inline)) { return __builtin_nontemporal_load(p); };
    auto load = [&](int u) __attribute__((always_inline)) {
        if (u - place_at >= 32 * NW) {
            place = places(u);
            place_at = u;
        }
        const int i = (u - place_at) / NW * 2;
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            const size_t tile = (size_t)__builtin_amdgcn_readlane(place, i + t) * (16 * D);
            const __half* kp = B.k + tile;
            const __half* vp = B.v + tile;
#pragma unroll
            for (int s = 0; s < KS; ++s) kr[t][s] = get(reinterpret_cast<const v4u*>(kp + pg_k_place(D, lo, 4 * s + hi) * 8));
#pragma unroll
            for (int k = 0; k < 4; ++k)
#pragma unroll
                for (int w = 0; w < H; ++w) {
                    const int j = 4 * hi + k;
                    if constexpr (D == 64) {
                        const u2 x = get(reinterpret_cast<const u2*>(vp + pg_v_place(D, j, lo >> 1) * 8 + (lo & 1) * 4));
                        vr[t][k][w] = v4u{x[0], x[1], 0u, 0u};
                    } else {
                        vr[t][k][w] = get(reinterpret_cast<const v4u*>(vp + pg_v_place(D, j, 16 * w + lo) * 8));
                    }
                }
        }
    };

    float mrun[RW], lsum[RW];
    pg_f4 o[RW][NB];
#pragma unroll
    for (int x = 0; x < RW; ++x) {
        mrun[x] = PG_NONE;
        lsum[x] = 0.0f;
#pragma unroll
        for (int n = 0; n < NB; ++n) o[x][n] = pg_f4{0.0f, 0.0f, 0.0f, 0.0f};
    }
    bool wild = false;
    const float second = PACK && lo >= 8 ? 1.0f : 0.0f;
    for (int u = u_begin + wave; u < u_end; u += NW) {
        load(u);
        pg_f4 s[RW][2];
#pragma unroll
        for (int x = 0; x < RW; ++x) s[x][0] = s[x][1] = pg_f4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int i = 0; i < KS; ++i)
#pragma unroll
                for (int x = 0; x < RW; ++x)
                    s[x][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(pg_h8, kr[t][i]), qf[x][i], s[x][t], 0, 0, 0);
        if (u * 32 + 32 > open) {  // (uniform)
            unsigned odd = 0;
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const int key = u * 32 + 16 * t + 4 * hi + k;
#pragma unroll
                    for (int x = 0; x < RW; ++x)
                        if (key >= lim[x]) s[x][t][k] = -INFINITY;
                    // (0 times what is not finite is NaN: such a value of a key that not
                    // every row sees is added after the last product)
                    const bool none = key >= seen;
#pragma unroll
                    for (int w = 0; w < H; ++w)
#pragma unroll
                        for (int i = 0; i < DW / 2; ++i) {
                            const unsigned v = vr[t][k][w][i];
                            unsigned drop = (v & 0x7C00u) == 0x7C00u ? 0xFFFFu : 0u;
                            drop |= (v & 0x7C000000u) == 0x7C000000u ? 0xFFFF0000u : 0u;
                            if (key < open) drop = 0u;
                            if (!none) odd |= drop;
                            vr[t][k][w][i] = none ? 0u : v & ~drop;
                        }
                }
            wild |= odd != 0;
        }
        float top[RW];
        bool over = false;
#pragma unroll
        for (int x = 0; x < RW; ++x) {
            float m[2];
#pragma unroll
            for (int t = 0; t < 2; ++t)
                m[t] = __builtin_elementwise_maximum(
                    __builtin_elementwise_maximum(float(s[x][t][0]), float(s[x][t][1])),
                    __builtin_elementwise_maximum(float(s[x][t][2]), float(s[x][t][3])));
            top[x] = c * __builtin_elementwise_maximum(m[0], m[1]);
            over |= top[x] > mrun[x] + (PG_LAZY + PG_SHIFT);
        }
        if (__builtin_amdgcn_ballot_w64(over) != 0) {
#pragma unroll
            for (int x = 0; x < RW; ++x) {
                const float tm = pg_rows4_max(top[x]) - PG_SHIFT;
                if (tm > mrun[x] + PG_LAZY) {
                    const float alpha = __builtin_amdgcn_exp2f(mrun[x] - tm);
                    mrun[x] = tm;
                    lsum[x] *= alpha;
#pragma unroll
                    for (int n = 0; n < NB; ++n) o[x][n] *= alpha;
                }
            }
        }
        pg_h8 ph[RW], pl[RW];
#pragma unroll
        for (int x = 0; x < RW; ++x) {
            float l[2] = {0.0f, 0.0f};
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int k = 0; k < 4; k += 2) {
                    const float p0 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[x][t][k], c, -mrun[x]));
                    const float p1 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[x][t][k + 1], c, -mrun[x]));
                    const pg_h2 y = pg_round2(p0, p1);
                    if constexpr (PACK) {
                        ph[x][4 * t + k] = (_Float16)__builtin_fmaf((float)y[0], -second, p0);
                        ph[x][4 * t + k + 1] = (_Float16)__builtin_fmaf((float)y[1], -second, p1);
                    } else {
                        ph[x][4 * t + k] = y[0];
                        ph[x][4 * t + k + 1] = y[1];
                        pl[x][4 * t + k] = (_Float16)(p0 - (float)y[0]);
                        pl[x][4 * t + k + 1] = (_Float16)(p1 - (float)y[1]);
                    }
                    l[t] += p0 + p1;
                }
            lsum[x] += l[0] + l[1];
        }
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
                const int n = w * DW + d;
#pragma unroll
                for (int x = 0; x < RW; ++x) {
                    o[x][n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(av, ph[x], o[x][n], 0, 0, 0);
                    if constexpr (!PACK) o[x][n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(av, pl[x], o[x][n], 0, 0, 0);
                }
            }
    }
    // Infinities and NaN among the values: the products leave NaN of them (0, or a
    // negative second fp16, times an infinity). A result that they reach is their sum,
    // whatever the weights, which are positive.
#pragma unroll
    for (int x = 0; x < RW; ++x) {
        lsum[x] = pg_rows4_sum(lsum[x]);
#pragma unroll
        for (int n = 0; n < NB; ++n)
#pragma unroll
            for (int k = 0; k < 4; ++k) wild |= !(fabsf(o[x][n][k]) < INFINITY);
    }
    if (__builtin_amdgcn_ballot_w64(wild) != 0) {
#pragma unroll 1
        for (int n = 0; n < NB; ++n) {
            float sum[RW][4] = {};
#pragma unroll 1
            for (int u = u_begin + wave; u < u_end; u += NW) {
#pragma unroll 1
                for (int key = u * 32; key < min(u * 32 + 32, seen); ++key) {
                    const __half* vp = B.v + (size_t)pg_tile(B, I.s, g, key) * (16 * D);
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const int dim = 128 * (n / DW) + (4 * hi + k) * DW + n % DW;
                        const float v = __half2float(vp[pg_v_place(D, key & 15, dim >> 3) * 8 + (dim & 7)]);
#pragma unroll
                        for (int x = 0; x < RW; ++x) sum[x][k] += key < lim[x] && !(fabsf(v) < INFINITY) ? v : 0.0f;
                    }
                }
            }
#pragma unroll
            for (int m = 0; m < NB; ++m)
#pragma unroll
                for (int x = 0; x < RW; ++x)
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        if (m == n) o[x][m][k] = fabsf(sum[x][k]) < INFINITY ? float(o[x][m][k]) : sum[x][k];
        }
    }
    // The waves meet. Lane (lo, hi) has dims 128 w + (4 hi + k) DW + d of its rows.
    if constexpr (PACK) {
#pragma unroll
        for (int n = 0; n < NB; ++n)
#pragma unroll
            for (int k = 0; k < 4; ++k) o[0][n][k] += dpp_move<0x128>(float(o[0][n][k]));  // row_ror:8
    }
    if (!PACK || lo < 8) {
#pragma unroll
        for (int x = 0; x < RW; ++x) {
#pragma unroll
            for (int w = 0; w < H; ++w)
#pragma unroll
                for (int k = 0; k < 4; ++k)
#pragma unroll
                    for (int d = 0; d < DW; d += 4) {
                        const int n = w * DW + d;
                        *reinterpret_cast<pg_f4*>(&acc[wave][16 * x + lo][128 * w + (4 * hi + k) * DW + d]) =
                            pg_f4{o[x][n][k], o[x][n + 1][k], o[x][n + 2][k], o[x][n + 3][k]};
                    }
            if (hi == 0) {
                ml[wave][0][16 * x + lo] = mrun[x];
                ml[wave][1][16 * x + lo] = lsum[x];
            }
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
            const size_t row_at = ((size_t)(I.split ? I.more + I.split : I.first) * B.kh + g) * COLS + row;
            float* p = P.part + row_at * D + d;
            *reinterpret_cast<pg_f4*>(p) = pg_f4{y[0], y[1], y[2], y[3]};
            *reinterpret_cast<pg_f4*>(p + 4) = pg_f4{y[4], y[5], y[6], y[7]};
            if (d == 0)
                *reinterpret_cast<float2*>(P.part + (size_t)P.slots * B.kh * COLS * D + row_at * 2) = float2{top, l};
        }
    }
}

// Many rows. Block: NW waves with W rows of one KV head of a sequence each; stages of U
// units of 32 keys come through LDS, a 16-key tile of K or of V a wave (or half a one).
// Operands of v_mfma_f32_32x32x16_f16 (W 32) and _16x16x32_ (W 16): A lane l = row
// l % W, k-slots 8 (l / W)..+7; C lane l = rows 8 b + 4 (l / 32)..+3, b < 4, or 4 (l / 16)..+3,
// of column l % W: again what B of O^T += V^T P^T wants, once V's slots name the same
// keys (ds_read_b64_tr_b16 hands lane l of 16 one dim of 4 keys).
//
// In step j a wave turns the scores of unit j into weights, computes those of unit
// j + 1 and multiplies V of unit j - 1: one straight piece of code in which matrix and
// vector instructions do not depend on each other. In stage t K of stage t + 2 and V of
// stage t + U - 1 go to LDS, loaded in the stage before.
//
// f32 output takes V's products twice, with 22 bits of a weight (SPLIT). fp16 output, which
// rounds by 2^-11 itself, takes them once: outputs are 2.9e-4 off instead of 2.0e-4 (twice
// cost 850 us for 631 in the first case below, 72 for 61 in the second, 512 rows of 8 heads
// of 64 after 8000 tokens 81 for 65; who wants more has f32 output). W: 32 rows a wave halve
// the LDS reads of a product; of 256 dims they need 448 registers, one wave a SIMD (57600
// keys, 1024 rows of 2 heads 239 us, with 16 rows 202; 4-wave blocks of 64 rows 267).
//
// Measured with the join: 512 rows of 32 heads over 8 of 128 after 65000 tokens 556 us, 0.98
// PFLOP/s of a large matrix product's 1.17; matrix cores 55 % busy, LDS 35 %, at 1.7 to 1.8
// GHz: the power limit holds the clock. LDS reads without turned places 28 % longer. 6
// prompts of 17 to 1365 rows 55 us: a long prompt's last block walks 43 units alone or beside
// one other (1.9 waves a SIMD of a busy CU). 100 to 200 rows of 16 heads over 2 of 256, f32
// output, 72: matrix cores 43 % busy (51 % and 1.5 GHz over longer contexts), two fp16 for a
// weight, the join 10. Matrix and vector instructions or LDS reads put in turns by scheduling
// groups: no difference of 128 dims or 256.
template <int D, int W, int U, int NW, bool SPLIT>
__global__ __launch_bounds__(64 * NW) void attn_paged_tile_kernel(AttnPagedParams P) {
    constexpr int CL = W * W / 64;                 // values of a lane in a C operand
    constexpr int SN = 32 / W, NS = SN * CL;       // C operands of a unit's scores, a lane's scores
    constexpr int KS = D * W / 512;                // steps of a score: 512 / W dims
    constexpr int NB = D / W, VS = NS / 8;         // C operands of the output, key steps of a unit
    constexpr int BUFS = U + 1, VA = U - 1, ROWS = NW * W;
    constexpr int TILE = 32 * D;                   // bytes of 16 keys of K or V
    constexpr int STAGE = 2 * U * TILE;            // of a stage's K, or V
    constexpr int WT = NW / (4 * U);               // waves of a tile
    constexpr int PT = TILE / 1024 / WT;           // 16-byte pieces of a lane's
    constexpr float LAZY = SPLIT ? 8.0f : 6.0f, SHIFT = (SPLIT ? 14.0f : 15.0f) - LAZY;
    static_assert(NW % (4 * U) == 0 && (U == 1 || U == 2) && (W == 16 || W == 32), "stage shape");
    static_assert(NW * W * 128 <= 2 * BUFS * STAGE, "room for the rows on their way out");
    typedef float fv __attribute__((ext_vector_type(CL)));
    typedef short s4 __attribute__((ext_vector_type(4)));
    typedef short s8 __attribute__((ext_vector_type(8)));
    typedef __attribute__((address_space(3))) s4 lds_s4;
    __shared__ __attribute__((aligned(1024))) uint8_t smem[2 * BUFS * STAGE];
    __shared__ int dropped;
    const PagedBatch& B = P.b;
    const int g = blockIdx.x % B.kh, at = blockIdx.x / B.kh;
    const int tid = threadIdx.x, lane = tid & 63, lo = lane % W, hi = lane / W;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const PagedItem I = pg_item(P, at, lane, false);
    if (!I.any) return;  // (block-uniform)
    const int G = P.qh / B.kh, R = G * I.n;
    const int rr = (I.tile * NW + wave) * W + lo;
    const bool live = rr < R;
    const int r = live ? rr / G : 0, h = live ? rr - r * G : 0;
    const int before = I.len - I.n;  // tokens before the rows' (causal)
    const int lim = !live ? 0 : P.causal ? max(0, min(I.len, before + r + 1)) : I.len;
    // keys below `open` every row of the wave sees (none without rows: what lies behind a
    // sequence may be NaN)
    const int first = live ? lim : 0x7fffffff, least = W == 32 ? pg_lo_min(first) : __builtin_amdgcn_readfirstlane(pg_row_min(first));
    const int open = least == 0x7fffffff ? 0 : least;
    // keys that the block's last row sees, their units, and this block's
    const int last = min(R, (I.tile + 1) * ROWS) - 1;
    const int seen = P.causal ? max(0, min(I.len, before + last / G + 1)) : I.len, all = (seen + 31) >> 5;
    const int each = (all + I.splits - 1) / I.splits;
    const int u_begin = I.split * each, u_end = min(all, u_begin + each);
    const int stages = (max(0, u_end - u_begin) + U - 1) / U;

    pg_h8 qf[KS];
    const long long q_at = (long long)(g * G + h) * P.q_head + (long long)(I.row + r) * P.q_row + 8 * hi;
#pragma unroll
    for (int i = 0; i < KS; ++i) qf[i] = pg_load_q(P, q_at + 512 / W * i);
    const float c = fminf(P.scale * 1.4426950408889634f, 0x1.fffffep127f);

    // The first half of the waves loads K, the other V. Lane l has the place of the
    // wave's tile in stage `place_at` + l.
    const bool isv = wave >= NW / 2;
    const int tile = wave % (NW / 2) / WT, part = wave % WT;
    const __half* pool = isv ? B.v : B.k;
    int place = 0, place_at = -64;
    v4u raw[PT];
    auto load = [&](int t) __attribute__((always_inline)) {
        if (t - place_at >= 64) {
            const int token = ((u_begin + (t + lane) * U) * 2 + tile) * 16;
            place = token < min(u_end * 32, I.len) ? pg_tile(B, I.s, g, token) : 0;
            place_at = t;
        }
        const __half* from = pool + (size_t)__builtin_amdgcn_readlane(place, t - place_at) * (16 * D) + (part * PT * 64 + lane) * 8;
#pragma unroll
        for (int i = 0; i < PT; ++i) raw[i] = *reinterpret_cast<const v4u*>(from + i * 512);
    };
    // (K's buffers, then V's; b: stage % BUFS)
    uint8_t* const mine = smem + (isv ? BUFS * STAGE : 0) + tile * TILE + part * PT * 1024 + lane * 16;
    // Values of V of keys that not every row of the block sees: what is not finite stays
    // out of the products (0 times it is NaN) and is added after the last one.
    const int sure = min(u_end * 32, P.causal ? max(0, min(I.len, before + I.tile * ROWS / G + 1)) : I.len);
    auto store = [&](int t, int b) __attribute__((always_inline)) {
        const int key0 = ((u_begin + t * U) * 2 + tile) * 16;
        if (__builtin_expect(isv && key0 + 16 > sure, 0)) {  // (uniform)
            bool odd = false;
#pragma unroll
            for (int i = 0; i < PT; ++i) {
                const int key = key0 + ((part * PT + i) * 64 + lane) / (D / 8);
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    unsigned drop = (raw[i][k] & 0x7C00u) == 0x7C00u ? 0xFFFFu : 0u;
                    drop |= (raw[i][k] & 0x7C000000u) == 0x7C000000u ? 0xFFFF0000u : 0u;
                    if (key < sure) drop = 0u;
                    odd |= drop != 0 && key < min(seen, u_end * 32);
                    raw[i][k] &= ~drop;
                }
            }
            if (odd) dropped = 1;
        }
#pragma unroll
        for (int i = 0; i < PT; ++i) *reinterpret_cast<v4u*>(mine + b * STAGE + i * 1024) = raw[i];
    };

    float mrun = PG_NONE, lsum = 0.0f;
    fv o[NB];
#pragma unroll
    for (int n = 0; n < NB; ++n) o[n] = fv{};
    bool wild = false;
    if (tid == 0) dropped = 0;
    __syncthreads();
    if (stages > 0) {
        // (zeros for V of stage -1, whose weights are 0)
        load(0);
        if (U == 2 || !isv) store(0, 0);
        if (isv) {
#pragma unroll
            for (int i = 0; i < PT; ++i) *reinterpret_cast<v4u*>(mine + (BUFS - 1) * STAGE + i * 1024) = v4u{0u, 0u, 0u, 0u};
        } else {
            load(1);
            store(1, 1);
        }
        // In stage t: K of t + 2, V of t + VA.
        if (U == 2 || !isv) load(isv ? VA : 2);
        __syncthreads();
        const int j4 = lane & 3;
        // lane's pieces of K: key lo of the unit or tile, pieces 64 / W i + hi
        const int kat = (W == 32 ? (lo >> 4) * TILE : 0) + ((lo & 15) >> 2) * (8 * D) + ((hi ^ pg_k_turn(lo >> 2)) * 4 + j4) * 16;
        auto kop = [&](const uint8_t* unit, int i) {
            return *reinterpret_cast<const pg_h8*>(unit + (W == 32 ? (kat ^ ((i & 1) * 128)) + (i >> 1) * 256 : kat + i * 256));
        };
        // lane's 4 halves of V: key 4 hi + (lane % 16) / 4 of 8 or 16, dims W n + 16 (lo / 16) + 4 (lane % 4)
        const int vj = 4 * hi + ((lane & 15) >> 2);
        const int vat = vj * 2 * D + (((lo >> 4) * 2 + (j4 >> 1)) ^ pg_v_turn(D, vj)) * 16 + (j4 & 1) * 8;
        auto vop = [&](const uint8_t* unit, int n, int t) {
            constexpr int MOST = 256 / (2 * W) - 1;  // (places turn within 256 bytes)
            const uint8_t* p = unit + (vat ^ ((n & MOST) * (2 * W))) + n / (MOST + 1) * 256 + t * TILE;
            const s4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)p);
            const s4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)(p + (W == 32 ? 16 * D : TILE)));
            return __builtin_bit_cast(pg_h8, s8{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]});
        };
        auto mfma = [](pg_h8 a, pg_h8 b, fv x) __attribute__((always_inline)) {
            if constexpr (W == 32)
                return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, x, 0, 0, 0);
            else
                return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, x, 0, 0, 0);
        };
        auto masked = [&](int j) { return (u_begin + j) * 32 + 32 > open || u_begin + j >= u_end; };
        // (unit `sub` of the stage in buffers b)
        auto scores = [&](fv (&s)[SN], int b, int sub) __attribute__((always_inline)) {
            const uint8_t* k = smem + b * STAGE + sub * (2 * TILE);
#pragma unroll
            for (int x = 0; x < SN; ++x) {
                s[x] = fv{};
#pragma unroll
                for (int i = 0; i < KS; ++i) s[x] = mfma(kop(k + x * TILE, i), qf[i], s[x]);
            }
        };
        auto products = [&](int b, int sub, const pg_h8 (&ph)[VS], const pg_h8 (&pl)[VS]) __attribute__((always_inline)) {
            const uint8_t* v = smem + (BUFS + b) * STAGE + sub * (2 * TILE);
#pragma unroll
            for (int n = 0; n < NB; ++n)
#pragma unroll
                for (int t = 0; t < VS; ++t) {
                    const pg_h8 a = vop(v, n, t);
                    o[n] = mfma(a, ph[t], o[n]);
                    if constexpr (SPLIT) o[n] = mfma(a, pl[t], o[n]);
                }
        };
        // What a unit's scores need before they are weighed: masks, and whether a
        // maximum moves.
        float top = 0.0f;
        auto look = [&](int j, fv (&s)[SN]) __attribute__((always_inline)) {
            if (__builtin_expect(masked(j), 0)) {  // (uniform)
                const bool none = u_begin + j >= u_end;
#pragma unroll
                for (int i = 0; i < NS; ++i) {
                    const int key = (u_begin + j) * 32 + (W == 32 ? 8 : 16) * (i >> 2) + 4 * hi + (i & 3);
                    if (none || key >= lim) s[i / CL][i % CL] = -INFINITY;
                }
            }
            float m[NS / 4];
#pragma unroll
            for (int i = 0; i < NS / 4; ++i) {
                const fv& x = s[4 * i / CL];
                const int k = 4 * i % CL;
                m[i] = __builtin_elementwise_maximum(__builtin_elementwise_maximum(float(x[k]), float(x[k + 1])),
                                                     __builtin_elementwise_maximum(float(x[k + 2]), float(x[k + 3])));
            }
            top = __builtin_elementwise_maximum(m[0], m[1]);
            if constexpr (NS == 16) top = __builtin_elementwise_maximum(top, __builtin_elementwise_maximum(m[2], m[3]));
            top *= c;
            return __builtin_amdgcn_ballot_w64(top > mrun + (LAZY + SHIFT)) != 0;
        };
        auto weigh = [&](const fv (&s)[SN], pg_h8 (&ph)[VS], pg_h8 (&pl)[VS]) __attribute__((always_inline)) {
            float l[NS / 4];
#pragma unroll
            for (int i = 0; i < NS; i += 2) {
                const float p0 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i / CL][i % CL], c, -mrun));
                const float p1 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i / CL][i % CL + 1], c, -mrun));
                const pg_h2 x = pg_round2(p0, p1);
                ph[i >> 3][i & 7] = x[0];
                ph[i >> 3][(i & 7) + 1] = x[1];
                if constexpr (SPLIT) {
                    pl[i >> 3][i & 7] = (_Float16)(p0 - (float)x[0]);
                    pl[i >> 3][(i & 7) + 1] = (_Float16)(p1 - (float)x[1]);
                }
                l[i >> 2] = i & 2 ? l[i >> 2] + (p0 + p1) : p0 + p1;
            }
            float sum = l[0] + l[1];
            if constexpr (NS == 16) sum += l[2] + l[3];
            lsum += sum;
        };
        fv sa[SN], sb[SN];
        pg_h8 pha[VS], pla[VS], phb[VS], plb[VS];
#pragma unroll
        for (int t = 0; t < VS; ++t) pha[t] = pla[t] = phb[t] = plb[t] = pg_h8{};
        scores(sa, 0, 0);
        bool moves = look(0, sa);
        // Unit j, the sub-th of stage t, whose buffers are b (bp, bn: those of the stages
        // before and after): s and (ph0, pl0) in, of this unit and the one before; sn and
        // (ph1, pl1) out, of the next and this one. A stage's first unit waits for the
        // stage and fills a later one.
        auto step = [&](int t, int sub, int bp, int b, int bn, fv (&s)[SN], pg_h8 (&ph0)[VS], pg_h8 (&pl0)[VS],
                        fv (&sn)[SN], pg_h8 (&ph1)[VS], pg_h8 (&pl1)[VS]) __attribute__((always_inline)) {
            if (sub == 0) __syncthreads();
            if (__builtin_expect(moves, 0)) {  // (uniform)
                // (whole powers of 2: the weights that wait to be added have the old maximum)
                float tm;
                if constexpr (W == 32) {
                    const auto x = __builtin_amdgcn_permlane32_swap(__float_as_uint(top), __float_as_uint(top), false, false);
                    tm = fmaxf(__uint_as_float(x[0]), __uint_as_float(x[1]));
                } else {
                    tm = pg_rows4_max(top);
                }
                tm = __builtin_ceilf(tm) - SHIFT;
                if (tm > mrun + LAZY) {
                    const float alpha = __builtin_amdgcn_exp2f(mrun - tm);
                    mrun = tm;
                    lsum *= alpha;
                    // (alpha may lie below fp16's range, and the weights that it scales up to 2^15:
                    // two factors, or f32 where both halves are split again. f32 for both, 65000
                    // keys and 512 rows of 8 heads of 128: 653 us, with two factors 640)
                    if constexpr (SPLIT) {
#pragma unroll
                        for (int t = 0; t < VS; ++t)
#pragma unroll
                            for (int i = 0; i < 8; i += 2) {
                                const float p0 = ((float)ph0[t][i] + (float)pl0[t][i]) * alpha;
                                const float p1 = ((float)ph0[t][i + 1] + (float)pl0[t][i + 1]) * alpha;
                                const pg_h2 x = pg_round2(p0, p1);
                                ph0[t][i] = x[0];
                                ph0[t][i + 1] = x[1];
                                pl0[t][i] = (_Float16)(p0 - (float)x[0]);
                                pl0[t][i + 1] = (_Float16)(p1 - (float)x[1]);
                            }
                    } else {
                        const _Float16 a = (_Float16)fmaxf(alpha, 0x1p-24f);
                        const _Float16 rest = (_Float16)(alpha < 0x1p-24f ? alpha * 0x1p24f : 1.0f);
#pragma unroll
                        for (int t = 0; t < VS; ++t) ph0[t] = ph0[t] * a * rest;
                    }
#pragma unroll
                    for (int n = 0; n < NB; ++n) o[n] *= alpha;
                }
            }
            if (sub == 0) {
                // (U = 2, three buffers: t + 2 is in those of t - 1; U = 1, two: in t's)
                store(isv ? t + VA : t + 2, isv ? (U == 2 ? bn : b) : (U == 2 ? bp : b));
                load(isv ? t + VA + 1 : t + 3);
            }
            scores(sn, sub == U - 1 ? bn : b, sub == U - 1 ? 0 : sub + 1);
            weigh(s, ph1, pl1);
            products(sub == 0 ? bp : b, sub == 0 ? U - 1 : sub - 1, ph0, pl0);
            moves = look(t * U + sub + 1, sn);
        };
        int b = 0, bn = 1, bp = BUFS - 1;
        auto next = [&] {
            bp = b;
            b = bn;
            bn = bn == BUFS - 1 ? 0 : bn + 1;
        };
        if constexpr (U == 2) {
            for (int t = 0; t < stages; ++t) {
                step(t, 0, bp, b, bn, sa, pha, pla, sb, phb, plb);
                step(t, 1, bp, b, bn, sb, phb, plb, sa, pha, pla);
                next();
            }
        } else {
            // (an odd count: one stage more than there is, its scores masked)
            for (int t = 0; t < stages; t += 2) {
                step(t, 0, bp, b, bn, sa, pha, pla, sb, phb, plb);
                next();
                step(t + 1, 0, bp, b, bn, sb, phb, plb, sa, pha, pla);
                next();
            }
        }
        __syncthreads();
        products(bp, U - 1, pha, pla);
        wild = dropped != 0;
    }
    if constexpr (W == 32) {
        const auto x = __builtin_amdgcn_permlane32_swap(__float_as_uint(lsum), __float_as_uint(lsum), false, false);
        lsum = __uint_as_float(x[0]) + __uint_as_float(x[1]);
    } else {
        lsum = pg_rows4_sum(lsum);
    }
    // Infinities and NaN among the values: the products leave NaN of them (0, or a
    // negative second fp16, times an infinity). A result that they reach is their sum,
    // whatever the weights, which are positive. (Lane: dims W n + 8 b + 4 hi..+3.)
    float most = 0.0f;
#pragma unroll
    for (int n = 0; n < NB; ++n)
#pragma unroll
        for (int k = 0; k < CL; ++k) {
            wild |= !(fabsf(o[n][k]) < INFINITY);
            most = fmaxf(most, fabsf(o[n][k]));
        }
    if (__builtin_expect(__builtin_amdgcn_ballot_w64(wild) != 0, 0)) {
#pragma unroll 1
        for (int n = 0; n < NB; ++n) {
            fv sum = {};
#pragma unroll 1
            for (int key = u_begin * 32; key < min(u_end * 32, seen); ++key) {
                const __half* vp = B.v + (size_t)pg_tile(B, I.s, g, key) * (16 * D);
#pragma unroll
                for (int k = 0; k < CL; ++k) {
                    const int dim = W * n + 8 * (k >> 2) + 4 * hi + (k & 3);
                    const float x = __half2float(vp[pg_v_place(D, key & 15, dim >> 3) * 8 + (dim & 7)]);
                    sum[k] += key < lim && !(fabsf(x) < INFINITY) ? x : 0.0f;
                }
            }
#pragma unroll
            for (int m = 0; m < NB; ++m)
#pragma unroll
                for (int k = 0; k < CL; ++k)
                    if (m == n) o[m][k] = fabsf(sum[k]) < INFINITY ? float(o[m][k]) : float(sum[k]);
        }
    }
    // Rows leave 32 dims at a time through LDS, so that 8 lanes store a row's 128 bytes:
    // 16-byte pieces, piece p of row r at place p ^ (r & 7).
    __syncthreads();
    float il = I.splits > 1 ? 1.0f : lim == 0 ? 0.0f : 1.0f / lsum;
    if (!SPLIT && I.splits == 1 && __builtin_expect(__builtin_amdgcn_ballot_w64(wild || most * il > 65504.0f) != 0, 0)) {
#pragma unroll
        for (int n = 0; n < NB; ++n)
#pragma unroll
            for (int k = 0; k < CL; ++k) o[n][k] = pg_in_range(o[n][k] * il);
        il = 1.0f;
    }
    const size_t part_at = ((size_t)at * B.kh + g) * ROWS + W * wave;
    if (I.splits > 1 && hi == 0 && live)
        *reinterpret_cast<float2*>(P.part + (size_t)P.slots * B.kh * ROWS * D + (part_at + lo) * 2) = float2{mrun, lsum};
    const long long own = I.splits > 1 ? (long long)(part_at + lo) * D
                                       : (long long)(g * G + h) * P.o_head + (long long)(I.row + r) * P.o_row;
    uint8_t* const box = smem + wave * (W * 128);
    constexpr int LR = W / 8;  // rows of a lane
    long long to[LR];
    bool write[LR];
#pragma unroll
    for (int i = 0; i < LR; ++i) {
        const int row = (lane >> 3) + 8 * i;
        to[i] = __shfl(own, row) + 4 * (lane & 7);
        write[i] = (I.tile * NW + wave) * W + row < R;
    }
#pragma unroll
    for (int x = 0; x < D / 32; ++x) {
#pragma unroll
        for (int k = 0; k < 32 * W / 64; k += 4) {
            const int n = (32 * x) / W + k / CL, piece = W == 32 ? 2 * (k >> 2) + hi : 4 * (k / CL) + hi;
            *reinterpret_cast<pg_f4*>(box + lo * 128 + ((piece ^ (lo & 7)) * 16)) =
                pg_f4{o[n][k % CL] * il, o[n][k % CL + 1] * il, o[n][k % CL + 2] * il, o[n][k % CL + 3] * il};
        }
        pg_f4 y[LR];
#pragma unroll
        for (int i = 0; i < LR; ++i) {
            const int row = (lane >> 3) + 8 * i;
            y[i] = *reinterpret_cast<const pg_f4*>(box + row * 128 + (((lane & 7) ^ (row & 7)) * 16));
        }
#pragma unroll
        for (int i = 0; i < LR; ++i) {
            if (!write[i]) continue;
            if (I.splits > 1)
                *reinterpret_cast<pg_f4*>(P.part + to[i] + 32 * x) = y[i];
            else
                pg_store4(P, to[i] + 32 * x, y[i][0], y[i][1], y[i][2], y[i][3]);
        }
    }
}

// The splits' partials of RPB rows of one row tile and KV head: out = sum_s w_s acc_s /
// sum_s w_s l_s with w_s = 2^(m_s - max m). T = 256 / RPB threads a row, thread t with 4
// dims of every GS-th split; their first loads do not wait for the weights, which the
// row's threads find meanwhile; sums over the GS groups meet in LDS.
//
// Measured: one row of 32 heads, 32 splits 4.7 us; 2048 rows of 8 heads, 4 splits (33 MB
// read) 11 (36 with a block a row).
template <int D, int RPB, bool BEHIND>
__global__ __launch_bounds__(256) void attn_paged_join_kernel(AttnPagedParams P) {
    constexpr int T = 256 / RPB, LD = D / 4, GS = T / LD, AHEAD = 8, W = PAGED_MAX_SPLITS / T;
    static_assert(GS >= 1 && T % LD == 0 && T >= 16, "threads per row");
    __shared__ float weight[RPB][PAGED_MAX_SPLITS];
    __shared__ float red[RPB][2][T / 64 + 1];
    __shared__ pg_f4 part[RPB][GS][LD];
    const PagedBatch& B = P.b;
    const int g = blockIdx.x, tid = threadIdx.x, lane = tid & 63;
    const PagedItem I = BEHIND ? pg_item_behind(P, blockIdx.y, lane) : pg_item(P, blockIdx.y, lane, true);
    // (a block past the grid of the batch's wrong offsets has written nothing)
    if (!I.any || I.splits == 1 || I.more + I.splits > P.slots) return;
    const int G = P.qh / B.kh, R = min(G * I.n - I.tile * P.tile_rows, P.tile_rows), row0 = blockIdx.z * RPB;
    if (row0 >= R) return;  // (block-uniform)
    const int mine = tid / T, t = tid % T, d4 = t % LD, gs = t / LD, S = I.splits;
    const int row = min(row0 + mine, R - 1);  // (threads past the last row: that row again, not written)
    // (split i's row lies i steps from that of slot `more`, the first one's `zero`)
    const long long step = (long long)B.kh * P.tile_rows, at = ((long long)I.more * B.kh + g) * P.tile_rows + row;
    const long long zero = (long long)(I.first - I.more) * step;
    const pg_f4* acc = reinterpret_cast<const pg_f4*>(P.part) + at * LD + d4;
    pg_f4 v[AHEAD];
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) v[i] = acc[(i || gs ? min(gs + i * GS, S - 1) * step : zero) * LD];
    const float2* ml = reinterpret_cast<const float2*>(P.part + (size_t)P.slots * step * D) + at;
    float2 x[W];
    float top = PG_NONE;
#pragma unroll
    for (int i = 0; i < W; ++i) {
        x[i] = t + i * T < S ? ml[i || t ? (t + i * T) * step : zero] : float2{PG_NONE, 0.0f};
        top = fmaxf(top, x[i].x);
    }
#pragma unroll
    for (int i = 1; i < (T < 64 ? T : 64); i <<= 1) top = fmaxf(top, __shfl_xor(top, i));
    if constexpr (T > 64) {
        if (lane == 0) red[mine][0][t / 64] = top;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < T / 64; ++i) top = fmaxf(top, red[mine][0][i]);
    }
    float den = 0.0f;
#pragma unroll
    for (int i = 0; i < W; ++i) {
        const float w = pg_weight(x[i].x, top);
        if (t + i * T < S) weight[mine][t + i * T] = w;
        // (a split that saw NaN scores has a NaN sum)
        den += x[i].y != x[i].y ? x[i].y : w * x[i].y;
    }
#pragma unroll
    for (int i = 1; i < (T < 64 ? T : 64); i <<= 1) den += __shfl_xor(den, i);
    if (T > 64 && lane == 0) red[mine][1][t / 64] = den;
    __syncthreads();
    if constexpr (T > 64) {
        den = 0.0f;
#pragma unroll
        for (int i = 0; i < T / 64; ++i) den += red[mine][1][i];
    }
    pg_f4 num = pg_f4{0.0f, 0.0f, 0.0f, 0.0f};
    for (int s = gs; s < S; s += AHEAD * GS) {
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) {
            if (s + i * GS < S) num += v[i] * weight[mine][s + i * GS];
            v[i] = acc[min(s + (AHEAD + i) * GS, S - 1) * step * LD];
        }
    }
    if constexpr (GS > 1) {
        part[mine][gs][d4] = num;
        __syncthreads();
        if (gs) return;
#pragma unroll
        for (int i = 1; i < GS; ++i) num += part[mine][i][d4];
    }
    if (row0 + mine >= R) return;
    const int rr = I.tile * P.tile_rows + row, r = rr / G, h = rr - r * G;
    const bool empty = P.causal ? I.len - I.n + r + 1 <= 0 : I.len == 0;
    num *= empty ? 0.0f : 1.0f / den;
    if (P.out_f16) num = pg_f4{pg_in_range(num[0]), pg_in_range(num[1]), pg_in_range(num[2]), pg_in_range(num[3])};
    pg_store4(P, (long long)(g * G + h) * P.o_head + (long long)(I.row + r) * P.o_row + 4 * d4, num[0], num[1], num[2], num[3]);
}

// The kernel of a run: attn_paged_tile_kernel in stages of `units` units, or
// attn_paged_rows_kernel, whose tiles hold all rows of a sequence; behind: the latter with
// the schedule of pg_item_behind.
struct PagedPlan {
    bool tile;
    int units;
    bool behind;
};

void launch_attn_paged_64(const AttnPagedParams& P, const PagedPlan& plan, hipStream_t s);
void launch_attn_paged_128(const AttnPagedParams& P, const PagedPlan& plan, hipStream_t s);
void launch_attn_paged_256(const AttnPagedParams& P, const PagedPlan& plan, hipStream_t s);

template <int D, int U>
static void launch_attn_paged_tile(const AttnPagedParams& P, hipStream_t s) {
    constexpr int W = D == 256 ? 16 : 32, NW = 128 * U / W;
    const dim3 grid(P.b.kh * P.items), block(64 * NW);
    if (P.out_f16)
        hipLaunchKernelGGL((attn_paged_tile_kernel<D, W, U, NW, false>), grid, block, 0, s, P);
    else
        hipLaunchKernelGGL((attn_paged_tile_kernel<D, W, U, NW, true>), grid, block, 0, s, P);
}

template <int D, bool BEHIND>
static void launch_attn_paged_rows(const AttnPagedParams& P, hipStream_t s) {
    const dim3 grid(P.b.kh * P.items), block(256);
    if (P.tile_rows == 8)
        hipLaunchKernelGGL((attn_paged_rows_kernel<D, 4, 1, true, BEHIND>), grid, block, 0, s, P);
    else if (P.tile_rows == 16)
        hipLaunchKernelGGL((attn_paged_rows_kernel<D, 4, 1, false, BEHIND>), grid, block, 0, s, P);
    else if constexpr (D < 256)
        hipLaunchKernelGGL((attn_paged_rows_kernel<D, 4, 2, false, BEHIND>), grid, block, 0, s, P);
}

template <int D, bool BEHIND>
static void launch_attn_paged_join(const AttnPagedParams& P, hipStream_t s) {
    // (many rows: as many a block as leave a row the threads for its dims)
    constexpr int MANY = 1024 / D < 8 ? 1024 / D : 8;
    if (P.tiles * P.tile_rows * P.b.kh >= 1024)
        hipLaunchKernelGGL((attn_paged_join_kernel<D, MANY, BEHIND>), dim3(P.b.kh, P.tiles, P.tile_rows / MANY), dim3(256), 0, s, P);
    else
        hipLaunchKernelGGL((attn_paged_join_kernel<D, 1, BEHIND>), dim3(P.b.kh, P.tiles, P.tile_rows), dim3(256), 0, s, P);
}

template <int D>
static void launch_attn_paged(const AttnPagedParams& P, const PagedPlan& plan, hipStream_t s) {
    if (plan.behind) {
        launch_attn_paged_rows<D, true>(P, s);
        launch_attn_paged_join<D, true>(P, s);
        return;
    }
    if (!plan.tile)
        launch_attn_paged_rows<D, false>(P, s);
    else if (D < 256 && plan.units == 2)
        launch_attn_paged_tile<D, D < 256 ? 2 : 1>(P, s);
    else
        launch_attn_paged_tile<D, 1>(P, s);
    if (P.target) launch_attn_paged_join<D, false>(P, s);
}

}  // namespace hm
