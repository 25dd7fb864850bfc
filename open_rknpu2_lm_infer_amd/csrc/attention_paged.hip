// The paged KV cache: its C ABI (include/rk_npu_attention_paged.h), and the kernels
// that write and read its pages. The attention over it: attention_paged.hpp, which
// also gives the layout.

#include <hip/hip_fp16.h>
#include <hip/hip_runtime.h>

#include <algorithm>
#include <climits>
#include <cmath>
#include <cstring>
#include <new>

#include "attention.hpp"
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Wunused-function"  // (the headers' other kernels)
#include "attention_paged.hpp"
#pragma clang diagnostic pop
#include "launch.hpp"

namespace hm {

constexpr uint32_t MAGIC_PAGED_POOL = 0x47504841u;

// 8 values of a row in f32, and 8 as fp16 or f32, of any alignment.
__device__ __forceinline__ void pg_get8(const HeadsView& a, long long at, float (&x)[8]) {
    if (a.f32) {
        const float* p = static_cast<const float*>(a.data) + at;
        const pg_f4a4 u = *reinterpret_cast<const pg_f4a4*>(p), v = *reinterpret_cast<const pg_f4a4*>(p + 4);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            x[i] = u[i];
            x[4 + i] = v[i];
        }
    } else {
        const pg_h8 u = __builtin_bit_cast(
            pg_h8, v4u(*reinterpret_cast<const pg_u4a2*>(static_cast<const __half*>(a.data) + at)));
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = (float)u[i];
    }
}
__device__ __forceinline__ v4u pg_halves(const float (&x)[8]) {
    pg_h8 h;
#pragma unroll
    for (int i = 0; i < 8; ++i) h[i] = (_Float16)x[i];
    return __builtin_bit_cast(v4u, h);
}
__device__ __forceinline__ void pg_put8(const HeadsView& a, long long at, const float (&x)[8]) {
    if (a.f32) {
        float* p = static_cast<float*>(a.data) + at;
        *reinterpret_cast<pg_f4a4*>(p) = pg_f4a4{x[0], x[1], x[2], x[3]};
        *reinterpret_cast<pg_f4a4*>(p + 4) = pg_f4a4{x[4], x[5], x[6], x[7]};
    } else {
        *reinterpret_cast<pg_u4a2*>(static_cast<__half*>(a.data) + at) = pg_u4a2(pg_halves(x));
    }
}

struct PagedRowsParams {
    PagedBatch b;
    HeadsView k, v, q, q_out;  // (data nullptr: none)
    const int* positions;
    const double* turns;       // frequencies in turns (radians / 2 pi) per position
    int D, qh, rotary, interleaved, heads_per_block;
};

// A row's token (-1: none) and page (-1: none), the same for all of a block's threads.
struct PagedRow {
    int token, page;
};
__device__ __forceinline__ PagedRow pg_row(const PagedBatch& B, int row, int* found) {
    int s = row < B.sequences ? row : -1;
    if (B.offsets) {
        if (threadIdx.x == 0) *found = -1;
        __syncthreads();
        for (int i = threadIdx.x; i < B.sequences; i += 256) {
            const int a = B.offsets[i], b = B.offsets[i + 1];
            if (a < 0 || b < a || b > B.rows || b - a > B.max_rows)
                pg_flaw(B);
            else if (a <= row && row < b)
                *found = i;  // (of overlapping offsets: one of them)
        }
        __syncthreads();
        s = __builtin_amdgcn_readfirstlane(*found);
    }
    PagedRow x{-1, -1};
    if (s < 0) return x;
    const PagedSeq q = pg_seq(B, s);
    const int t = q.len - q.n + (row - q.row);
    if (t < 0 || t >= q.len) return x;
    x.token = t;
    x.page = pg_page(B, s, t);
    return x;
}
// The row of block b. Blocks go to the 8 XCDs in turn, so 16 rows' blocks are 8 apart:
// the 4 tokens of a line of K, 16 bytes each, meet in one L2 (3677 rows' append 38 us, 40
// in the blocks' order, their read-back 8.9 and 10.5, 262144 rows of 8 heads 0.92 ms and 1.04).
__device__ __forceinline__ int pg_block_row(int b, int rows) {
    return b < (rows & ~127) ? (b & ~127) + (b & 7) * 16 + ((b >> 3) & 15) : b;
}
// Where a row's piece of 8 dims lies in its page.
__device__ __forceinline__ size_t pg_at(const PagedBatch& B, int D, const PagedRow& x, int g, bool v, int piece) {
    const int place = x.token & ((1 << B.page_shift) - 1), j = place & 15;
    return ((((size_t)x.page * B.kh + g) << B.page_shift) + (place & ~15)) * D +
           (size_t)(v ? pg_v_place(D, j, piece) : pg_k_place(D, j, piece)) * 8;
}

constexpr int PAGED_APPEND_UNITS = 2;  // 16-value units of a thread

// Append. Block: one row of some of the heads, counted q heads, K heads, V heads. A
// thread takes two units of 16 values of a row, each the two pieces of 8 dims that turn
// into each other (or neighbours); their loads come first, as the row's place, three
// loads that wait for one another, has nothing to do with them. The angle's 64-bit
// product and its reduction cost one multiplication and one rounding a pair; sine and
// cosine of a row are computed once, into LDS.
//
// Measured: one row each of 64 sequences, 32 + 16 heads of 128, 5.0 us: launch, three
// memory round trips, sine and cosine, a store (6.0 with the loads last). 3677 f32 rows
// 36: 3.7 TB/s read and written, two rounds of blocks; 14 where the rows are still in the
// last-level cache.
__global__ __launch_bounds__(256) void paged_append_kernel(PagedRowsParams P) {
    __shared__ float2 turn[128];
    __shared__ int found;
    const PagedBatch& B = P.b;
    const int tid = threadIdx.x, row = pg_block_row(blockIdx.x, B.rows), qh = P.qh;
    const int per_head = P.D >> 4, h0 = blockIdx.y * P.heads_per_block, hn = min(P.heads_per_block, qh + 2 * B.kh - h0);
    const int turned_units = P.rotary >> 4;
    float x[PAGED_APPEND_UNITS][8], y[PAGED_APPEND_UNITS][8];
    int kind[PAGED_APPEND_UNITS], g[PAGED_APPEND_UNITS], a[PAGED_APPEND_UNITS], b[PAGED_APPEND_UNITS];
#pragma unroll
    for (int n = 0; n < PAGED_APPEND_UNITS; ++n) {
        const int i = n * 256 + tid, unit = i % per_head, h = h0 + i / per_head;
        kind[n] = i >= hn * per_head ? -1 : h < qh ? 0 : h < qh + B.kh ? 1 : 2;
        if (kind[n] < 0) continue;
        g[n] = kind[n] == 0 ? h : h - qh - (kind[n] - 1) * B.kh;
        // (units from turned_units on: the dims that stay)
        const bool halves = unit < turned_units && !P.interleaved;
        a[n] = halves ? unit : 2 * unit;
        b[n] = halves ? unit + turned_units : 2 * unit + 1;
        const HeadsView& src = kind[n] == 0 ? P.q : kind[n] == 1 ? P.k : P.v;
        const long long at = (long long)g[n] * src.head + (long long)row * src.row;
        pg_get8(src, at + 8 * a[n], x[n]);
        pg_get8(src, at + 8 * b[n], y[n]);
    }
    const PagedRow R = pg_row(B, row, &found);
    if (R.token < 0) return;  // (block-uniform)
    const int pairs = P.rotary >> 1;
    if (tid < pairs) {
        const double at = (double)(P.positions ? P.positions[row] : R.token) * P.turns[tid];
        float s, c;
        sincospif(2.0f * (float)(at - __builtin_rint(at)), &s, &c);
        turn[tid] = float2{c, s};
    }
    __syncthreads();
#pragma unroll
    for (int n = 0; n < PAGED_APPEND_UNITS; ++n) {
        if (kind[n] < 0) continue;
        const int unit = (n * 256 + tid) % per_head;
        if (unit < turned_units && kind[n] != 2) {
            const float2* t = turn + 8 * unit;
            if (!P.interleaved) {
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    const float u = x[n][k], v = y[n][k];
                    x[n][k] = u * t[k].x - v * t[k].y;
                    y[n][k] = v * t[k].x + u * t[k].y;
                }
            } else {
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const float u = x[n][2 * k], v = x[n][2 * k + 1], w = y[n][2 * k], z = y[n][2 * k + 1];
                    x[n][2 * k] = u * t[k].x - v * t[k].y;
                    x[n][2 * k + 1] = v * t[k].x + u * t[k].y;
                    y[n][2 * k] = w * t[4 + k].x - z * t[4 + k].y;
                    y[n][2 * k + 1] = z * t[4 + k].x + w * t[4 + k].y;
                }
            }
        }
        if (kind[n] == 0) {
            const long long to = (long long)g[n] * P.q_out.head + (long long)row * P.q_out.row;
            pg_put8(P.q_out, to + 8 * a[n], x[n]);
            pg_put8(P.q_out, to + 8 * b[n], y[n]);
        } else if (R.page >= 0) {
            __half* to = kind[n] == 1 ? B.k : B.v;
            *reinterpret_cast<v4u*>(to + pg_at(B, P.D, R, g[n], kind[n] == 2, a[n])) = pg_halves(x[n]);
            *reinterpret_cast<v4u*>(to + pg_at(B, P.D, R, g[n], kind[n] == 2, b[n])) = pg_halves(y[n]);
        }
    }
}

// Read. Block: one row, its K heads, then its V heads; a thread takes a piece of 8 dims
// at a time.
__global__ __launch_bounds__(256) void paged_read_kernel(PagedRowsParams P) {
    __shared__ int found;
    const PagedBatch& B = P.b;
    const int row = pg_block_row(blockIdx.x, B.rows), per_head = P.D >> 3;
    const PagedRow R = pg_row(B, row, &found);
    if (R.page < 0) return;  // (block-uniform)
    for (int i = threadIdx.x; i < 2 * B.kh * per_head; i += 256) {
        const int piece = i % per_head, h = i / per_head;
        const bool v = h >= B.kh;
        const int g = v ? h - B.kh : h;
        const HeadsView& dst = v ? P.v : P.k;
        if (!dst.data) continue;
        const pg_h8 u = __builtin_bit_cast(pg_h8, *reinterpret_cast<const v4u*>((v ? B.v : B.k) + pg_at(B, P.D, R, g, v, piece)));
        float x[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) x[k] = (float)u[k];
        pg_put8(dst, (long long)g * dst.head + (long long)row * dst.row + 8 * piece, x);
    }
}

// ---------------------------------------------------------------------------
// Host side.
// ---------------------------------------------------------------------------
struct PagedPool {
    uint32_t magic;
    Domain* domain;
    rk_npu_hip_attention_paged_config cfg;
    __half* kv[2];
    double* turns;  // [rotary / 2], or nullptr
    int* flaw;
    size_t kv_bytes, turn_bytes;  // of one array each
    DevFence fence;               // device calls that note flaws
    std::atomic<bool> captured{false};  // graphs hold some, whose launches the fence does not see

    void note(hipStream_t s) {
        if (fence.note(s)) captured = true;
    }
    // The host waits for the device calls made, and for launches of graphs that hold any.
    hipError_t wait() { return captured ? hipDeviceSynchronize() : fence.wait(nullptr); }
};

constexpr size_t PAGED_FLAW_BYTES = 256;

static PagedPool* as_pool(const void* p) {
    PagedPool* c = static_cast<PagedPool*>(const_cast<void*>(p));
    return (c && c->magic == MAGIC_PAGED_POOL) ? c : nullptr;
}

// Turns (radians / 2 pi) of pair j per position.
static double paged_turns(const rk_npu_hip_attention_paged_config& c, int j) {
    const double around = 6.283185307179586476925286766559;
    return (c.frequencies ? c.frequencies[j] : std::pow(c.rope_theta, -2.0 * j / c.rotary_dim)) / around;
}

static bool valid_paged(const rk_npu_hip_attention_paged_config* c) {
    if (!c || !valid_config(&c->attention)) return false;
    if (c->page != 16 && c->page != 32 && c->page != 64 && c->page != 128 && c->page != 256) return false;
    if (c->rotary_dim < 0 || c->rotary_dim > c->attention.head_dim || c->rotary_dim % 16) return false;
    if (c->interleaved != 0 && c->interleaved != 1) return false;
    if (c->rotary_dim > 0 && !c->frequencies && !(std::isfinite(c->rope_theta) && c->rope_theta > 0.0)) return false;
    // (the angles of all 32-bit positions are finite)
    for (int j = 0; j < c->rotary_dim / 2; ++j)
        if (!std::isfinite(paged_turns(*c, j) * 0x1p31)) return false;
    // (kernels count the pool's 16-token tiles in 32 bits)
    return c->pages >= 1 && (int64_t)c->pages * c->attention.kv_heads * (c->page / 16) <= INT_MAX &&
           c->attention.max_capacity <= RK_NPU_HIP_PAGED_MAX_TOKENS;
}
static size_t paged_kv_bytes(const rk_npu_hip_attention_paged_config& c) {
    return (size_t)c.pages * c.page * c.attention.kv_heads * c.attention.head_dim * sizeof(__half);
}

// A batch a call may plan by; the arrays on the device are the kernels' to check.
static bool valid_batch(const PagedPool* c, const rk_npu_hip_paged_batch* b) {
    if (!b || b->sequences < 1 || b->sequences > RK_NPU_HIP_PAGED_MAX_SEQUENCES || b->rows < 1 ||
        b->rows > RK_NPU_HIP_PAGED_MAX_ROWS)
        return false;
    if (b->max_rows < 1 || b->max_rows > b->rows || b->table_stride < 1 || b->max_tokens < 1) return false;
    if (!b->row_offsets && (b->max_rows != 1 || b->rows < b->sequences)) return false;
    if (b->max_tokens > (int64_t)b->table_stride * c->cfg.page || b->max_tokens > c->cfg.attention.max_capacity)
        return false;
    const int device = device_of(c->domain);
    auto ints = [&](const int32_t* p) {
        return p && reinterpret_cast<uintptr_t>(p) % sizeof(int32_t) == 0 && kernel_readable(p, device);
    };
    return ints(b->lengths) && ints(b->table) && (!b->row_offsets || ints(b->row_offsets));
}

static PagedBatch batch_of(const PagedPool* c, const rk_npu_hip_paged_batch* b) {
    PagedBatch B;
    B.lengths = b->lengths;
    B.offsets = b->row_offsets;
    B.table = b->table;
    B.flaw = c->flaw;
    B.k = c->kv[0];
    B.v = c->kv[1];
    B.sequences = b->sequences;
    B.rows = b->rows;
    B.max_rows = b->max_rows;
    B.max_tokens = b->max_tokens;
    B.table_stride = b->table_stride;
    B.kh = c->cfg.attention.kv_heads;
    B.pages = c->cfg.pages;
    B.page_shift = __builtin_ctz(c->cfg.page);
    return B;
}

static PagedRowsParams rows_params(const PagedPool* c, const rk_npu_hip_paged_batch* b) {
    PagedRowsParams P{};
    P.b = batch_of(c, b);
    P.turns = c->turns;
    P.D = c->cfg.attention.head_dim;
    P.rotary = c->cfg.rotary_dim;
    P.interleaved = c->cfg.interleaved;
    return P;
}

static bool paged_same_geometry(const AttnWork* w, const PagedPool* c) {
    const rk_npu_attention_f16_config &a = w->cfg, &b = c->cfg.attention;
    return a.query_heads == b.query_heads && a.kv_heads == b.kv_heads && a.head_dim == b.head_dim &&
           a.mask_mode == b.mask_mode && a.softmax_scale == b.softmax_scale &&
           device_of(w->domain) == device_of(c->domain);
}

// Which kernel, its row tiles, and the blocks that splits aim at. R: query rows of a
// sequence and KV head, at most. Times in us.
//
// attn_paged_rows_kernel while a tile holds R, so that pages are read once: 5 rows of 12
// sequences (R = 20, 240 MB) 51 to 56 with tiles of 32, 61 with two of 16. (Two row groups
// of 256 dims have no registers.)
//
// attn_paged_tile_kernel with blocks of 128 rows for short sequences, whose long blocks
// are what a call lasts, of 256 for long ones, whose K and V then meet twice as many rows
// in LDS: one sequence's 2048 rows 64 and 74, 8 x 1024 131 and 142, 64 rows after 4000
// tokens 25 and 29; 8192 rows 720 and 709, 4 x 512 after 8000 327 and 308, 2 x 4096 of 64
// dims 118 and 113.
//
// Splits, in blocks a CU. Rows kernel: one for few sequences, as a block's rows leave
// partials, four for more than 4, whose pieces are then of like length. With one and with
// four, 32 heads over 8 of 128, contexts not in the last-level cache: sequences of 16000
// tokens, 1 20 and 23, 2 30 and 32, 3 49 and 43, 4 52 and 55, 5 74 and 62, 6 85 and 73, 8 91
// and 94, 12 160 and 142, 24 245 and 247; of 1000 to 16000, 4 36 and 35, 5 44 and 39, 8 63 and
// 58, 24 168 and 144. Of 16 over 2 of 256 four win from 12 on (96 and 80; ragged 57 and 52),
// 5 37 and 47, 8 53 and 59. A split holds a unit a wave at least: one sequence of 4000 tokens
// 12.7 and 13.3 with two, 16 with four. Tile kernel: as many as stay on a CU; 8 units at least:
// 128 rows of 256 dims after 3600 tokens 35, with 16 units 44, with 24 50.
//
// Rows kernel, more sequences than blocks to aim at (128 of 8 KV heads): where one may be
// longer than 4096 tokens, further splits of long ones follow the sequences' own blocks, as
// many as are aimed at, of 32 units at least (256 sequences of 300 to 700 tokens and one of
// 131072 188 and unsplit 1450, of 8192 101 and 146, of 4096 99 and 103; none longer, but
// allowed, 90 and 88; 200 of up to 8100 557 and 580; 1000 of 16 heads over 8 of 64 with a
// long one 250 and 965, without 190 and 170).
static PagedPlan paged_plan(AttnPagedParams& P, int D) {
    const PagedBatch& B = P.b;
    const int G = P.qh / B.kh, cus = device_cus();
    const int64_t R = (int64_t)B.max_rows * G;
    // (each sequence ends a tile of its own)
    auto tiles = [&](int rows) {
        return std::min<int64_t>(B.sequences * ((R + rows - 1) / rows), (int64_t)B.rows * G / rows + B.sequences);
    };
    const int units = (B.max_tokens + 31) / 32;
    PagedPlan plan{R > (D == 256 ? 16 : 32), D < 256 && units > 128 ? 2 : 1, false};
    P.tile_rows = plan.tile ? 128 * plan.units : R <= 8 ? 8 : R <= 16 ? 16 : 32;
    P.tiles = (int)tiles(P.tile_rows);
    P.least = plan.tile ? 8 : 4;
    P.target = 0;
    const int blocks = plan.tile ? (plan.units == 1 && D < 256 ? 2 : 1) : B.sequences > 4 ? 4 : 1;
    // (as many as the workspace holds partials for)
    const int64_t slots = (int64_t)(attn_partial_rows(D) / ((size_t)B.kh * P.tile_rows));
    const int aim = std::max(1, blocks * cus / B.kh), want = (int)std::min<int64_t>(aim, slots - P.tiles);
    // (units are added up in 32 bits)
    if (units > 16 && (int64_t)P.tiles * units < (1 << 30)) {
        if (P.tiles < want) {
            P.target = want;
        } else if (!plan.tile && units > 128) {
            plan.behind = true;
            P.least = 32;
            P.target = (int)std::min<int64_t>(aim, slots / 2);
        }
    }
    P.items = P.target ? P.tiles + P.target : P.tiles;
    P.slots = plan.behind ? 2 * P.target : P.items;
    P.wave = plan.tile && P.causal ? std::max(1, cus / B.kh) : 0;
    return plan;
}

}  // namespace hm

using namespace hm;

extern "C" {

void rk_npu_hip_attention_paged_config_init(rk_npu_hip_attention_paged_config* c) {
    if (!c) return;
    std::memset(c, 0, sizeof(*c));
    rk_npu_attention_f16_config_init(&c->attention);
    c->page = 64;
    c->rope_theta = 10000.0;
}

int rk_npu_hip_attention_paged_query(const rk_npu_hip_attention_paged_config* c, rk_npu_attention_f16_sizes* sizes) {
    if (!valid_paged(c) || !sizes) return RK_NPU_ERR_PARAM;
    const int rc = rk_npu_attention_f16_query(&c->attention, 0, 1, 0, sizes);
    if (rc != RK_NPU_OK) return rc;
    sizes->key_bytes = sizes->value_bytes = paged_kv_bytes(*c);
    sizes->tail_bytes = 0;
    return RK_NPU_OK;
}

int rk_npu_hip_attention_paged_pool_create(rk_npu_iommu_domain* domain,
                                           const rk_npu_hip_attention_paged_config* config,
                                           rk_npu_hip_attention_paged_pool** out) {
    if (out) *out = nullptr;
    Domain* d = static_cast<Domain*>(domain);
    if (!d || !out || !valid_paged(config)) return RK_NPU_ERR_PARAM;
    if (!supported_dim(config->attention.head_dim)) return RK_NPU_ERR_UNSUPPORTED;
    DeviceGuard dev(device_of(d));
    if (!dev.ok) return RK_NPU_ERR_DEVICE;
    PagedPool* c = new (std::nothrow) PagedPool();
    if (!c) return RK_NPU_ERR_NOMEM;
    c->magic = MAGIC_PAGED_POOL;
    c->domain = d;
    c->cfg = *config;
    c->cfg.frequencies = nullptr;
    c->kv_bytes = paged_kv_bytes(*config);
    const int pairs = config->rotary_dim / 2;
    c->turn_bytes = std::max<size_t>(1, pairs) * sizeof(double);
    double turns[128];
    for (int j = 0; j < pairs; ++j) turns[j] = paged_turns(*config, j);
    auto* raw = reinterpret_cast<rk_npu_hip_attention_paged_pool*>(c);
    c->flaw = static_cast<int*>(domain_alloc(d, PAGED_FLAW_BYTES));
    c->turns = c->flaw ? static_cast<double*>(domain_alloc(d, c->turn_bytes)) : nullptr;
    c->kv[0] = c->turns ? static_cast<__half*>(domain_alloc(d, c->kv_bytes)) : nullptr;
    c->kv[1] = c->kv[0] ? static_cast<__half*>(domain_alloc(d, c->kv_bytes)) : nullptr;
    if (!c->kv[1]) {
        rk_npu_hip_attention_paged_pool_free(raw);
        return RK_NPU_ERR_NOMEM;
    }
    const int zero = 0;
    if (hipMemcpy(c->flaw, &zero, sizeof(zero), hipMemcpyHostToDevice) != hipSuccess ||
        (pairs && hipMemcpy(c->turns, turns, pairs * sizeof(double), hipMemcpyHostToDevice) != hipSuccess)) {
        (void)hipGetLastError();
        rk_npu_hip_attention_paged_pool_free(raw);
        return RK_NPU_ERR_DEVICE;
    }
    *out = raw;
    return RK_NPU_OK;
}

void rk_npu_hip_attention_paged_pool_free(rk_npu_hip_attention_paged_pool* pool) {
    PagedPool* c = as_pool(pool);
    if (!c) return;
    DeviceGuard dev(device_of(c->domain));
    (void)c->wait();
    c->fence.destroy();
    for (int i = 0; i < 2; ++i) domain_free(c->domain, c->kv[i], c->kv_bytes);
    domain_free(c->domain, c->turns, c->turn_bytes);
    domain_free(c->domain, c->flaw, PAGED_FLAW_BYTES);
    c->magic = 0;
    delete c;
}

int rk_npu_hip_attention_paged_status(rk_npu_hip_attention_paged_pool* pool) {
    PagedPool* c = as_pool(pool);
    if (!c) return RK_NPU_ERR_PARAM;
    DeviceGuard dev(device_of(c->domain));
    if (!dev.ok || c->wait() != hipSuccess) return RK_NPU_ERR_DEVICE;
    int flaw = 0;
    const int zero = 0;
    if (hipMemcpy(&flaw, c->flaw, sizeof(flaw), hipMemcpyDeviceToHost) != hipSuccess) return RK_NPU_ERR_DEVICE;
    if (flaw && hipMemcpy(c->flaw, &zero, sizeof(zero), hipMemcpyHostToDevice) != hipSuccess) return RK_NPU_ERR_DEVICE;
    return flaw ? RK_NPU_ERR_PARAM : RK_NPU_OK;
}

int rk_npu_hip_attention_paged_append(rk_npu_hip_attention_paged_pool* pool, const rk_npu_hip_paged_batch* batch,
                                      const rk_npu_hip_heads* k, const rk_npu_hip_heads* v, const int32_t* positions,
                                      const rk_npu_hip_heads* q, const rk_npu_hip_heads* q_out, void* stream) {
    PagedPool* c = as_pool(pool);
    if (!c || !valid_batch(c, batch) || !q != !q_out) return RK_NPU_ERR_PARAM;
    const int device = device_of(c->domain), kh = c->cfg.attention.kv_heads, qh = c->cfg.attention.query_heads;
    const int D = c->cfg.attention.head_dim, rows = batch->rows;
    if (!valid_heads(k, device, D, false, kh, rows) || !valid_heads(v, device, D, false, kh, rows))
        return RK_NPU_ERR_PARAM;
    if (q && (!valid_heads(q, device, D, false, qh, rows) || !valid_heads(q_out, device, D, true, qh, rows)))
        return RK_NPU_ERR_PARAM;
    // (in place: each thread writes what it alone has read)
    if (q && q->data == q_out->data &&
        (q->type != q_out->type || q->head_stride != q_out->head_stride || q->row_stride != q_out->row_stride))
        return RK_NPU_ERR_PARAM;
    if (positions && (reinterpret_cast<uintptr_t>(positions) % sizeof(int32_t) || !kernel_readable(positions, device)))
        return RK_NPU_ERR_PARAM;
    DeviceGuard dev(device);
    if (!dev.ok) return RK_NPU_ERR_DEVICE;
    PagedRowsParams P = rows_params(c, batch);
    P.k = view_of(*k);
    P.v = view_of(*v);
    if (q) {
        P.q = view_of(*q);
        P.q_out = view_of(*q_out);
        P.qh = qh;
    }
    P.positions = positions;
    hipStream_t s = static_cast<hipStream_t>(stream);
    const int heads = P.qh + 2 * kh;
    P.heads_per_block = 256 * PAGED_APPEND_UNITS / (D / 16);
    hipLaunchKernelGGL(paged_append_kernel, dim3(rows, (heads + P.heads_per_block - 1) / P.heads_per_block), dim3(256), 0, s, P);
    if (hipGetLastError() != hipSuccess) return RK_NPU_ERR_DEVICE;
    c->note(s);
    return RK_NPU_OK;
}

int rk_npu_hip_attention_paged_read(rk_npu_hip_attention_paged_pool* pool, const rk_npu_hip_paged_batch* batch,
                                    const rk_npu_hip_heads* k, const rk_npu_hip_heads* v, void* stream) {
    PagedPool* c = as_pool(pool);
    if (!c || !valid_batch(c, batch) || (!k && !v)) return RK_NPU_ERR_PARAM;
    const int device = device_of(c->domain), kh = c->cfg.attention.kv_heads, D = c->cfg.attention.head_dim;
    if ((k && !valid_heads(k, device, D, true, kh, batch->rows)) || (v && !valid_heads(v, device, D, true, kh, batch->rows)))
        return RK_NPU_ERR_PARAM;
    DeviceGuard dev(device);
    if (!dev.ok) return RK_NPU_ERR_DEVICE;
    PagedRowsParams P = rows_params(c, batch);
    if (k) P.k = view_of(*k);
    if (v) P.v = view_of(*v);
    hipStream_t s = static_cast<hipStream_t>(stream);
    hipLaunchKernelGGL(paged_read_kernel, dim3(batch->rows), dim3(256), 0, s, P);
    if (hipGetLastError() != hipSuccess) return RK_NPU_ERR_DEVICE;
    c->note(s);
    return RK_NPU_OK;
}

int rk_npu_hip_attention_paged_run(rk_npu_attention_f16_workspace* workspace, rk_npu_hip_attention_paged_pool* pool,
                                   const rk_npu_hip_paged_batch* batch, const rk_npu_hip_heads* q,
                                   const rk_npu_hip_heads* out, void* stream) {
    AttnWork* w = as_attn_work(workspace);
    PagedPool* c = as_pool(pool);
    if (!w || !c || !paged_same_geometry(w, c) || !valid_batch(c, batch)) return RK_NPU_ERR_PARAM;
    const rk_npu_attention_f16_config& cfg = c->cfg.attention;
    const int device = device_of(c->domain), D = cfg.head_dim;
    if ((int64_t)batch->rows * cfg.query_heads > RK_NPU_HIP_PAGED_MAX_QUERIES) return RK_NPU_ERR_PARAM;
    if (!valid_heads(q, device, D, false, cfg.query_heads, batch->rows) ||
        !valid_heads(out, device, D, true, cfg.query_heads, batch->rows))
        return RK_NPU_ERR_PARAM;
    DeviceGuard dev(device);
    if (!dev.ok) return RK_NPU_ERR_DEVICE;
    AttnPagedParams P;
    P.b = batch_of(c, batch);
    P.q = q->data;
    P.q_f32 = q->type == RK_NPU_HIP_F32;
    P.q_head = q->head_stride;
    P.q_row = q->row_stride;
    P.out = out->data;
    P.out_f16 = out->type == RK_NPU_HIP_F16;
    P.o_head = out->head_stride;
    P.o_row = out->row_stride;
    P.part = w->part;
    P.qh = cfg.query_heads;
    P.causal = cfg.mask_mode == RK_NPU_ATTENTION_F16_CAUSAL ? 1 : 0;
    P.scale = cfg.softmax_scale;
    const PagedPlan plan = paged_plan(P, D);
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (D == 64)
        launch_attn_paged_64(P, plan, s);
    else if (D == 128)
        launch_attn_paged_128(P, plan, s);
    else
        launch_attn_paged_256(P, plan, s);
    if (hipGetLastError() != hipSuccess) return RK_NPU_ERR_DEVICE;
    c->note(s);
    w->fence.note(s);
    return RK_NPU_OK;
}

}  // extern "C"
