/*
 * rk_npu_attention_q8.h — a KV cache held in 8 bits, with one scale for each
 * block of tokens and KV head, and the grouped-query attention over it. No
 * counterpart in the reference, whose caches are fp16: the calls stand beside
 * rk_npu_attention_f16.h (same geometry, masks, workspace and array layouts)
 * for contexts whose fp16 rows cost too much memory or time to read.
 *
 * What a cache holds. Rows come as fp16 (f32 rows of the device calls are
 * rounded to nearest fp16 first). Tokens form blocks of `block` tokens from
 * token 0 on. A complete block of one KV head, K and V apart, is `block` x
 * head_dim codes and one f32 scale; with a the largest magnitude among its
 * values
 *     RK_NPU_HIP_KV_I8    code = 127 x / a rounded half to even, -127..127;
 *                         value = code * scale, scale = a / 127
 *     RK_NPU_HIP_KV_E4M3  code = 448 x / a rounded half to even to e4m3 (1
 *                         sign, 4 exponent, 3 fraction bits, largest 448);
 *                         value = code * scale, scale = a / 448
 * (a = 0: values 0). A block that holds an infinity or a NaN has no scale: all
 * of its values read as NaN. The tokens after the last complete block (the
 * tail) stay fp16 until their block is complete, so the contents do not depend
 * on how the rows are split over calls.
 *
 * Truncation. Besides the tail, two sets of fp16 rows are kept until the next
 * append: the last complete block's, and those that were the tail before the last
 * append. Truncating into the tail or one of these is exact: the cache is as if
 * the dropped rows had never come (drafts that a verification rejects; the undoing
 * of the last append). A truncation into another block keeps that block's codes;
 * the next append continues from their values rounded to fp16.
 *
 * Attention is rk_npu_attention_f16.h's formula over the cache's values: f32
 * scores, weights and sums, for |scale q k| up to 10^7 (beyond, a row may come out as
 * NaN). Into the products with V a weight goes times its block's V scale, as two fp16
 * (22 bits), or as one (11 bits) where the output is fp16 and there are more than 16
 * query rows per KV head (rows x query heads / KV heads). Where fp16 has fewer bits it
 * is off by up to 2^-30 of the row's largest such product: the values of keys that
 * light are lost, their weights are not. A value of the tail that is infinite or NaN
 * counts for the query rows that see its token and for no other.
 *
 * Workspaces are rk_npu_attention_f16_workspace of the same geometry
 * (rk_npu_attention_f16_prepare with &config.attention).
 */
#ifndef RK_NPU_ATTENTION_Q8_H
#define RK_NPU_ATTENTION_Q8_H

#include <stdint.h>

#include "rk_npu_attention_f16.h"
#include "rk_npu_hip.h"

#ifdef __cplusplus
extern "C" {
#endif

/* format values */
#define RK_NPU_HIP_KV_I8 0
#define RK_NPU_HIP_KV_E4M3 1

typedef struct rk_npu_hip_attention_q8_config {
    rk_npu_attention_f16_config attention; /* head_dim 64, 128 or 256; capacities are rounded up to whole blocks */
    int32_t format;                        /* RK_NPU_HIP_KV_I8 or _E4M3 */
    int32_t block;                         /* tokens per scale: 32, 64 or 128 */
} rk_npu_hip_attention_q8_config;

typedef struct rk_npu_hip_attention_q8_cache rk_npu_hip_attention_q8_cache;

/* A [heads][rows][head_dim] array on the device: element (h, r, d) is at
 * data[h * head_stride + r * row_stride + d]. Strides count elements and are
 * not negative; heads and rows of an array that is written do not overlap. Any
 * alignment of the element type serves. */
typedef struct rk_npu_hip_heads {
    void* data;
    int32_t type; /* RK_NPU_HIP_F16 or RK_NPU_HIP_F32 */
    int64_t head_stride;
    int64_t row_stride;
} rk_npu_hip_heads;

/* rk_npu_attention_f16_config_init's defaults, RK_NPU_HIP_KV_I8, blocks of 32. */
void rk_npu_hip_attention_q8_config_init(rk_npu_hip_attention_q8_config* config);

/* Storage of a cache of `capacity` rows: codes and scales of K and of V, and the
 * fp16 rows (tail_bytes); workspace_bytes for `query_rows`. */
int rk_npu_hip_attention_q8_query(const rk_npu_hip_attention_q8_config* config, int32_t capacity,
                                  int32_t query_rows, rk_npu_attention_f16_sizes* sizes);

/* An empty cache of initial_capacity rows. */
int rk_npu_hip_attention_q8_cache_create(rk_npu_iommu_domain* domain, const rk_npu_hip_attention_q8_config* config,
                                         rk_npu_hip_attention_q8_cache** cache);
void rk_npu_hip_attention_q8_cache_free(rk_npu_hip_attention_q8_cache* cache);
/* Grow to at least `capacity` rows (at most max_capacity), keeping the contents. */
int rk_npu_hip_attention_q8_cache_reserve(rk_npu_ctx* ctx, rk_npu_hip_attention_q8_cache* cache, int32_t capacity);
/* Keep the first `length` rows. Host bookkeeping: enqueues nothing. */
int rk_npu_hip_attention_q8_cache_truncate(rk_npu_hip_attention_q8_cache* cache, int32_t length);
int rk_npu_hip_attention_q8_cache_get_info(const rk_npu_hip_attention_q8_cache* cache,
                                           rk_npu_attention_f16_cache_info* info);

/* ---- host buffers: [heads][rows][head_dim] fp16 arrays, done on return ------
 * Calls on one cache from several threads exclude each other, runs on workspaces
 * of their own excepted; a workspace takes one run at a time (RK_NPU_ERR_BUSY).
 * load replaces the contents (rows == 0: empties the cache, k and v may be
 * NULL); append grows the cache as needed, up to max_capacity; read gives the
 * values of rows first..first + rows - 1 rounded to fp16; run and run_half are
 * rk_npu_attention_f16_run and _run_half over the 8-bit cache. */
int rk_npu_hip_attention_q8_cache_load(rk_npu_ctx* ctx, rk_npu_hip_attention_q8_cache* cache, const uint16_t* k,
                                       const uint16_t* v, int32_t rows);
int rk_npu_hip_attention_q8_cache_append(rk_npu_ctx* ctx, rk_npu_hip_attention_q8_cache* cache, const uint16_t* k,
                                         const uint16_t* v, int32_t rows);
int rk_npu_hip_attention_q8_cache_read(rk_npu_ctx* ctx, rk_npu_hip_attention_q8_cache* cache, int32_t first,
                                       int32_t rows, uint16_t* k, uint16_t* v);
int rk_npu_hip_attention_q8_run(rk_npu_ctx* ctx, rk_npu_attention_f16_workspace* workspace,
                                rk_npu_hip_attention_q8_cache* cache, const uint16_t* q, int32_t rows,
                                int32_t position, float* output, rk_npu_attention_f16_timings* timings);
int rk_npu_hip_attention_q8_run_half(rk_npu_ctx* ctx, rk_npu_attention_f16_workspace* workspace,
                                     rk_npu_hip_attention_q8_cache* cache, const uint16_t* q, int32_t rows,
                                     int32_t position, uint16_t* output, rk_npu_attention_f16_timings* timings);

/* ---- device arrays, on the caller's stream (NULL: the null stream) -----------
 * The arrays lie in the memory of the cache's GPU (RK_NPU_ERR_PARAM otherwise);
 * nothing is synchronized and nothing allocated (append: reserve first). An array
 * that is written overlaps no other of the call. Calls on one cache take effect
 * in the order they are made, so they go to one stream, or the caller orders
 * their streams; runs and reads may overlap each other, runs on workspaces of
 * their own.
 *
 * Under stream capture a call is recorded, and the length moves on, as if it had
 * run: launch the graph before anything else uses what it writes. Each launch does
 * what was recorded, at the recorded positions:
 *   - a graph of reads and runs may be launched as long as the rows up to the
 *     recorded length are the cache's, its storage has not grown, and no later
 *     append has completed the block that was open (the run read its fp16 rows);
 *   - a graph of appends may be launched again (with new rows in k and v, to the
 *     same positions) until another append is made to the cache; several appends
 *     to one cache in a graph complete one block of it at most, together;
 *   - an append that continues from codes (after a truncation deeper than the rows
 *     kept) is refused under capture: RK_NPU_ERR_UNSUPPORTED.
 * Host-buffer calls wait for device calls made before them; for a graph's launch
 * the caller waits. */
int rk_npu_hip_attention_q8_device_append(rk_npu_hip_attention_q8_cache* cache, const rk_npu_hip_heads* k,
                                          const rk_npu_hip_heads* v, int32_t rows, void* stream);
/* The values of rows first..first + rows - 1 (k or v may be NULL): f32 values,
 * or rounded to fp16, by the arrays' types. */
int rk_npu_hip_attention_q8_device_read(rk_npu_hip_attention_q8_cache* cache, int32_t first, int32_t rows,
                                        const rk_npu_hip_heads* k, const rk_npu_hip_heads* v, void* stream);
/* Attention of `rows` query rows of every query head, the first at `position`
 * (f32 queries are rounded to fp16). */
int rk_npu_hip_attention_q8_device_run(rk_npu_attention_f16_workspace* workspace,
                                       rk_npu_hip_attention_q8_cache* cache, const rk_npu_hip_heads* q, int32_t rows,
                                       int32_t position, const rk_npu_hip_heads* out, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* RK_NPU_ATTENTION_Q8_H */
