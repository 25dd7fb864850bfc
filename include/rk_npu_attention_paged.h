/*
 * rk_npu_attention_paged.h — the KV cache of a batch of sequences in pages of one
 * pool, the append that rotates rows by their positions on the way, and the
 * grouped-query attention of each sequence's newest rows over its pages. No
 * counterpart in the reference, whose caches hold one sequence each: the calls
 * stand beside rk_npu_attention_f16.h and rk_npu_attention_q8.h (same geometry,
 * masks, workspace and array layouts) for servers of many sequences.
 *
 * What a pool holds. `pages` pages of `page` tokens, fp16 K and V of every KV
 * head. Which page belongs to which sequence is the caller's: token t of sequence
 * s lies in page table[s][t / page], at place t % page. Sequences may share pages
 * that no call of theirs writes (a common prefix). The table, the sequences'
 * lengths and the rows of a call lie in device memory and are read when the work
 * runs, so a captured graph may be launched again after they have changed.
 *
 * A batch. Arrays are [heads][rows][head_dim]; the rows of one sequence follow
 * those of another. Sequence s has rows row_offsets[s]..row_offsets[s + 1] - 1 (row
 * s where there are no row_offsets), which are its newest tokens: row i of its n
 * is token lengths[s] - n + i. Rows with a token below 0 have none: they are not
 * stored, not read, and in causal attention see nothing. Rows before
 * row_offsets[0] and from row_offsets[sequences] on are left as they are, in every
 * array.
 *
 * Append. K and V rows (f16 or f32) go to their tokens' places, K rotated. The
 * first rotary_dim dims of a row are pairs, (j, j + rotary_dim / 2), or (2j, 2j + 1)
 * where interleaved; pair (x, y) becomes
 *     (x cos a - y sin a, y cos a + x sin a),   a = position * frequency[j]
 * with a in 64 bits, its sine and cosine and the products in 32, and one rounding
 * to fp16 at the end. V and the other dims are rounded to fp16 alone. Query rows
 * are rotated the same way into an array of their own in the same call.
 *
 * Attention is rk_npu_attention_f16.h's formula: queries in fp16 (f32 ones are
 * rounded), f32 scores, weights and sums, for |scale q k| up to 10^7 (beyond, a row
 * may come out as NaN). A weight goes into the products with V as two fp16 (22
 * bits), or as one (11 bits) where the output is fp16 and a sequence may have more
 * than 32 query rows per KV head (max_rows x query heads / KV heads; more than 16 of
 * head_dim 256); f32 output always takes two. Where fp16 has fewer bits a weight is
 * off by up to 2^-30 of the row's largest. A causal row sees the tokens up to its own,
 * a row without a mask all lengths[s]. A row that sees no token is 0. Infinities and
 * NaN in K or V count for the rows that see their token and for no other; those in V
 * however small the token's weight (calls whose rows see some take up to 70 times as
 * long). Means of finite values are finite.
 *
 * What the device finds wrong. A length below 0 or above max_tokens, row_offsets
 * that fall or pass `rows` or give a sequence more than max_rows, and a page
 * outside 0..pages - 1 (or a negative one) under a token of its sequence are noted
 * on the device, and nothing is read or written out of bounds: the sequence counts
 * as one of no rows (wrong row_offsets) or of no tokens; to the page nothing is
 * appended, from it nothing is read, and the attention of the rows that see it has
 * no meaning. rk_npu_hip_attention_paged_status() tells of it.
 *
 * Workspaces are rk_npu_attention_f16_workspace of the same geometry
 * (rk_npu_attention_f16_prepare with &config.attention).
 */
#ifndef RK_NPU_ATTENTION_PAGED_H
#define RK_NPU_ATTENTION_PAGED_H

#include <stdint.h>

#include "rk_npu_attention_f16.h"
#include "rk_npu_attention_q8.h"
#include "rk_npu_hip.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Sequences and rows of a batch, rows x query heads of an attention call, and tokens of a sequence, at most. */
#define RK_NPU_HIP_PAGED_MAX_SEQUENCES 1024
#define RK_NPU_HIP_PAGED_MAX_ROWS (1 << 23)
#define RK_NPU_HIP_PAGED_MAX_QUERIES (1 << 26)
#define RK_NPU_HIP_PAGED_MAX_TOKENS (1 << 30)

typedef struct rk_npu_hip_attention_paged_config {
    rk_npu_attention_f16_config attention; /* head_dim 64, 128 or 256; max_capacity: the longest sequence
                                              (max_query_rows and initial_capacity serve the workspace alone) */
    int32_t page;                          /* tokens per page: 16, 32, 64, 128 or 256 */
    int32_t pages;                         /* pages of the pool */
    int32_t rotary_dim;                    /* dims rotated, a multiple of 16 up to head_dim; 0: none */
    int32_t interleaved;                   /* 0: pairs (j, j + rotary_dim / 2); 1: pairs (2j, 2j + 1) */
    double rope_theta;                     /* frequency[j] = rope_theta^(-2j / rotary_dim), where frequencies is NULL */
    const double* frequencies;             /* rotary_dim / 2 of them, radians per position (below 2^995, as
                                              rope_theta's are); read by query and create only */
} rk_npu_hip_attention_paged_config;

typedef struct rk_npu_hip_attention_paged_pool rk_npu_hip_attention_paged_pool;

/* The sequences of a call. lengths, row_offsets and table lie in the memory of
 * the pool's GPU. */
typedef struct rk_npu_hip_paged_batch {
    int32_t sequences;          /* 1..RK_NPU_HIP_PAGED_MAX_SEQUENCES */
    int32_t rows;               /* rows of the call's arrays, 1..RK_NPU_HIP_PAGED_MAX_ROWS */
    int32_t max_rows;           /* no sequence has more rows: 1..rows, 1 without row_offsets */
    int32_t max_tokens;         /* no sequence is longer: 1..table_stride x page, max_capacity at most */
    const int32_t* lengths;     /* [sequences]: tokens, the call's rows among them */
    const int32_t* row_offsets; /* [sequences + 1], or NULL: a row each, rows >= sequences */
    const int32_t* table;       /* [sequences][table_stride] */
    int32_t table_stride;
} rk_npu_hip_paged_batch;

/* rk_npu_attention_f16_config_init's defaults, pages of 64 tokens, none of them, no rotation,
 * rope_theta 10000. */
void rk_npu_hip_attention_paged_config_init(rk_npu_hip_attention_paged_config* config);

/* Storage of the pool (key_bytes, value_bytes), workspace_bytes. */
int rk_npu_hip_attention_paged_query(const rk_npu_hip_attention_paged_config* config,
                                     rk_npu_attention_f16_sizes* sizes);

/* The contents of a new pool are not defined. */
int rk_npu_hip_attention_paged_pool_create(rk_npu_iommu_domain* domain,
                                           const rk_npu_hip_attention_paged_config* config,
                                           rk_npu_hip_attention_paged_pool** pool);
void rk_npu_hip_attention_paged_pool_free(rk_npu_hip_attention_paged_pool* pool);

/* Waits for the device calls made with the pool (for calls on several streams, and
 * always once a call has been captured, for the whole device: graphs may be launched
 * at any time) and tells whether one since the last status found something wrong in
 * its batch: RK_NPU_ERR_PARAM, or RK_NPU_OK. What a call that another thread makes
 * meanwhile finds wrong is told by this status or the next. Not while a stream is
 * being captured. */
int rk_npu_hip_attention_paged_status(rk_npu_hip_attention_paged_pool* pool);

/* ---- on the caller's stream (NULL: the null stream) ---------------------------
 * Arrays lie in the memory of the pool's GPU (RK_NPU_ERR_PARAM otherwise) and have
 * `rows` rows; nothing is synchronized and nothing allocated. An array that is
 * written overlaps no other of the call, save that q_out may be q itself. Calls
 * on a pool take effect in the order of their streams: the caller orders streams
 * that write pages others use. Calls on one workspace must not overlap; calls on
 * workspaces of their own may. All may be captured. */

/* positions: [rows] on the device, or NULL: the rows' tokens. q and q_out: the
 * batch's query rows and their rotation, or both NULL. */
int rk_npu_hip_attention_paged_append(rk_npu_hip_attention_paged_pool* pool, const rk_npu_hip_paged_batch* batch,
                                      const rk_npu_hip_heads* k, const rk_npu_hip_heads* v, const int32_t* positions,
                                      const rk_npu_hip_heads* q, const rk_npu_hip_heads* q_out, void* stream);
/* The batch's rows as the pool holds them (k or v may be NULL). Rows of a wrong
 * page are left as they are. */
int rk_npu_hip_attention_paged_read(rk_npu_hip_attention_paged_pool* pool, const rk_npu_hip_paged_batch* batch,
                                    const rk_npu_hip_heads* k, const rk_npu_hip_heads* v, void* stream);
/* Attention of the batch's rows over their sequences' pages. */
int rk_npu_hip_attention_paged_run(rk_npu_attention_f16_workspace* workspace, rk_npu_hip_attention_paged_pool* pool,
                                   const rk_npu_hip_paged_batch* batch, const rk_npu_hip_heads* q,
                                   const rk_npu_hip_heads* out, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* RK_NPU_ATTENTION_PAGED_H */
