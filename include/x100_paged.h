/*
 * x100_paged.h -- attention for a batch of sequences over a paged KV cache (libx100hip, gfx950).
 *
 * The batch form of the attention half of the reference's forward() (qwen_moe.c:284-292: head norms,
 * rotation, cache write, grouped-query attention), for any number of sequences and new rows (single
 * tokens, prompts, pieces of prompts behind a cached prefix) on a cache in pages of 16-bit or 4-bit
 * elements.  x100_decode.h has the one-token form on an fp32 cache.
 *
 * Batch: the new rows of all sequences are consecutive; sequence s has rows q_start[s] ..
 * q_start[s+1] - 1 and kv_len[s] cached positions, its new rows included: row i of the sequence is
 * position kv_len[s] - q_len + i.  Position p is entry p % page of page block_table[s * table_ld +
 * p / page].  The arrays are device memory, so a captured graph replays with their new contents;
 * max_q and max_kv are the host's upper bounds of the rows and positions of a sequence (they size the
 * launch and the workspace, so a graph is captured with the largest).
 *   - Rows before position 0 (q_len > kv_len): not appended, read as zeros, attention output zeros.
 *   - A sequence whose entries break the bounds (q_start decreasing or outside 0 .. n_rows, more than
 *     max_q rows, kv_len < 0 or > max_kv) and rows at or behind q_start[n_seq]: nothing of them is
 *     stored, and their outputs are left as they were.  Where q_start decreases, accepted sequences may
 *     name the same rows: outputs of such rows, and of rows behind the break, may be of one of them, mixed
 *     or left, and positions of accepted sequences may keep what they held; nothing else is touched.
 *   - A page number outside 0 .. n_pages - 1: nothing is stored there, its positions are not attended
 *     to, and they read as zeros.
 *   - Sequences may share pages that are only read; a page that gets new rows belongs to one sequence
 *     and stands once in its table row.
 *
 * Pools: x100_kv_pool_bytes bytes each for K and V, 256-byte aligned.  Page g, KV head h:
 *   16 bits  K [n_pages][n_head_kv][page][head_dim], V [n_pages][n_head_kv][page / 8][head_dim][8]
 *            (8 positions of one element together, the order in which the matrix cores take V);
 *   4 bits   X100_KV_Q4, 5 bits per element: groups of 32 elements of a head row have fp16 d, m and
 *            codes n in 0 .. 15, and stand for fp16(m + d * n) (one rounding).  Per page and head
 *            K: codes [page][head_dim / 8] 32-bit words, then [page][head_dim / 32][2] fp16 (d, m);
 *            V: codes [page / 8][head_dim] words, then [page / 8][head_dim / 32][2][8] fp16 (d of 8
 *            positions, m of 8).  A K word holds 8 elements of a row, a V word 8 positions of an
 *            element: number e at bit 16 * (e % 2) + 4 * (e / 2).
 *            d = fp16((hi - lo) * fp32(1/15)), m = fp16(lo), n = rint((x - m) * (1 / d)) within 0 .. 15,
 *            in fp32; d is the fp16 below that where m + 15 d would round past 65504.
 *            Values up to 65504 in size, whose codes stand for finite numbers; a group with a larger one,
 *            an infinity or a NaN stands for NaN (d = m = NaN).
 *
 * All pointers are device pointers unless they are the argument structures; every call is
 * asynchronous on stream and capturable.  All arguments that the host can see are checked before
 * anything is enqueued.  X100_EINVAL also for a batch that no launch can hold, with G query heads per KV
 * head: (n_rows * G / 256 + n_seq) * n_head_kv * splits of 2^23 and more in the attention of prompts,
 * n_seq * n_head_kv * splits of about 2^22 in that of single tokens (splits: of the positions, 1 where
 * there are many sequences), n_rows * n_head_kv of about 2^28 in the append.  Outputs overlap no input.
 */
#ifndef X100_HIP_PAGED_H
#define X100_HIP_PAGED_H

#include <stddef.h>
#include <stdint.h>

#include "x100_rows.h"

#ifdef __cplusplus
extern "C" {
#endif

#define X100_KV_Q4 256   /* kv_type: 4-bit codes (above); not a ggml type */

typedef struct {
    int n_head, n_head_kv;   /* query heads (<= 1024), KV heads: 1 to 16 query heads per KV head  */
    int head_dim;            /* 64 or 128                                                         */
    int page;                /* positions of a page: 16, 32, 64, 128 or 256                       */
    int n_pages;             /* pages in each pool                                                */
    int act_type;            /* queries and outputs: X100_T_F16 or X100_T_BF16                    */
    int kv_type;             /* act_type, or X100_KV_Q4                                           */
} x100_kv_cfg;

typedef struct {
    int n_seq, n_rows;       /* sequences (<= 65535), rows of the row arrays (< 2^24)             */
    int max_q, max_kv;       /* bounds of q_len (1 .. 2^20) and kv_len (1 .. 2^26)                */
    int table_ld;            /* entries of a block_table row, table_ld * page >= max_kv           */
    const int *q_start;      /* [n_seq + 1]                                                       */
    const int *kv_len;       /* [n_seq]                                                           */
    const int *block_table;  /* [n_seq][table_ld]                                                 */
} x100_kv_batch;

/* What x100_kv_append_hip takes per row: projections q [n_head * head_dim], k, v [n_head_kv *
 * head_dim] (the three of one type; they may be columns of one matrix), the optional head norms
 * (RMSNorm over head_dim with weights q_norm / k_norm [head_dim]; NULL: none) and the optional
 * rotation table (NULL: none). */
typedef struct {
    x100_rows q, k, v;            /* q.p NULL (with q_out NULL): keys and values only            */
    const float *q_norm, *k_norm;
    float eps;
    const float *rope;            /* [rope_len][head_dim / 2][2]: cos, sin of each pair (i, i +
                                     head_dim / 2) at a position; rope_len >= max_kv              */
    int rope_len;
} x100_kv_rows;

/* Bytes of each pool (K and V alike); 0 for an invalid configuration. */
size_t x100_kv_pool_bytes(const x100_kv_cfg *cfg);

/* table[p][i] = (cos, sin)(p * base^(-2 i / head_dim)) for p < n_pos, angles in fp64: the rotation
 * of the reference (table qwen_moe_hp.c:799-804).  n_pos <= 2^25.  Once per model. */
int x100_rope_table_hip(int head_dim, int n_pos, float base, float *table, void *stream);

/* Head norms and rotation of q and k, rotated queries to q_out [n_rows][n_head * head_dim] (act_type),
 * keys and values into the pools at the rows' positions.  fp32 throughout (squares of the head norms
 * added by fours, then as a tree over neighbours: heads with norms up to 1e18 in size; with eps = 0 a
 * head of zeros gives 0 / 0, a NaN), one rounding at the store (and the codes' for 4 bits). */
int x100_kv_append_hip(const x100_kv_cfg *cfg, const x100_kv_batch *batch, const x100_kv_rows *rows, void *k_pool,
                       void *v_pool, void *q_out, void *stream);

/* The cached keys and values at the rows' positions, as the cache holds them: k_out, v_out
 * [n_rows][n_head_kv * head_dim] of act_type (4 bits: the value, rounded to act_type).  With q_start
 * spanning whole sequences this unpacks a cache. */
int x100_kv_read_hip(const x100_kv_cfg *cfg, const x100_kv_batch *batch, const void *k_pool, const void *v_pool,
                     void *k_out, void *v_out, void *stream);

/* out[row][head] = sum_p softmax_p(scale * q[row][head] . K_p) V_p over the positions p <= the row's own;
 * q: row r at element r * ldq, out: at r * ldo, heads contiguous, act_type; 0 < scale <= 1e38.  Query head h
 * reads KV head h / (n_head / n_head_kv).  Scores, softmax and sums in fp32, the weights divided by
 * their sum at the end (so bf16 V up to 2^100 in size); for the product with V they are rounded to 16
 * bits (act_type, or fp16 for 4-bit pages), and in fp16 a weight below 2^-29 of the largest is zero.
 * A row that attends to nothing (no position, no valid page, or every score -inf) gives zeros; one
 * with a score that is NaN gives NaN.  Infinities and NaN in positions that a row does not attend to
 * do not reach it.
 * Scratch: x100_attn_paged_workspace_bytes(cfg, batch) bytes (0: none needed, ws may be NULL; it
 * depends on n_rows, n_seq, max_q and max_kv only), 256-byte aligned, any contents, for the _ws form;
 * overlapping calls need distinct buffers.  The plain form uses the library's workspace of the
 * (device, stream), as moe_layer_hip does (x100_moe.h). */
size_t x100_attn_paged_workspace_bytes(const x100_kv_cfg *cfg, const x100_kv_batch *batch);
int x100_attn_paged_hip_ws(const x100_kv_cfg *cfg, const x100_kv_batch *batch, const void *q, int64_t ldq,
                           const void *k_pool, const void *v_pool, float scale, void *out, int64_t ldo, void *ws,
                           size_t ws_bytes, void *stream);
int x100_attn_paged_hip(const x100_kv_cfg *cfg, const x100_kv_batch *batch, const void *q, int64_t ldq,
                        const void *k_pool, const void *v_pool, float scale, void *out, int64_t ldo, void *stream);

#ifdef __cplusplus
}
#endif
#endif
