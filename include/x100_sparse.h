/*
 * x100_sparse.h -- sparse attention over the paged KV cache (libx100hip, gfx950): every query attends to a few
 * blocks of its sequence, which a cheap score selects.
 *
 * No counterpart in the reference (its attention reads the whole cache, qwen_moe.c:284-292).  A block is a page of the
 * cache (x100_paged.h has the cache, the batch and what happens to bad lengths and pages); block b of a sequence has the
 * positions b * page .. b * page + page - 1.  After x100_kv_append_hip, per layer:
 *   x100_kv_means_hip      the mean key of each page that the new rows complete, beside the cache;
 *   x100_attn_select_hip   per row and KV head, the blocks with the largest scores (row's queries) . (mean key);
 *   x100_attn_sparse_hip   attention over the positions of those blocks up to the row's own.
 * The query heads of a KV head share their blocks.  Where a row has no more than n_sel blocks, all are selected and
 * the attention is the dense one.
 *
 * All pointers are device pointers unless they are the argument structures; every call is asynchronous on
 * stream and capturable.  All arguments that the host can see are checked before anything is enqueued.
 * X100_EINVAL also for a batch that no launch can hold: n_rows * n_head_kv above 2^28 - 2^14 in the means, of 2^24 and
 * more in the selection, and n_rows * n_head_kv * splits of 2^24 in the attention (splits: 1 where there are many rows).
 * Outputs overlap no input.
 */
#ifndef X100_HIP_SPARSE_H
#define X100_HIP_SPARSE_H

#include <stddef.h>
#include <stdint.h>

#include "x100_paged.h"

#ifdef __cplusplus
extern "C" {
#endif

#define X100_SPARSE_MAX_SEL 512        /* blocks of a list                                                       */
#define X100_SPARSE_MAX_BLOCKS 16384   /* blocks of a sequence that x100_attn_select_hip looks at: max_kv / page */

typedef struct {
    int n_sel;     /* blocks of a row's list, 1 .. X100_SPARSE_MAX_SEL                                   */
    int n_first;   /* the sequence's first blocks that every list has (0: none)                          */
    int n_last;    /* and its last ones up to the row's own, which is the last (>= 1); n_first + n_last <= n_sel */
} x100_kv_sel;

/* Bytes of the means of a cache, one pool per layer: [n_pages][n_head_kv][head_dim] of act_type; 0 for an invalid
 * configuration. */
size_t x100_kv_means_bytes(const x100_kv_cfg *cfg);

/* means of every page whose last position is one of the batch's rows: the mean of the page's keys as the cache holds
 * them (summed in fp64, one rounding to act_type by way of fp32).  Other entries are left as they were: those of pages
 * that are not full are never read.  means: 16-byte aligned. */
int x100_kv_means_hip(const x100_kv_cfg *cfg, const x100_kv_batch *batch, const void *k_pool, void *means, void *stream);

/* sel[row][KV head][n_sel]: the blocks of each row's list, ascending, -1 behind them.  A row at position p has the blocks
 * 0 .. p / page.  Its first n_first and last n_last ones are in its list; of the others those with the largest
 * scores sum_h q[row][h] . means[page of the block][KV head] (the KV head's query heads h; in fp64), a tie to the
 * lower block, a NaN as -infinity.  A block without a page (a number outside 0 .. n_pages - 1) is in no list.
 * Rows before position 0 have empty lists; rows of no sequence keep what sel held.
 * q as in x100_attn_paged_hip; (max_kv - 1) / page < X100_SPARSE_MAX_BLOCKS; sel 4-byte aligned. */
int x100_attn_select_hip(const x100_kv_cfg *cfg, const x100_kv_batch *batch, const x100_kv_sel *pick, const void *q,
                         int64_t ldq, const void *means, int *sel, void *stream);

/* out[row][head] = sum_p softmax_p(scale * q[row][head] . K_p) V_p over the positions p <= the row's own of the blocks of
 * sel[row][KV head][0 .. n_sel - 1]; q, ldq, scale, out, ldo, numerics, rows that attend to nothing, infinities and NaN as in
 * x100_attn_paged_hip.  A list ends at its first entry that is not above the one before it (so at the first -1), or
 * lies behind the row's own block.
 * Scratch as there: x100_attn_sparse_workspace_bytes(cfg, batch, n_sel) bytes (0: none needed; it depends on n_rows only),
 * 256-byte aligned, any contents; the plain form takes the library's workspace of the (device, stream). */
size_t x100_attn_sparse_workspace_bytes(const x100_kv_cfg *cfg, const x100_kv_batch *batch, int n_sel);
int x100_attn_sparse_hip_ws(const x100_kv_cfg *cfg, const x100_kv_batch *batch, const void *q, int64_t ldq,
                            const void *k_pool, const void *v_pool, float scale, const int *sel, int n_sel, void *out,
                            int64_t ldo, void *ws, size_t ws_bytes, void *stream);
int x100_attn_sparse_hip(const x100_kv_cfg *cfg, const x100_kv_batch *batch, const void *q, int64_t ldq,
                         const void *k_pool, const void *v_pool, float scale, const int *sel, int n_sel, void *out,
                         int64_t ldo, void *stream);

#ifdef __cplusplus
}
#endif
#endif
