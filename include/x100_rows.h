/*
 * x100_rows.h -- int8 rows for the int8 GEMM (libx100hip, gfx950): the residual's addition with
 * RMSNorm, and plain rows, to int8 codes with one fp32 scale per row.
 *
 * No counterpart in the reference (its linears quantize one token's activations inside the call,
 * qwen_moe.c:101-107).  The rows of gemm_hip_i8_dev's A matrix are made here, and the int32 rows of
 * its C matrix are read here: a row tensor of type X100_T_I32 stands for
 * ((float)c * row_scale[row]) * col_scale[column].  With A's codes and scales from these calls and
 * int8 weights with a scale per column, row_scale is A's scale array and col_scale the weights'.
 *
 * Codes: t = the row's values, amax = max |t|, code = rint(t * f) with f = 127 * (1 / amax) in fp32
 * (two roundings; ties to even), scale = amax / 127.  A row of zeros (or amax < 2^-100) has codes 0 and
 * scale 0; a row with a t that is an infinity or a NaN has codes 0 and scale NaN.  In add_rmsnorm_i8
 * t = h * weight and the norm's factor goes into the scale alone (it cancels in the code), so that the
 * codes do not depend on the order in which a sum was taken: they are the same for every layout,
 * alignment and launch.
 *
 * All pointers are device pointers; asynchronous on stream (a hipStream_t as void *, NULL = the
 * default stream); no workspace; capturable.  Every argument is checked before anything is
 * enqueued.
 */
#ifndef X100_HIP_ROWS_H
#define X100_HIP_ROWS_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* Element types (ggml type ids). */
#define X100_T_F32   0
#define X100_T_F16   1
#define X100_T_I32  26
#define X100_T_BF16 30

#define X100_ROWS_MAX_D 16384   /* longest row of add_rmsnorm_i8 / quant_i8 */

/* Rows of a device matrix: row r starts at element r * ld.  row_scale [n_rows] and col_scale [d]
 * belong to X100_T_I32 (both required there, and NULL for the other types). */
typedef struct {
    int type;
    const void *p;
    int64_t ld;
    const float *row_scale, *col_scale;
} x100_rows;

/* q[n_rows][d] (contiguous) and scale[n_rows] from the rows x (any of the four types).
 * 1 <= d <= X100_ROWS_MAX_D, x->ld >= d, 0 <= n_rows < 2^24 (2^22 for d > 4096). */
int x100_quant_i8_hip(int n_rows, int d, const x100_rows *x, int8_t *q, float *scale, void *stream);

/* h = x + delta, rounded to x's type and stored (h: row r at element r * ldh; h == x->p with ldh ==
 * x->ld updates in place; no other output overlaps an input); then RMSNorm of the stored h with
 * weight[d] and eps, as codes and scales:
 *   r = 1 / sqrt(mean(h^2) + eps),  t = h * weight,  scale = max|t| * r / 127.
 * x: F32, F16 or BF16; delta: any of the four types, or NULL for no addition (h is then not written
 * and may be NULL); n_rows and d as in quant_i8.  Squares are summed in fp64, so h of any size;
 * eps >= 0, and a row of zeros has scale 0 for eps = 0 too. */
int x100_add_rmsnorm_i8_hip(int n_rows, int d, const x100_rows *x, const x100_rows *delta, const float *weight,
                            float eps, void *h, int64_t ldh, int8_t *q, float *scale, void *stream);

#ifdef __cplusplus
}
#endif
#endif
