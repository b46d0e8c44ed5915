// Internal launch interfaces between the C-ABI layer (capi.hip) and the kernel files.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "gemm_plan.h"
#include "x100_decode.h"
#include "x100_fp8.h"
#include "x100_moe.h"
#include "x100_paged.h"
#include "x100_rows.h"
#include "x100_sparse.h"

// acc: C += A.B; otherwise the overwrite form C = A.B.
hipError_t x100_gemm_i8_launch(int M, int N, int K, const int8_t *A, const int8_t *B, int32_t *C,
                               hipStream_t s, int variant, bool acc);
hipError_t x100_zero_i32_launch(int32_t *C, size_t n, hipStream_t s);

size_t x100_q_packed_bytes(int qtype, int N, int K);
hipError_t x100_q_pack_launch(int qtype, int N, int K, const void *src, void *dst, hipStream_t s);
hipError_t x100_qgemv_launch(int qtype, int M, int N, int K, const void *w, const float *x, float *y,
                             hipStream_t s);
// Two one-row GEMVs of one weight type on the same x (packed weights w0: N0 x K, w1: N1 x K) in one
// launch, each row's result that of x100_qgemv_launch; hipErrorNotSupported (nothing launched)
// for shapes or types that have no merged form.
hipError_t x100_qgemv2_launch(int qtype, int N0, const void *w0, float *y0, int N1, const void *w1, float *y1, int K,
                              const float *x, hipStream_t s);
// The same two plus a third one-row GEMV on the int8 path (qtype2: Q8_0, Q5_K or Q6_K, packed
// w2: N2 x K) in one launch; hipErrorNotSupported (nothing launched) outside the shapes it has.
// With nrm, x is a raw row and the products take RMSNorm(x) with weights nrm and eps (the
// operations of the norm launch it replaces, bit for bit).
hipError_t x100_qgemv3_launch(int qtype, int N0, const void *w0, float *y0, int N1, const void *w1, float *y1,
                              int qtype2, int N2, const void *w2, float *y2, int K, const float *x, const float *nrm,
                              float eps, hipStream_t s);
// True when x100_qgemv_launch accepts the shape (it then launches without further checks).
bool x100_qgemv_supported(int qtype, int M, int N, int K);
hipError_t x100_check_quant_div_launch(uint32_t lo, uint32_t hi, unsigned long long *cnt, hipStream_t s);

size_t x100_moe_workspace_bytes(int M, int d, int ff, int n_exp, int n_act);
// flags: X100_MOE_RESIDUAL, X100_MOE_TILED (x100_moe.h).
hipError_t x100_moe_launch(int M, int d, int ff, int n_exp, int n_act, const float *hn, const float *R,
                           const void *Wg, const void *Wu, const void *Wd, float *out, int flags,
                           int *sel, float *sw, void *workspace, hipStream_t s);
hipError_t x100_moe_tile_pack(int n_exp, int rows, int K, const void *src, void *dst, hipStream_t s);
// One token row of a decoder layer with the step before the MoE block folded in: h <- (h + o) +
// MoE(rmsnorm(h + o, nrm)), the bits of h += o, hn = rmsnorm(h, nrm), x100_moe_launch(hn, out = h,
// residual).  Supported (x100_moe_norm_supported) for d = 2048, flags X100_MOE_RESIDUAL (ggml-layout
// experts, as the decoder layer keeps them).
bool x100_moe_norm_supported(int d, int ff, int n_exp, int n_act, int flags);
hipError_t x100_moe_norm_launch(int d, int ff, int n_exp, int n_act, float *h, const float *o, const float *nrm,
                                float eps, const float *R, const void *Wg, const void *Wu, const void *Wd, int flags,
                                int *sel, float *sw, void *workspace, hipStream_t s);

hipError_t x100_gemv_tile_launch(int int4, int M, int N, int K, const void *W, const int8_t *x, int32_t *y,
                                 hipStream_t s);

// Attention half of a decoder layer (attn.hip).  ws holds x100_attn_workspace_bytes(c) bytes; with
// w->ffn_norm set, *hn_out receives rmsnorm(h, ffn_norm) (inside ws) for the MoE block.  With
// o_out, h += o and the norm are left to the caller (x100_moe_norm_launch): *o_out receives o.
size_t x100_attn_workspace_bytes(const x100_layer_cfg *c);
hipError_t x100_attn_launch(const x100_layer_cfg *c, const x100_layer_weights *w, int pos, float *h,
                            float *ws, float **hn_out, hipStream_t s, float **o_out = nullptr);


// int8 rows (rows.hip); arguments as checked by the entry points.
hipError_t x100_quant_i8_launch(int n_rows, int d, const x100_rows *x, int8_t *q, float *scale, hipStream_t s);
hipError_t x100_add_rmsnorm_i8_launch(int n_rows, int d, const x100_rows *x, const x100_rows *delta,
                                      const float *weight, float eps, void *h, int64_t ldh, int8_t *q, float *scale,
                                      hipStream_t s);

// 8-bit floating point (x100_fp8.h): rows (rows.hip), and the product (gemm_fp8.hip); arguments as checked.
hipError_t x100_quant_fp8_launch(int n_rows, int d, const x100_rows *x, const x100_fp8 *q, hipStream_t s);
hipError_t x100_add_rmsnorm_fp8_launch(int n_rows, int d, const x100_rows *x, const x100_rows *delta,
                                       const float *weight, float eps, void *h, int64_t ldh, const x100_fp8 *q,
                                       hipStream_t s);
hipError_t x100_gemm_fp8_launch(int M, int N, int K, const x100_fp8 *a, const x100_fp8 *w, int c_type, void *c,
                                int64_t ldc, hipStream_t s);

// Paged KV cache (paged.hip) and attention over it (attn_paged.hip).  ws holds the bytes that
// x100_attn_paged_workspace gives; a batch that it refuses is not launched.
hipError_t x100_rope_table_launch(int head_dim, int n_pos, float base, float *table, hipStream_t s);
hipError_t x100_kv_append_launch(const x100_kv_cfg &c, const x100_kv_batch &b, const x100_kv_rows &r, void *kp,
                                 void *vp, void *q_out, hipStream_t s);
hipError_t x100_kv_read_launch(const x100_kv_cfg &c, const x100_kv_batch &b, const void *kp, const void *vp,
                               void *k_out, void *v_out, hipStream_t s);
bool x100_attn_paged_workspace(const x100_kv_cfg &c, const x100_kv_batch &b, size_t *bytes);   // false: past one launch
hipError_t x100_attn_paged_launch(const x100_kv_cfg &c, const x100_kv_batch &b, const void *q, int64_t ldq,
                                  const void *kp, const void *vp, float scale, void *out, int64_t ldo, void *ws,
                                  hipStream_t s);

// Sparse attention: block means and selection (sparse.hip), attention over lists of blocks (attn_paged.hip).
hipError_t x100_kv_means_launch(const x100_kv_cfg &c, const x100_kv_batch &b, const void *kp, void *means, hipStream_t s);
hipError_t x100_attn_select_launch(const x100_kv_cfg &c, const x100_kv_batch &b, const x100_kv_sel &pick, const void *q,
                                   int64_t ldq, const void *means, int *sel, hipStream_t s);
bool x100_attn_sparse_workspace(const x100_kv_cfg &c, const x100_kv_batch &b, int n_sel, size_t *bytes);   // false: past one launch
hipError_t x100_attn_sparse_launch(const x100_kv_cfg &c, const x100_kv_batch &b, const void *q, int64_t ldq,
                                   const void *kp, const void *vp, float scale, const int *sel, int n_sel, void *out,
                                   int64_t ldo, void *ws, hipStream_t s);
