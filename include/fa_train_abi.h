/*
 * frame_analytics_amd -- C ABI of the operators of a training step that stand
 * beside the losses: attention with a learned relative position bias, that bias
 * by itself, and the orthogonalised update of weight matrices.
 *
 * The conventions are those of fa_abi.h: int status (FA_OK, a code of fa_abi.h, or
 * a negated hipError_t), caller-owned buffers, an explicit device ordinal and
 * stream, no allocation and no synchronisation.  None of these entry points has a
 * counterpart in the reference.
 */
#ifndef FRAME_ANALYTICS_AMD_TRAIN_ABI_H
#define FRAME_ANALYTICS_AMD_TRAIN_ABI_H

#include "fa_abi.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Relative positions.  Token t has the whole-number code c(t): on a line (grid_w
 * = 0) its position, in a window grid_w tokens wide t + (grid_w - 1) * (t / grid_w),
 * so that the difference of two codes tells the two coordinates' differences.
 * A pair (query i, key j) takes the table's row row_of[clamp(c(i) - c(j) - lo, 0,
 * n - 1)]: row_of is a device array of n int32, each in [0, rows), equal rows
 * standing next to one another.  1 <= n <= FA_REL_MAX. */
#define FA_REL_MAX 4225

/* OR-ed into an attention's dtype: table and dtable are float32, whatever q is. */
#define FA_TABLE_F32 0x100

/*
 * out[h, i, j] = table[row(i, j), h], i < Lq, j < Lk, query i standing at position
 * q_start + i of a line (0 in a window).  table: [rows, H] contiguous, out: [H, Lq,
 * Lk] contiguous, both of `dtype` (FA_F16, FA_BF16, FA_F32).
 */
FA_API int fa_gpu_rel_bias(const void* table, int dtype, int rows, int H, int Lq, int Lk,
                           const int* row_of, int lo, int n, int grid_w, int64_t q_start,
                           void* out, int device, void* stream);

/* Bytes of fa_gpu_rel_bias_backward's workspace (8-byte aligned). */
FA_API int fa_gpu_rel_bias_workspace(int H, int Lq, int Lk, int n, int64_t* out_bytes);

/*
 * dtable[r, h] = sum of up[h, i, j] over row(i, j) = r, in float32 and a fixed
 * order, rounded once to `dtype`.  up: strides {head, query, key} in elements.
 */
FA_API int fa_gpu_rel_bias_backward(const void* up, const int64_t* up_strides, int dtype,
                                    int rows, int H, int Lq, int Lk, const int* row_of, int lo,
                                    int n, int grid_w, int64_t q_start, void* dtable,
                                    void* workspace, int64_t workspace_bytes, int device,
                                    void* stream);

/*
 * out = softmax(scale * q k^T + bias) v over the keys that query i of batch entry
 * b may see: j < key_lengths[b] (null: Lk), j <= start + i where causal, and
 * mask[b % mask_b, h, i, j] is 1 (bytes, 0 or 1; null: all).  A row that sees none is 0.
 *
 * q, out: [B, H, Lq, D]; k, v: [B, Hk, Lk, D], H a multiple of Hk: query head h
 * reads key head h / (H / Hk).  strides: 12 int64 in elements, {batch, head, token}
 * of q, k, v and out; the last dimension has stride 1, and 256 tokens lie within 2^31
 * bytes (FA_E_SHAPE).  1 <= D <= 128.
 * start: q_starts[b] (int32, device) or, where that is null, q_start; both are taken
 * as within +-2^30.  mask_strides: {batch, head, query, key} in bytes.
 * lse: null, or what the backward pass reads, 16-byte aligned: [2, B, H, Lq] float32, with
 * which a row's weights are 2^(score log2(e) - the first) times the second (the first +inf
 * for a row that sees nothing); for FA_F16 and FA_BF16 with grid_w 0, from the next multiple
 * of 16 bytes on, [B, H, Lq, D] of dtype: what the rounding of out left.  (Windows of up to
 * 64 tokens may leave it unwritten.)
 * workspace: fa_gpu_rel_attention_workspace bytes, 16-byte aligned (0: may be null).
 */
FA_API int fa_gpu_rel_attention_workspace(int B, int H, int Hk, int Lq, int Lk, int D, int n,
                                          int device, int64_t* out_bytes);
FA_API int fa_gpu_rel_attention(const void* q, const void* k, const void* v, int dtype, int B,
                                int H, int Hk, int Lq, int Lk, int D, const int64_t* strides,
                                const void* table, int rows, const int* row_of, int lo, int n,
                                int grid_w, int64_t q_start, const int* q_starts,
                                const int* key_lengths, const uint8_t* mask, int mask_b,
                                const int64_t* mask_strides, int causal, double scale, void* out,
                                float* lse, void* workspace, int64_t workspace_bytes, int device,
                                void* stream);

/*
 * Gradients of the above.  strides: 24 int64, {batch, head, token} of q, k, v, out,
 * dout, dq, dk, dv.  out and lse are the forward's.  dtable: [rows, H] or null.
 * Sums over heads that share a key head and over the batch are taken in float32 in
 * a fixed order; each result is rounded once.
 */
FA_API int fa_gpu_rel_attention_backward_workspace(int B, int H, int Hk, int Lq, int Lk, int D, int n,
                                                   int grid_w, int need_table, int device,
                                                   int64_t* out_bytes);
FA_API int fa_gpu_rel_attention_backward(
    const void* q, const void* k, const void* v, const void* out, const void* dout,
    const float* lse, int dtype, int B, int H, int Hk, int Lq, int Lk, int D,
    const int64_t* strides, const void* table, int rows, const int* row_of, int lo, int n,
    int grid_w, int64_t q_start, const int* q_starts, const int* key_lengths, const uint8_t* mask,
    int mask_b, const int64_t* mask_strides, int causal, double scale, void* dq, void* dk,
    void* dv, void* dtable, void* workspace, int64_t workspace_bytes, int device, void* stream);

/*
 * out = X_steps of X_0 = g / (|g| + eps), X <- a X + (b A + c A^2) X, A = X X^T,
 * for each of `batch` contiguous [rows, cols] matrices (transposed inside where rows
 * > cols); |g| is the Frobenius norm.  g, out: `dtype` (FA_F16, FA_BF16, FA_F32).
 * FA_E_ARG where float16 would not hold what these coefficients lead to: the largest
 * singular value that a step may be given, from 1 on, has to stay within 1/64 and 5.6,
 * and |b s^2 + c s^4| below 63 for all up to it.
 */
FA_API int fa_gpu_orthogonalize_workspace(int dtype, int batch, int rows, int cols,
                                          int64_t* out_bytes);
FA_API int fa_gpu_orthogonalize(const void* g, int dtype, int batch, int rows, int cols, int steps,
                                double a, double b, double c, double eps, void* out,
                                void* workspace, int64_t workspace_bytes, int device,
                                void* stream);

#ifdef __cplusplus
}
#endif
#endif
