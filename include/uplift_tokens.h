/*
 * uplift_tokens.h -- C ABI of the B200 (sm_100a) token-sequence operators:
 * the attention of transformer tokens (the backbone features the upsampler
 * consumes, or any packed token sequences) and the per-head norm with
 * position rotation that feeds it.
 *
 * Token tensors are [rows, heads, D] with channel stride 1; `strides` gives
 * the row and head strides in elements (views into a fused projection
 * output work).  Sequences are packed: sequence b owns the rows
 * cu[b] .. cu[b + 1] - 1 of its tensor; cu is a device array of B + 1
 * ascending int32 values.  Row numbers read from device arrays are clamped
 * to the tensors, so no content of these arrays makes a kernel leave them.
 *
 * dtype: UPLIFT_LA_F32 / BF16 / F16 (uplift_la.h).  Products, softmax
 * statistics, norms and sums are fp32; each result is rounded once to the
 * storage type.  The entry points allocate nothing, never synchronise, are
 * deterministic (no floating-point atomics) and can be captured into CUDA
 * graphs; each returns UPLIFT_LA_OK or an error code (message in
 * uplift_la_last_error()).
 */
#ifndef UPLIFT_TOKENS_H_
#define UPLIFT_TOKENS_H_

#include <stddef.h>
#include <stdint.h>

#include "uplift_la.h"

#ifdef __cplusplus
extern "C" {
#endif

/* largest head dimension of each operator */
#define UPLIFT_TOK_MAX_NORM_DIM 256
#define UPLIFT_TOK_MAX_ATTN_DIM 128

/*
 * RMS norm of every query and key head and the position rotation, one pass:
 *
 *   y = x / sqrt(mean(x^2) + eps) * weight            (over the D channels)
 *   (a, b) -> (a c - b s, b c + a s)                  for R / 2 channel pairs
 *
 * with c, s = cos, sin [positions[t]][i] for pair i: channels (i, i + R/2),
 * or (2i, 2i + 1) when interleaved; channels R .. D - 1 are not rotated.
 *
 *   q [T, Hq, D], k [T, Hk, D]; q_out, k_out the same shapes, not overlapping
 *   q_weight, k_weight [D] of weight_dtype, or NULL (ones)
 *   cos, sin  [P, R / 2] fp32, contiguous
 *   positions [T] int32 or int64 (positions64 = 1), or NULL: row t of the
 *             table for token t (then P >= T).  A negative position leaves
 *             the token unrotated (class and register tokens); a position
 *             >= P makes the token's rotated outputs and its gradients NaN.
 *   D <= UPLIFT_TOK_MAX_NORM_DIM; R even, 0 <= R <= D
 */
int uplift_tok_norm_rotate(const void* q, const int64_t q_strides[2], void* q_out, const int64_t q_out_strides[2],
                           const void* k, const int64_t k_strides[2], void* k_out, const int64_t k_out_strides[2],
                           const void* q_weight, const void* k_weight, int weight_dtype,
                           const float* cos, const float* sin, const void* positions, int positions64,
                           int64_t T, int64_t P, int Hq, int Hk, int D, int R, float eps, int interleaved,
                           int dtype, void* stream);

/*
 * Gradients of uplift_tok_norm_rotate: dq, dk from dq_out, dk_out (rows of
 * the forward's outputs) and the forward's inputs, and dweights: the
 * gradients of q_weight and k_weight, [2][D] fp32 (written, not added to).
 * partial: workspace of uplift_tok_norm_rotate_partial_floats(D) floats.
 */
int64_t uplift_tok_norm_rotate_partial_floats(int D);
int uplift_tok_norm_rotate_backward(const void* dq_out, const int64_t dq_out_strides[2],
                                    const void* dk_out, const int64_t dk_out_strides[2],
                                    const void* q, const int64_t q_strides[2], const void* k,
                                    const int64_t k_strides[2], void* dq, const int64_t dq_strides[2],
                                    void* dk, const int64_t dk_strides[2], float* dweights,
                                    const void* q_weight, const void* k_weight, int weight_dtype,
                                    const float* cos, const float* sin, const void* positions, int positions64,
                                    float* partial, int64_t T, int64_t P, int Hq, int Hk, int D, int R, float eps,
                                    int interleaved, int dtype, void* stream);

/*
 * Attention over packed sequences with grouped heads.  Sequence b has the
 * queries cu_q[b] .. cu_q[b + 1] - 1 and the n_k keys from cu_k[b] on, n_k
 * the length of its key segment, or used_k[b] if that is smaller.  Query i
 * of n_q sees key j if j < n_k and, when causal, j <= i + n_k - n_q (the
 * last query sees every key).  Query head h reads key head h / (Hq / Hk).
 *
 *   out_i = sum_j softmax_j(scale q_i . k_j) v_j
 *   lse_i = log sum_j exp(scale q_i . k_j)
 *
 * A query that sees no key gets out = 0 and lse = -inf, and so do rows of
 * no sequence.  What keys that a query does not see hold (NaN, infinities)
 * does not reach its output.
 *
 *   q, out [T, Hq, D]; k, v [S, Hk, D]; lse [Hq, T] fp32 or NULL
 *   used_k [B] int32 or NULL; Hq a multiple of Hk; D <= UPLIFT_TOK_MAX_ATTN_DIM
 *   scale  positive and finite
 *   workspace: uplift_tok_attention_workspace(...) bytes, 16-byte aligned
 *             (may be 0 / NULL)
 * bf16 / fp16: D a multiple of 8; pointers 16-byte aligned, strides
 * multiples of 8 elements and row strides multiples of the head stride
 * (UPLIFT_LA_ERR_LAYOUT otherwise).
 */
int64_t uplift_tok_attention_workspace(int B, int64_t T, int64_t S, int Hq, int Hk, int D, int dtype);
int uplift_tok_attention_forward(const void* q, const int64_t q_strides[2], const void* k,
                                 const int64_t k_strides[2], const void* v, const int64_t v_strides[2],
                                 void* out, const int64_t out_strides[2], float* lse,
                                 const int32_t* cu_q, const int32_t* cu_k, const int32_t* used_k,
                                 int B, int64_t T, int64_t S, int Hq, int Hk, int D, float scale, int causal,
                                 int dtype, void* workspace, int64_t workspace_bytes, void* stream);

/*
 * Gradients of uplift_tok_attention_forward from dout, its inputs, out and
 * lse.  dq, dk, dv are written whole: zero for rows of no sequence and keys
 * that no query sees.  delta: workspace of T * Hq floats.
 */
int uplift_tok_attention_backward(const void* dout, const int64_t dout_strides[2], const void* q,
                                  const int64_t q_strides[2], const void* k, const int64_t k_strides[2],
                                  const void* v, const int64_t v_strides[2], const void* out,
                                  const int64_t out_strides[2], const float* lse, void* dq,
                                  const int64_t dq_strides[2], void* dk, const int64_t dk_strides[2], void* dv,
                                  const int64_t dv_strides[2], float* delta, const int32_t* cu_q,
                                  const int32_t* cu_k, const int32_t* used_k, int B, int64_t T, int64_t S, int Hq,
                                  int Hk, int D, float scale, int causal, int dtype, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* UPLIFT_TOKENS_H_ */
