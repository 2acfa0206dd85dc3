/*
 * uplift_tokens.h -- C ABI of the B200 (sm_100a) token-sequence operators:
 * the attention of transformer tokens (the backbone features the upsampler
 * consumes, or any packed token sequences) and the per-head norm with
 * position rotation that feeds it.
 *
 * Token tensors are [rows, heads, D] with channel stride 1, given as
 * uplift_tok_rows: views into a fused projection output work.  Sequences are
 * packed: sequence b owns the rows cu[b] .. cu[b + 1] - 1 of its tensor; cu is a device array of B + 1
 * ascending int32 values.  Row numbers read from device arrays are clamped
 * to the tensors, so no content of these arrays makes a kernel leave them.
 *
 * dtype: UPLIFT_LA_F32 / BF16 / F16 (uplift_la.h).  Products, softmax
 * statistics, norms and sums are fp32; each result is rounded once to the
 * storage type.  The entry points allocate nothing, never synchronise, are
 * deterministic (no floating-point atomics) and can be captured into CUDA
 * graphs; each returns UPLIFT_LA_OK or an error code (message in
 * uplift_la_last_error()).  uplift_la_set_max_ctas() holds for the attention's
 * tensor-core launches.  A tensor-core launch whose bounded wait ran out is
 * reported by uplift_la_device_status() and the registered host status word.
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

/* A token tensor: first element, and the row and head strides in elements. */
typedef struct {
  void* data;
  int64_t row, head;
} uplift_tok_rows;

/*
 * RMS norm of every query and key head and the position rotation, one pass:
 *
 *   y = x / sqrt(mean(x^2) + eps) * weight            (over the D channels)
 *   (a, b) -> (a c - b s, b c + a s)                  for R / 2 channel pairs
 *
 * with c, s = cos, sin [positions[t]][i] for pair i: channels (i, i + R/2),
 * or (2i, 2i + 1) when interleaved; channels R .. D - 1 are not rotated.
 */
typedef struct {
  int64_t size;               /* sizeof(uplift_tok_norm_rotate_args) */
  uplift_tok_rows q, k;       /* [T, Hq, D], [T, Hk, D] */
  uplift_tok_rows q_out, k_out; /* the outputs (not overlapping the inputs); backward: their gradients */
  uplift_tok_rows dq, dk;     /* backward only: gradients of q and k */
  const void* q_weight;       /* [D] of weight_dtype, or NULL: ones */
  const void* k_weight;
  const float* cos;           /* [P, R / 2], contiguous */
  const float* sin;
  const void* positions;      /* [T] int32, or int64 (positions64), or NULL: row t of the table for token t (P >= T).
                                 Negative: the token is not rotated (class and register tokens).  >= P: its rotated
                                 outputs and its gradients are NaN. */
  void* dweights;             /* backward only: gradients of q_weight and k_weight, [2][D] of weight_dtype, or NULL */
  float* partial;             /* backward only: workspace of uplift_tok_norm_rotate_partial_floats(D) floats */
  int64_t T, P;
  int32_t Hq, Hk;
  int32_t D, R;               /* D <= UPLIFT_TOK_MAX_NORM_DIM; R even, 0 <= R <= D */
  float eps;
  int32_t interleaved, weight_dtype, positions64, dtype;
  int32_t reserved;           /* 0 */
} uplift_tok_norm_rotate_args;

int uplift_tok_norm_rotate(const uplift_tok_norm_rotate_args* args, void* stream);
/* The gradients dq, dk and dweights from the inputs and the outputs' gradients. */
int uplift_tok_norm_rotate_backward(const uplift_tok_norm_rotate_args* args, void* stream);
int64_t uplift_tok_norm_rotate_partial_floats(int D);

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
 * does not reach its output or its gradient, nor does what that query and its
 * dout hold reach the gradients of these keys.
 *
 * fp16 gradients: the weights' gradients are rounded to fp16 as those of dout
 * times a power of two, which is 1 while the largest |dout| lies between 2^-5 and
 * 2^9 and brings it there otherwise.
 *
 * bf16 / fp16: D a multiple of 8; tensors 16-byte aligned, strides
 * multiples of 8 elements and row strides multiples of the head stride
 * (UPLIFT_LA_ERR_LAYOUT otherwise).
 */
typedef struct {
  int64_t size;             /* sizeof(uplift_tok_attention_args) */
  uplift_tok_rows q;        /* [T, Hq, D] */
  uplift_tok_rows k, v;     /* [S, Hk, D] */
  uplift_tok_rows out;      /* [T, Hq, D] */
  uplift_tok_rows out_lo;   /* [T, Hq, D] or data = NULL; 16-bit types only: what the rounding of out left
                               (forward: written; backward: read, so that the gradients do not carry it) */
  uplift_tok_rows dout;     /* backward only: gradient of out */
  uplift_tok_rows dq, dk, dv; /* backward only: the gradients, written whole: zero for rows of no sequence and keys that
                                 no query sees */
  float* lse;               /* [Hq, T]; forward: written unless NULL; backward: read */
  float* delta;             /* backward only: workspace of T * Hq + 16 floats */
  const int32_t* cu_q;      /* [B + 1] */
  const int32_t* cu_k;
  const int32_t* used_k;    /* [B] or NULL */
  void* workspace;          /* forward only: uplift_tok_attention_workspace(...) bytes, 16-byte aligned */
  int64_t workspace_bytes;
  int64_t T, S;
  int32_t B, Hq, Hk;        /* Hq a multiple of Hk */
  int32_t D;                /* <= UPLIFT_TOK_MAX_ATTN_DIM */
  float scale;              /* positive and finite */
  int32_t causal, dtype;
  int32_t reserved;         /* 0 */
} uplift_tok_attention_args;

int uplift_tok_attention_forward(const uplift_tok_attention_args* args, void* stream);
/* The gradients dq, dk and dv from the inputs, out, lse and dout. */
int uplift_tok_attention_backward(const uplift_tok_attention_args* args, void* stream);
int64_t uplift_tok_attention_workspace(int B, int64_t T, int64_t S, int Hq, int Hk, int D, int dtype);

#ifdef __cplusplus
}
#endif

#endif /* UPLIFT_TOKENS_H_ */
