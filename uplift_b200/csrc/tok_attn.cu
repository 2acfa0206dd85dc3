// C entry points of the packed-sequence attention (include/uplift_tokens.h):
// argument validation, choice of the kernel and launch.

#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include "tok_attn.h"

namespace ula {
namespace tok {
namespace {

int check_sizes(const char* what, int B, int64_t T, int64_t S, int Hq, int Hk, int D, float scale, int dtype) {
  if (dtype != UPLIFT_LA_F32 && dtype != UPLIFT_LA_BF16 && dtype != UPLIFT_LA_F16)
    return fail(UPLIFT_LA_ERR_ARG, "%s: unknown dtype %d", what, dtype);
  // the row limit leaves room for tile arithmetic in 32 bits
  if (B < 0 || T < 0 || S < 0 || T >= (1ll << 31) - 65536 || S >= (1ll << 31) - 65536 || Hq < 1 || Hk < 1 || Hq > 65536)
    return fail(UPLIFT_LA_ERR_SHAPE, "%s: bad sizes B=%d T=%lld S=%lld Hq=%d Hk=%d", what, B, (long long)T,
                (long long)S, Hq, Hk);
  if (Hq % Hk != 0)
    return fail(UPLIFT_LA_ERR_SHAPE, "%s: %d query heads are not a multiple of %d key heads", what, Hq, Hk);
  if (D < 1 || D > UPLIFT_TOK_MAX_ATTN_DIM)
    return fail(UPLIFT_LA_ERR_SHAPE, "%s: head dimension %d not in 1..%d", what, D, UPLIFT_TOK_MAX_ATTN_DIM);
  if (dtype != UPLIFT_LA_F32 && D % 8 != 0)
    return fail(UPLIFT_LA_ERR_SHAPE, "%s: 16-bit tensors need a head dimension that is a multiple of 8 (got %d)", what, D);
  if (!(scale > 0.f) || isinf(scale)) return fail(UPLIFT_LA_ERR_ARG, "%s: scale must be positive and finite", what);
  return UPLIFT_LA_OK;
}

// 16-bit tensors are moved in 16-byte pieces.
int check_rows(const char* what, const char* name, const Rows& r, int64_t rows, int heads, int dtype) {
  if (rows > 0 && r.p == nullptr) return fail(UPLIFT_LA_ERR_ARG, "%s: null %s", what, name);
  if (dtype == UPLIFT_LA_F32 || rows == 0) return UPLIFT_LA_OK;
  if ((reinterpret_cast<uintptr_t>(r.p) & 15u) != 0)
    return fail(UPLIFT_LA_ERR_LAYOUT, "%s: %s is not 16-byte aligned", what, name);
  if ((rows > 1 && (r.t % 8 != 0 || r.t <= 0)) || (heads > 1 && (r.h % 8 != 0 || r.h <= 0)))
    return fail(UPLIFT_LA_ERR_LAYOUT, "%s: the strides of %s must be positive multiples of 8 elements", what, name);
  if (rows > 1 && heads > 1 && r.t % r.h != 0)  // as tensor maps want it
    return fail(UPLIFT_LA_ERR_LAYOUT, "%s: the row stride of %s must be a multiple of its head stride", what, name);
  return UPLIFT_LA_OK;
}

// Strides of axes of one entry do not matter: give them values that do not
// trouble the tensor maps.
Rows rows_of(const void* p, const int64_t* st, int64_t rows, int heads, int D) {
  Rows r{p, st[0], st[1]};
  if (heads == 1) r.h = (D + 7) / 8 * 8;
  if (rows <= 1) r.t = (int64_t)r.h * heads;
  return r;
}

}  // namespace
}  // namespace tok

int tok_device_status(bool clear) {
  const int f = tok::attn_fwd_device_status(clear), b = tok::attn_bwd_device_status(clear);
  return f < 0 || b < 0 ? -1 : (f != 0 ? f : b);
}

}  // namespace ula

extern "C" {

int64_t uplift_tok_attention_workspace(int B, int64_t T, int64_t S, int Hq, int Hk, int D, int dtype) {
  using namespace ula::tok;
  if (T < 1 || Hk < 1 || Hq < Hk || D < 1 || !attn_step_applies(B, T, dtype)) return 0;
  return attn_step_workspace(T, Hq, Hk, D);
}

int uplift_tok_attention_forward(const void* q, const int64_t q_strides[2], const void* k,
                                 const int64_t k_strides[2], const void* v, const int64_t v_strides[2],
                                 void* out, const int64_t out_strides[2], float* lse,
                                 const int32_t* cu_q, const int32_t* cu_k, const int32_t* used_k,
                                 int B, int64_t T, int64_t S, int Hq, int Hk, int D, float scale, int causal,
                                 int dtype, void* workspace, int64_t workspace_bytes, void* stream) {
  using namespace ula;
  using namespace ula::tok;
  const char* what = "uplift_tok_attention_forward";
  int rc = check_sizes(what, B, T, S, Hq, Hk, D, scale, dtype);
  if (rc != UPLIFT_LA_OK) return rc;
  if (q_strides == nullptr || k_strides == nullptr || v_strides == nullptr || out_strides == nullptr)
    return fail(UPLIFT_LA_ERR_ARG, "%s: null strides", what);
  if (T == 0) return UPLIFT_LA_OK;
  if (B > 0 && (cu_q == nullptr || cu_k == nullptr)) return fail(UPLIFT_LA_ERR_ARG, "%s: null sequence starts", what);
  AttnArgs a = {};
  a.q = rows_of(q, q_strides, T, Hq, D);
  a.k = rows_of(k, k_strides, S, Hk, D);
  a.v = rows_of(v, v_strides, S, Hk, D);
  a.out = rows_of(out, out_strides, T, Hq, D);
  if ((rc = check_rows(what, "q", a.q, T, Hq, dtype)) != UPLIFT_LA_OK) return rc;
  if ((rc = check_rows(what, "k", a.k, S, Hk, dtype)) != UPLIFT_LA_OK) return rc;
  if ((rc = check_rows(what, "v", a.v, S, Hk, dtype)) != UPLIFT_LA_OK) return rc;
  if ((rc = check_rows(what, "out", a.out, T, Hq, dtype)) != UPLIFT_LA_OK) return rc;
  a.lse = lse;
  a.pk = Packing{cu_q, cu_k, used_k, B, (int)T, (int)S, causal != 0};
  a.Hq = Hq; a.Hk = Hk; a.D = D; a.scale = scale; a.dtype = dtype;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (dtype == UPLIFT_LA_F32) return attn_simt_forward(a, s);
  if (!attn_step_applies(B, T, dtype)) return attn_tc_forward(a, s);
  if (workspace == nullptr || workspace_bytes < attn_step_workspace(T, Hq, Hk, D) ||
      (reinterpret_cast<uintptr_t>(workspace) & 15u) != 0)
    return fail(UPLIFT_LA_ERR_ARG, "%s: needs a 16-byte aligned workspace of %lld bytes", what,
                (long long)attn_step_workspace(T, Hq, Hk, D));
  return attn_step_forward(a, workspace, s);
}

int uplift_tok_attention_backward(const void* dout, const int64_t dout_strides[2], const void* q,
                                  const int64_t q_strides[2], const void* k, const int64_t k_strides[2],
                                  const void* v, const int64_t v_strides[2], const void* out,
                                  const int64_t out_strides[2], const float* lse, void* dq,
                                  const int64_t dq_strides[2], void* dk, const int64_t dk_strides[2], void* dv,
                                  const int64_t dv_strides[2], float* delta, const int32_t* cu_q,
                                  const int32_t* cu_k, const int32_t* used_k, int B, int64_t T, int64_t S, int Hq,
                                  int Hk, int D, float scale, int causal, int dtype, void* stream) {
  using namespace ula;
  using namespace ula::tok;
  const char* what = "uplift_tok_attention_backward";
  int rc = check_sizes(what, B, T, S, Hq, Hk, D, scale, dtype);
  if (rc != UPLIFT_LA_OK) return rc;
  if (dout_strides == nullptr || q_strides == nullptr || k_strides == nullptr || v_strides == nullptr ||
      out_strides == nullptr || dq_strides == nullptr || dk_strides == nullptr || dv_strides == nullptr)
    return fail(UPLIFT_LA_ERR_ARG, "%s: null strides", what);
  if (T == 0 && S == 0) return UPLIFT_LA_OK;
  if (B > 0 && (cu_q == nullptr || cu_k == nullptr)) return fail(UPLIFT_LA_ERR_ARG, "%s: null sequence starts", what);
  if (T > 0 && (lse == nullptr || delta == nullptr)) return fail(UPLIFT_LA_ERR_ARG, "%s: null lse or delta", what);
  AttnArgs a = {};
  a.q = rows_of(q, q_strides, T, Hq, D);
  a.k = rows_of(k, k_strides, S, Hk, D);
  a.v = rows_of(v, v_strides, S, Hk, D);
  a.out = rows_of(out, out_strides, T, Hq, D);
  a.dout = rows_of(dout, dout_strides, T, Hq, D);
  a.dq = rows_of(dq, dq_strides, T, Hq, D);
  a.dk = rows_of(dk, dk_strides, S, Hk, D);
  a.dv = rows_of(dv, dv_strides, S, Hk, D);
  const struct { const char* name; const Rows* r; int64_t rows; int heads; } all[] = {
      {"q", &a.q, T, Hq}, {"k", &a.k, S, Hk}, {"v", &a.v, S, Hk}, {"out", &a.out, T, Hq},
      {"dout", &a.dout, T, Hq}, {"dq", &a.dq, T, Hq}, {"dk", &a.dk, S, Hk}, {"dv", &a.dv, S, Hk}};
  for (const auto& e : all)
    if ((rc = check_rows(what, e.name, *e.r, e.rows, e.heads, dtype)) != UPLIFT_LA_OK) return rc;
  a.lse = const_cast<float*>(lse);
  a.delta = delta;
  a.pk = Packing{cu_q, cu_k, used_k, B, (int)T, (int)S, causal != 0};
  a.Hq = Hq; a.Hk = Hk; a.D = D; a.scale = scale; a.dtype = dtype;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return dtype == UPLIFT_LA_F32 ? attn_simt_backward(a, s) : attn_tc_backward(a, s);
}

}  // extern "C"
