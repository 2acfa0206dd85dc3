// C entry points of the packed-sequence attention (include/uplift_tokens.h):
// argument validation, choice of the kernel and launch.

#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include <algorithm>

#include "tok_attn.h"

namespace ula {
namespace tok {
namespace {

int check_sizes(const char* what, const uplift_tok_attention_args* a) {
  if (a == nullptr || a->size != (int64_t)sizeof(*a)) return fail(UPLIFT_LA_ERR_ARG, "%s: no arguments, or of another version", what);
  if (a->dtype != UPLIFT_LA_F32 && a->dtype != UPLIFT_LA_BF16 && a->dtype != UPLIFT_LA_F16)
    return fail(UPLIFT_LA_ERR_ARG, "%s: unknown dtype %d", what, a->dtype);
  // the row limit leaves room for tile arithmetic in 32 bits
  constexpr int64_t kMaxRows = (1ll << 31) - 65536;
  if (a->B < 0 || a->B >= kMaxRows || a->T < 0 || a->S < 0 || a->T >= kMaxRows || a->S >= kMaxRows || a->Hq < 1 || a->Hk < 1 || a->Hq > 65536)
    return fail(UPLIFT_LA_ERR_SHAPE, "%s: bad sizes B=%d T=%lld S=%lld Hq=%d Hk=%d", what, a->B, (long long)a->T,
                (long long)a->S, a->Hq, a->Hk);
  if (a->Hq % a->Hk != 0)
    return fail(UPLIFT_LA_ERR_SHAPE, "%s: %d query heads are not a multiple of %d key heads", what, a->Hq, a->Hk);
  if (a->D < 1 || a->D > UPLIFT_TOK_MAX_ATTN_DIM)
    return fail(UPLIFT_LA_ERR_SHAPE, "%s: head dimension %d not in 1..%d", what, a->D, UPLIFT_TOK_MAX_ATTN_DIM);
  if (a->dtype != UPLIFT_LA_F32 && a->D % 8 != 0)
    return fail(UPLIFT_LA_ERR_SHAPE, "%s: 16-bit tensors need a head dimension that is a multiple of 8 (got %d)", what, a->D);
  if (!(a->scale > 0.f) || isinf(a->scale)) return fail(UPLIFT_LA_ERR_ARG, "%s: scale must be positive and finite", what);
  if (a->B > 0 && (a->T > 0 || a->S > 0) && (a->cu_q == nullptr || a->cu_k == nullptr))
    return fail(UPLIFT_LA_ERR_ARG, "%s: null sequence starts", what);
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
Rows rows_of(const uplift_tok_rows& t, int64_t rows, int heads, int D) {
  Rows r{t.data, t.row, t.head};
  if (heads == 1) r.h = (D + 7) / 8 * 8;
  if (rows <= 1) r.t = (int64_t)r.h * heads;
  return r;
}

int prepare(const char* what, const uplift_tok_attention_args* in, bool bwd, AttnArgs* a) {
  int rc = check_sizes(what, in);
  if (rc != UPLIFT_LA_OK) return rc;
  *a = AttnArgs{};
  const struct { const char* name; const uplift_tok_rows* in; Rows* r; bool keys, used; } all[] = {
      {"q", &in->q, &a->q, false, true},        {"k", &in->k, &a->k, true, true},
      {"v", &in->v, &a->v, true, true},         {"out", &in->out, &a->out, false, true},
      {"dout", &in->dout, &a->dout, false, bwd}, {"dq", &in->dq, &a->dq, false, bwd},
      {"dk", &in->dk, &a->dk, true, bwd},       {"dv", &in->dv, &a->dv, true, bwd}};
  if (in->out_lo.data != nullptr && in->dtype != UPLIFT_LA_F32) {
    a->out_lo = rows_of(in->out_lo, in->T, in->Hq, in->D);
    if ((rc = check_rows(what, "out_lo", a->out_lo, in->T, in->Hq, in->dtype)) != UPLIFT_LA_OK) return rc;
  }
  for (const auto& e : all) {
    if (!e.used) continue;
    const int64_t rows = e.keys ? in->S : in->T;
    const int heads = e.keys ? in->Hk : in->Hq;
    *e.r = rows_of(*e.in, rows, heads, in->D);
    if ((rc = check_rows(what, e.name, *e.r, rows, heads, in->dtype)) != UPLIFT_LA_OK) return rc;
  }
  if (bwd && ((in->T > 0 && in->lse == nullptr) || (in->T + in->S > 0 && in->delta == nullptr)))
    return fail(UPLIFT_LA_ERR_ARG, "%s: null lse or delta", what);
  // the items of a pass of the gradients are counted in 32 bits
  auto items = [&](int64_t rows, int heads) { return (rows / 128 + std::min<int64_t>(rows, in->B)) * heads; };
  if (bwd && in->dtype != UPLIFT_LA_F32 && std::max(items(in->T, in->Hq), items(in->S, in->Hk)) >= (1ll << 31) - 65536)
    return fail(UPLIFT_LA_ERR_SHAPE, "%s: too many sequences: B=%d T=%lld S=%lld Hq=%d Hk=%d", what, in->B,
                (long long)in->T, (long long)in->S, in->Hq, in->Hk);
  a->lse = in->lse;
  a->delta = in->delta;
  a->pk = Packing{in->cu_q, in->cu_k, in->used_k, in->B, (int)in->T, (int)in->S, in->causal != 0};
  a->Hq = in->Hq; a->Hk = in->Hk; a->D = in->D; a->scale = in->scale; a->dtype = in->dtype;
  return UPLIFT_LA_OK;
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
  if (T < 1 || Hk < 1 || Hq < Hk || D < 1 || !attn_step_applies(B, T, Hq / Hk, dtype)) return 0;
  return attn_step_workspace(T, Hq, Hk, D);
}

int uplift_tok_attention_forward(const uplift_tok_attention_args* args, void* stream) {
  using namespace ula;
  using namespace ula::tok;
  const char* what = "uplift_tok_attention_forward";
  AttnArgs a;
  const int rc = prepare(what, args, false, &a);
  if (rc != UPLIFT_LA_OK || args->T == 0) return rc;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (a.dtype == UPLIFT_LA_F32) return attn_simt_forward(a, s);
  if (!attn_step_applies(a.pk.B, a.pk.T, a.Hq / a.Hk, a.dtype)) return attn_tc_forward(a, s);
  const int64_t need = attn_step_workspace(a.pk.T, a.Hq, a.Hk, a.D);
  if (need > 0 && (args->workspace == nullptr || args->workspace_bytes < need ||
                   (reinterpret_cast<uintptr_t>(args->workspace) & 15u) != 0))
    return fail(UPLIFT_LA_ERR_ARG, "%s: needs a 16-byte aligned workspace of %lld bytes", what, (long long)need);
  return attn_step_forward(a, args->workspace, s);
}

int uplift_tok_attention_backward(const uplift_tok_attention_args* args, void* stream) {
  using namespace ula;
  using namespace ula::tok;
  AttnArgs a;
  const int rc = prepare("uplift_tok_attention_backward", args, true, &a);
  if (rc != UPLIFT_LA_OK || (args->T == 0 && args->S == 0)) return rc;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return a.dtype == UPLIFT_LA_F32 ? attn_simt_backward(a, s) : attn_tc_backward(a, s);
}

}  // extern "C"
