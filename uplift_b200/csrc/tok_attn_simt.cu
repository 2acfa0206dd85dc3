// Attention over packed sequences on CUDA cores, forward and backward: any
// storage type, D <= 128.  A warp owns one row (query, head) -- in the
// backward's second pass one key row of one key head -- and takes the other
// side 32 rows at a time: lane j forms the products with row j, then the
// warp adds the 32 weighted rows, a lane owning channels lane, lane + 32, ..

#include <math.h>

#include <algorithm>

#include "tok_attn.h"

namespace ula {
namespace tok {
namespace simt {

constexpr int kWarps = 4;
constexpr int kCh = UPLIFT_TOK_MAX_ATTN_DIM / 32;

// Sequence of row t: the last one that starts at or before it.
__device__ __forceinline__ int sequence_of(const int32_t* cu, int B, int t) {
  int lo = 0, hi = B;  // cu[lo] <= t < cu[hi], as far as such bounds exist
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (__ldg(cu + mid) <= t) lo = mid;
    else hi = mid;
  }
  return lo;
}

template <typename T>
__device__ __forceinline__ const T* row_of(const Rows& r, int64_t t, int h) {
  return static_cast<const T*>(r.p) + t * r.t + h * r.h;
}
template <typename T>
__device__ __forceinline__ T* out_row(const Rows& r, int64_t t, int h) {
  return static_cast<T*>(const_cast<void*>(r.p)) + t * r.t + h * r.h;
}

__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}
__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

template <typename T>
__device__ __forceinline__ float dot(const float* a, const T* b, int D) {
  float s = 0.f;
#pragma unroll 8
  for (int c = 0; c < D; ++c) s = fmaf(a[c], St<T>::f(b[c]), s);
  return s;
}

template <typename T>
__global__ void __launch_bounds__(kWarps * 32) forward_kernel(const AttnArgs a) {
  __shared__ float sq[kWarps][UPLIFT_TOK_MAX_ATTN_DIM];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t item = (int64_t)blockIdx.x * kWarps + warp;
  if (item >= (int64_t)a.pk.T * a.Hq) return;
  const int t = (int)(item / a.Hq), h = (int)(item % a.Hq), hk = h / (a.Hq / a.Hk);
  int n = 0;
  Seq s{};
  if (a.pk.B > 0) {
    s = sequence(a.pk, sequence_of(a.pk.cu_q, a.pk.B, t));
    if (t >= s.q0 && t < s.q0 + s.nq) n = keys_seen(s, t - s.q0, a.pk.causal);
  }
  const T* q = row_of<T>(a.q, t, h);
  for (int c = lane; c < a.D; c += 32) sq[warp][c] = St<T>::f(q[c]) * a.scale;
  __syncwarp();
  float m = -INFINITY, l = 0.f, acc[kCh];
#pragma unroll
  for (int i = 0; i < kCh; ++i) acc[i] = 0.f;
  for (int j0 = 0; j0 < n; j0 += 32) {
    const int j = j0 + lane;
    float x = -INFINITY;
    if (j < n) x = dot<T>(sq[warp], row_of<T>(a.k, s.k0 + j, hk), a.D);
    const float mn = fmaxf(m, warp_max(x));
    const float ms = mn == -INFINITY ? 0.f : mn;
    const float f = expf(m - ms);
    const float p = j < n ? expf(x - ms) : 0.f;
    l = l * f + warp_sum(p);
    m = mn;
#pragma unroll
    for (int i = 0; i < kCh; ++i) acc[i] *= f;
    const int cnt = min(32, n - j0);
    for (int jj = 0; jj < cnt; ++jj) {
      const float pj = __shfl_sync(0xffffffffu, p, jj);
      const T* v = row_of<T>(a.v, s.k0 + j0 + jj, hk);
#pragma unroll
      for (int i = 0; i < kCh; ++i)
        if (lane + 32 * i < a.D) acc[i] = fmaf(pj, St<T>::f(v[lane + 32 * i]), acc[i]);
    }
  }
  const bool none = l == 0.f;  // no key seen, or all scores -inf
  T* o = out_row<T>(a.out, t, h);
#pragma unroll
  for (int i = 0; i < kCh; ++i)
    if (lane + 32 * i < a.D) o[lane + 32 * i] = St<T>::t(none ? 0.f : acc[i] / l);
  if (a.lse != nullptr && lane == 0) a.lse[(int64_t)h * a.pk.T + t] = none ? -INFINITY : m + logf(l);
}

// delta_i = dO_i . O_i
template <typename T>
__global__ void __launch_bounds__(kWarps * 32) delta_kernel(const AttnArgs a) {
  const int lane = threadIdx.x & 31;
  const int64_t item = (int64_t)blockIdx.x * kWarps + (threadIdx.x >> 5);
  if (item >= (int64_t)a.pk.T * a.Hq) return;
  const int t = (int)(item / a.Hq), h = (int)(item % a.Hq);
  const T* o = row_of<T>(a.out, t, h);
  const T* g = row_of<T>(a.dout, t, h);
  float s = 0.f;
  for (int c = lane; c < a.D; c += 32) s = fmaf(St<T>::f(o[c]), St<T>::f(g[c]), s);
  s = warp_sum(s);
  if (lane == 0) a.delta[(int64_t)h * a.pk.T + t] = s;
}

// dQ_i = sum_j dS_ij K_j
template <typename T>
__global__ void __launch_bounds__(kWarps * 32) dq_kernel(const AttnArgs a) {
  __shared__ float sq[kWarps][UPLIFT_TOK_MAX_ATTN_DIM], sg[kWarps][UPLIFT_TOK_MAX_ATTN_DIM];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t item = (int64_t)blockIdx.x * kWarps + warp;
  if (item >= (int64_t)a.pk.T * a.Hq) return;
  const int t = (int)(item / a.Hq), h = (int)(item % a.Hq), hk = h / (a.Hq / a.Hk);
  int n = 0;
  Seq s{};
  if (a.pk.B > 0) {
    s = sequence(a.pk, sequence_of(a.pk.cu_q, a.pk.B, t));
    if (t >= s.q0 && t < s.q0 + s.nq) n = keys_seen(s, t - s.q0, a.pk.causal);
  }
  const T* q = row_of<T>(a.q, t, h);
  const T* g = row_of<T>(a.dout, t, h);
  for (int c = lane; c < a.D; c += 32) {
    sq[warp][c] = St<T>::f(q[c]) * a.scale;
    sg[warp][c] = St<T>::f(g[c]);
  }
  __syncwarp();
  const float lse = a.lse[(int64_t)h * a.pk.T + t], delta = a.delta[(int64_t)h * a.pk.T + t];
  float acc[kCh];
#pragma unroll
  for (int i = 0; i < kCh; ++i) acc[i] = 0.f;
  if (lse == -INFINITY) n = 0;
  for (int j0 = 0; j0 < n; j0 += 32) {
    const int j = j0 + lane;
    float ds = 0.f;
    if (j < n) {
      const float p = expf(dot<T>(sq[warp], row_of<T>(a.k, s.k0 + j, hk), a.D) - lse);
      ds = p * (dot<T>(sg[warp], row_of<T>(a.v, s.k0 + j, hk), a.D) - delta) * a.scale;
    }
    const int cnt = min(32, n - j0);
    for (int jj = 0; jj < cnt; ++jj) {
      const float x = __shfl_sync(0xffffffffu, ds, jj);
      const T* k = row_of<T>(a.k, s.k0 + j0 + jj, hk);
#pragma unroll
      for (int i = 0; i < kCh; ++i)
        if (lane + 32 * i < a.D) acc[i] = fmaf(x, St<T>::f(k[lane + 32 * i]), acc[i]);
    }
  }
  T* o = out_row<T>(a.dq, t, h);
#pragma unroll
  for (int i = 0; i < kCh; ++i)
    if (lane + 32 * i < a.D) o[lane + 32 * i] = St<T>::t(acc[i]);
}

// dV_j = sum_i P_ij dO_i, dK_j = sum_i dS_ij Q_i over the heads of the group
// and the queries that see key j.
template <typename T>
__global__ void __launch_bounds__(kWarps * 32) dkv_kernel(const AttnArgs a) {
  __shared__ float sk[kWarps][UPLIFT_TOK_MAX_ATTN_DIM], sv[kWarps][UPLIFT_TOK_MAX_ATTN_DIM];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t item = (int64_t)blockIdx.x * kWarps + warp;
  if (item >= (int64_t)a.pk.S * a.Hk) return;
  const int t = (int)(item / a.Hk), hk = (int)(item % a.Hk), group = a.Hq / a.Hk;
  Seq s{};
  int i0 = 0;  // first query that sees the key
  bool seen = false;
  if (a.pk.B > 0) {
    s = sequence(a.pk, sequence_of(a.pk.cu_k, a.pk.B, t));
    const int j = t - s.k0;
    seen = j >= 0 && j < s.nk;
    i0 = a.pk.causal ? max(0, j - s.nk + s.nq) : 0;
  }
  const T* k = row_of<T>(a.k, t, hk);
  const T* v = row_of<T>(a.v, t, hk);
  for (int c = lane; c < a.D; c += 32) {
    sk[warp][c] = St<T>::f(k[c]) * a.scale;
    sv[warp][c] = St<T>::f(v[c]);
  }
  __syncwarp();
  float dk[kCh], dv[kCh];
#pragma unroll
  for (int i = 0; i < kCh; ++i) dk[i] = dv[i] = 0.f;
  if (seen) {
    for (int h = hk * group; h < (hk + 1) * group; ++h) {
      for (int b0 = i0; b0 < s.nq; b0 += 32) {
        const int i = b0 + lane;
        float p = 0.f, ds = 0.f;
        if (i < s.nq) {
          const int64_t at = (int64_t)h * a.pk.T + s.q0 + i;
          const float lse = a.lse[at];
          if (lse != -INFINITY) {
            p = expf(dot<T>(sk[warp], row_of<T>(a.q, s.q0 + i, h), a.D) - lse);
            ds = p * (dot<T>(sv[warp], row_of<T>(a.dout, s.q0 + i, h), a.D) - a.delta[at]) * a.scale;
          }
        }
        const int cnt = min(32, s.nq - b0);
        for (int ii = 0; ii < cnt; ++ii) {
          const float pi = __shfl_sync(0xffffffffu, p, ii), di = __shfl_sync(0xffffffffu, ds, ii);
          const T* q = row_of<T>(a.q, s.q0 + b0 + ii, h);
          const T* g = row_of<T>(a.dout, s.q0 + b0 + ii, h);
#pragma unroll
          for (int c = 0; c < kCh; ++c) {
            if (lane + 32 * c < a.D) {
              dv[c] = fmaf(pi, St<T>::f(g[lane + 32 * c]), dv[c]);
              dk[c] = fmaf(di, St<T>::f(q[lane + 32 * c]), dk[c]);
            }
          }
        }
      }
    }
  }
  T* ok = out_row<T>(a.dk, t, hk);
  T* ov = out_row<T>(a.dv, t, hk);
#pragma unroll
  for (int c = 0; c < kCh; ++c) {
    if (lane + 32 * c < a.D) {
      ok[lane + 32 * c] = St<T>::t(dk[c]);
      ov[lane + 32 * c] = St<T>::t(dv[c]);
    }
  }
}

int blocks_for(int64_t items, int* blocks) {
  const int64_t n = (items + kWarps - 1) / kWarps;
  if (n >= (1ll << 31)) return fail(UPLIFT_LA_ERR_SHAPE, "attention: too many rows");
  *blocks = (int)n;
  return UPLIFT_LA_OK;
}

template <typename T>
int forward(const AttnArgs& a, cudaStream_t s) {
  int blocks = 0;
  const int rc = blocks_for((int64_t)a.pk.T * a.Hq, &blocks);
  if (rc != UPLIFT_LA_OK || blocks == 0) return rc;
  forward_kernel<T><<<blocks, kWarps * 32, 0, s>>>(a);
  return launched("attention");
}

template <typename T>
int backward(const AttnArgs& a, cudaStream_t s) {
  int bq = 0, bk = 0;
  int rc = blocks_for((int64_t)a.pk.T * a.Hq, &bq);
  if (rc == UPLIFT_LA_OK) rc = blocks_for((int64_t)a.pk.S * a.Hk, &bk);
  if (rc != UPLIFT_LA_OK) return rc;
  if (bq > 0) {
    delta_kernel<T><<<bq, kWarps * 32, 0, s>>>(a);
    dq_kernel<T><<<bq, kWarps * 32, 0, s>>>(a);
  }
  if (bk > 0) dkv_kernel<T><<<bk, kWarps * 32, 0, s>>>(a);
  return launched("attention backward");
}

}  // namespace simt

int attn_simt_forward(const AttnArgs& a, cudaStream_t s) { return simt::forward<float>(a, s); }
int attn_simt_backward(const AttnArgs& a, cudaStream_t s) { return simt::backward<float>(a, s); }

}  // namespace tok
}  // namespace ula
