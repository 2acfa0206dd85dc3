// RMS norm of query and key heads with the position rotation, and its
// gradients (C ABI in include/uplift_tokens.h).
//
//   r = 1 / sqrt(mean(x^2) + eps),  y = x r w,
//   z = R(pos) y: (a, b) -> (a c - b s, b c + a s) per channel pair.
//
// Backward, with g = R^T dz ((a, b) -> (a c + b s, b c - a s)) and h = x r:
//
//   dw = sum over rows of g h,   dx = r (g w - h mean(g w h)).
//
// Both are one pass over HBM: a row (token, head) sits in the registers of a
// group of lanes, two 8-byte pieces per lane, so the forward reads and writes
// each element once and the backward reads x and dz and writes dx.  A lane
// holds both channels of its pairs, and keeps the cos / sin row of its token
// (times the weights) over several heads.
//
// Bound by HBM.  12347 tokens of 32 + 8 heads of 128, bf16: 51 us, 5.1 TB/s (0.78
// of a copy); 42640 of 6 + 6 heads of 64, fp32: 47 us, 5.5 TB/s (0.85); the
// gradients of 8192 tokens of 32 + 8 heads of 128, bf16: 57 + 4 us, 4.4 TB/s (0.68).
// Shapes that the lanes cannot take (D or R no multiple of 16 bytes, odd
// addresses, more than 32 lanes to a row: fp32 heads above 128) run at a warp per
// row: 8192 tokens of 32 + 8 heads of 36, bf16: 131 and 365 us.

#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include <algorithm>
#include <type_traits>

#include "tok_common.h"

namespace ula {
namespace tok {
namespace nr {

constexpr int kThreads = 256;
constexpr int kManyHeads = 8, kManyHeadsBwd = 4;  // heads that a group of lanes takes, forward and backward
constexpr int kBwdBlocks = 148 * 2;  // of the backward: what the SMs hold at once
constexpr int kMaxBwdY = 64;         // of these, over the heads of one side

struct Side {  // queries or keys
  const void* x; int64_t x_t, x_h;
  const void* g; int64_t g_t, g_h;   // backward: gradient of the output
  void* out;     int64_t o_t, o_h;   // forward: the output; backward: dx
  const void* w;
  int heads, chunks;                 // chunks of heads that one group of lanes takes
  int blocks_y;                      // backward: blockIdx.y values of this side
};

struct Args {
  Side side[2];
  const float* cos;
  const float* sin;
  const void* pos;
  int pos64, wtype;
  int weight_rows;  // the weights have the tensors' type and 8-byte alignment
  int64_t T, P;
  int D, R;
  float eps, inv_d;
  float* partial;  // backward: a row of D sums per block
  int want_dw;
};

// Row of the cos / sin table for token t: >= 0, -1 = not rotated, -2 = out
// of the table.
__device__ __forceinline__ int64_t table_row(const Args& a, int64_t t) {
  if (a.pos == nullptr) return t;
  const int64_t p = a.pos64 ? static_cast<const int64_t*>(a.pos)[t] : static_cast<const int32_t*>(a.pos)[t];
  return p < 0 ? -1 : (p < a.P ? p : -2);
}

__device__ __forceinline__ float weight_at(const void* w, int wtype, int i) {
  if (w == nullptr) return 1.f;
  if (wtype == UPLIFT_LA_F32) return static_cast<const float*>(w)[i];
  if (wtype == UPLIFT_LA_BF16) return __bfloat162float(static_cast<const __nv_bfloat16*>(w)[i]);
  return __half2float(static_cast<const __half*>(w)[i]);
}

// One lane's channels of a row: V / 2 channel pairs (a, b), packed in the
// storage type as two 8-byte pieces.  Half-split: the first piece holds the
// a's, the second, R / 2 channels on, the b's; interleaved: the pieces are
// neighbours and hold a, b, a, b, ..  So a rotation stays within the lane.
template <typename T, bool INTER>
struct Row {
  static constexpr int kVec = 16 / sizeof(T);
  static constexpr int kPairs = kVec / 2;
  uint2 lo, hi;
  __device__ __forceinline__ void load(const T* p, int step) {
    lo = __ldg(reinterpret_cast<const uint2*>(p));
    hi = __ldg(reinterpret_cast<const uint2*>(p + step));
  }
  __device__ __forceinline__ void store(T* p, int step) const {
    *reinterpret_cast<uint2*>(p) = lo;
    *reinterpret_cast<uint2*>(p + step) = hi;
  }
  __device__ __forceinline__ void to(float* a, float* b) const {
    const uint32_t u[4] = {lo.x, lo.y, hi.x, hi.y};
    if constexpr (sizeof(T) == 4) {
      a[0] = __uint_as_float(u[0]);
      (INTER ? b[0] : a[1]) = __uint_as_float(u[1]);
      (INTER ? a[1] : b[0]) = __uint_as_float(u[2]);
      b[1] = __uint_as_float(u[3]);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 f = St<T>::unpack(u[i]);
        if (INTER) {
          a[i] = f.x;
          b[i] = f.y;
        } else {
          float* d = i < 2 ? a + 2 * i : b + 2 * (i - 2);
          d[0] = f.x;
          d[1] = f.y;
        }
      }
    }
  }
  __device__ __forceinline__ void from(const float* a, const float* b) {
    uint32_t u[4];
    if constexpr (sizeof(T) == 4) {
      u[0] = __float_as_uint(a[0]);
      u[1] = __float_as_uint(INTER ? b[0] : a[1]);
      u[2] = __float_as_uint(INTER ? a[1] : b[0]);
      u[3] = __float_as_uint(b[1]);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        u[i] = INTER ? St<T>::pack(a[i], b[i]) : (i < 2 ? St<T>::pack(a[2 * i], a[2 * i + 1]) : St<T>::pack(b[2 * i - 4], b[2 * i - 3]));
    }
    lo = make_uint2(u[0], u[1]);
    hi = make_uint2(u[2], u[3]);
  }
};

// Arithmetic on two fp32 values at a time: d = x y + z, x y, for N values.
template <int N>
__device__ __forceinline__ void fma_n(float* d, const float* x, const float* y, const float* z) {
#pragma unroll
  for (int i = 0; i < N; i += 2) {
    const float2 r = __ffma2_rn(make_float2(x[i], x[i + 1]), make_float2(y[i], y[i + 1]), make_float2(z[i], z[i + 1]));
    d[i] = r.x;
    d[i + 1] = r.y;
  }
}
template <int N>
__device__ __forceinline__ void mul_n(float* d, const float* x, const float* y) {
#pragma unroll
  for (int i = 0; i < N; i += 2) {
    const float2 r = __fmul2_rn(make_float2(x[i], x[i + 1]), make_float2(y[i], y[i + 1]));
    d[i] = r.x;
    d[i + 1] = r.y;
  }
}
template <int N>
__device__ __forceinline__ void scale_n(float* d, const float* x, float f) {
#pragma unroll
  for (int i = 0; i < N; i += 2) {
    const float2 r = __fmul2_rn(make_float2(x[i], x[i + 1]), make_float2(f, f));
    d[i] = r.x;
    d[i + 1] = r.y;
  }
}
// sum of x y over N values of both elements of the pairs
template <int N>
__device__ __forceinline__ float dot_n(const float* xa, const float* ya, const float* xb, const float* yb) {
  float2 s = make_float2(0.f, 0.f);
#pragma unroll
  for (int i = 0; i < N; i += 2) {
    s = __ffma2_rn(make_float2(xa[i], xa[i + 1]), make_float2(ya[i], ya[i + 1]), s);
    s = __ffma2_rn(make_float2(xb[i], xb[i + 1]), make_float2(yb[i], yb[i + 1]), s);
  }
  return s.x + s.y;
}

template <int LANES>
__device__ __forceinline__ float group_sum(float v) {
#pragma unroll
  for (int o = LANES / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// What a lane needs to know of its channels, the same for every row.
template <typename T, int LANES, bool INTER>
struct Lane {
  static constexpr int V = Row<T, INTER>::kVec, N = V / 2;
  int c0;        // first channel of the first piece
  int step;      // channels from the first piece to the second
  bool active;   // it has channels
  bool rotated;  // they are rotated
  int pair;      // its first pair of the table
  __device__ __forceinline__ Lane(const Args& a) {
    const int l = threadIdx.x & (LANES - 1);
    active = l * V < a.D;
    rotated = l * V < a.R;
    const bool split = !INTER && rotated;
    c0 = split ? l * N : l * V;
    step = split ? a.R / 2 : N;
    pair = l * N;
  }
  // The weights of its channels.
  __device__ __forceinline__ void weights(const Args& a, const void* w, float* wa, float* wb) const {
    if (a.weight_rows && w != nullptr) {  // of the tensors' type
      Row<T, INTER> r{};
      if (active) r.load(static_cast<const T*>(w) + c0, step);
      r.to(wa, wb);
      return;
    }
#pragma unroll
    for (int i = 0; i < N; ++i) {
      wa[i] = wb[i] = 0.f;
      if (active) {
        const int ca = INTER ? c0 + 2 * i : c0 + i, cb = INTER ? ca + 1 : ca + step;
        wa[i] = weight_at(w, a.wtype, ca);
        wb[i] = weight_at(w, a.wtype, cb);
      }
    }
  }
  // c and s of its pairs for a row of the table; false if they are not rotated.
  __device__ __forceinline__ bool angles(const Args& a, int64_t row, float* c, float* s) const {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      c[i] = 1.f;
      s[i] = 0.f;
    }
    if (!rotated || row == -1) return false;
    if (row == -2) {
#pragma unroll
      for (int i = 0; i < N; ++i) c[i] = s[i] = __int_as_float(0x7fc00000);
      return true;
    }
    const float2* pc = reinterpret_cast<const float2*>(a.cos + row * (a.R / 2) + pair);
    const float2* ps = reinterpret_cast<const float2*>(a.sin + row * (a.R / 2) + pair);
#pragma unroll
    for (int i = 0; i < N / 2; ++i) {
      const float2 fc = __ldg(pc + i), fs = __ldg(ps + i);
      c[2 * i] = fc.x; c[2 * i + 1] = fc.y;
      s[2 * i] = fs.x; s[2 * i + 1] = fs.y;
    }
    return true;
  }
};

// Forward.  A group of LANES lanes takes one token and HPG heads of one side
// (blockIdx.y).  All rows are loaded before the first is used, and the token's angles times
// the weights serve all of them:
//   za = r (xa (wa c) - xb (wb s)),  zb = r (xb (wb c) + xa (wa s)).
// Groups behind the last token compute on its rows and store nothing, so that
// every lane of a warp takes part in the shuffles.
template <typename T, int LANES, bool INTER, int HPG>
__global__ void __launch_bounds__(kThreads) forward_kernel(const Args a) {
  constexpr int N = Row<T, INTER>::kPairs;
  const Lane<T, LANES, INTER> ln(a);
  const int which = blockIdx.y >= a.side[0].chunks;
  const Side& sd = a.side[which];
  const int h0 = ((int)blockIdx.y - (which ? a.side[0].chunks : 0)) * HPG;
  const int64_t at = (int64_t)blockIdx.x * (kThreads / LANES) + threadIdx.x / LANES;
  const bool live = at < a.T;
  const int64_t t = min(at, a.T - 1);
  const T* x = static_cast<const T*>(sd.x) + t * sd.x_t + h0 * sd.x_h + ln.c0;
  T* out = static_cast<T*>(sd.out) + t * sd.o_t + h0 * sd.o_h + ln.c0;
  Row<T, INTER> rows[HPG] = {};
#pragma unroll
  for (int j = 0; j < HPG; ++j)
    if (ln.active && h0 + j < sd.heads) rows[j].load(x + j * sd.x_h, ln.step);
  float c[N], s[N], wa[N], wb[N];
  const bool turn = ln.angles(a, table_row(a, t), c, s);
  ln.weights(a, sd.w, wa, wb);
  float ca[N], sb[N], cb[N], sa[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    ca[i] = wa[i] * c[i];
    sb[i] = -wb[i] * s[i];
    cb[i] = wb[i] * c[i];
    sa[i] = wa[i] * s[i];
  }
#pragma unroll
  for (int j = 0; j < HPG; ++j) {
    float xa[N], xb[N];
    rows[j].to(xa, xb);
    const float sq = group_sum<LANES>(dot_n<N>(xa, xa, xb, xb));
    const float r = rsqrtf(fmaf(sq, a.inv_d, a.eps));
    if (live && ln.active && h0 + j < sd.heads) {
      float za[N], zb[N];
      mul_n<N>(za, xa, ca);
      mul_n<N>(zb, xb, cb);
      if (turn) {  // else a partner's infinity would make NaN of s = 0
        fma_n<N>(za, xb, sb, za);
        fma_n<N>(zb, xa, sa, zb);
      }
      scale_n<N>(za, za, r);
      scale_n<N>(zb, zb, r);
      Row<T, INTER> o;
      o.from(za, zb);
      o.store(out + j * sd.o_h, ln.step);
    }
  }
}

// Backward.  Blocks stride over the tokens with the heads of one chunk
// (blockIdx.y); each lane sums its channels' dw over its rows.
template <typename T, int LANES, bool INTER, int HPG>
__global__ void __launch_bounds__(kThreads, 2) backward_kernel(const Args a) {
  constexpr int V = Row<T, INTER>::kVec, N = V / 2;
  constexpr int kGroups = kThreads / LANES;
  __shared__ float red[kGroups * LANES * V];
  const Lane<T, LANES, INTER> ln(a);
  const int gi = threadIdx.x / LANES;
  const int which = blockIdx.y >= a.side[0].blocks_y;
  const Side& sd = a.side[which];
  float wa[N], wb[N], dwa[N], dwb[N];
  ln.weights(a, sd.w, wa, wb);
#pragma unroll
  for (int i = 0; i < N; ++i) dwa[i] = dwb[i] = 0.f;
  for (int ch = (int)blockIdx.y - (which ? a.side[0].blocks_y : 0); ch < sd.chunks; ch += sd.blocks_y) {
    const int h0 = ch * HPG;
    for (int64_t t0 = (int64_t)blockIdx.x * kGroups; t0 < a.T; t0 += (int64_t)gridDim.x * kGroups) {
      const bool live = t0 + gi < a.T;
      const int64_t t = min(t0 + gi, a.T - 1);
      const T* x = static_cast<const T*>(sd.x) + t * sd.x_t + h0 * sd.x_h + ln.c0;
      const T* gz = static_cast<const T*>(sd.g) + t * sd.g_t + h0 * sd.g_h + ln.c0;
      T* out = static_cast<T*>(sd.out) + t * sd.o_t + h0 * sd.o_h + ln.c0;
      Row<T, INTER> rx[HPG] = {}, rg[HPG] = {};
#pragma unroll
      for (int j = 0; j < HPG; ++j) {
        if (ln.active && h0 + j < sd.heads) {
          rx[j].load(x + j * sd.x_h, ln.step);
          rg[j].load(gz + j * sd.g_h, ln.step);
        }
      }
      float c[N], s[N], ns[N];
      const bool turn = ln.angles(a, table_row(a, t), c, s);
#pragma unroll
      for (int i = 0; i < N; ++i) ns[i] = -s[i];
#pragma unroll
      for (int j = 0; j < HPG; ++j) {
        float xa[N], xb[N], ga[N], gb[N];
        rx[j].to(xa, xb);
        rg[j].to(ga, gb);
        if (turn) {  // transpose of the rotation
          float ya[N], yb[N];
          mul_n<N>(ya, ga, c);
          mul_n<N>(yb, gb, c);
          fma_n<N>(ya, gb, s, ya);
          fma_n<N>(gb, ga, ns, yb);
#pragma unroll
          for (int i = 0; i < N; ++i) ga[i] = ya[i];
        }
        float gwa[N], gwb[N];
        mul_n<N>(gwa, ga, wa);
        mul_n<N>(gwb, gb, wb);
        const float sq = group_sum<LANES>(dot_n<N>(xa, xa, xb, xb));
        const float dot = group_sum<LANES>(dot_n<N>(xa, gwa, xb, gwb));
        const float r = rsqrtf(fmaf(sq, a.inv_d, a.eps));
        const float m = -dot * r * a.inv_d;  // -mean(g w h)
        if (live && ln.active && h0 + j < sd.heads) {
          const float mm[2] = {m, m};
          scale_n<N>(xa, xa, r);  // h
          scale_n<N>(xb, xb, r);
          fma_n<N>(dwa, ga, xa, dwa);
          fma_n<N>(dwb, gb, xb, dwb);
#pragma unroll
          for (int i = 0; i < N; i += 2) {
            fma_n<2>(gwa + i, xa + i, mm, gwa + i);
            fma_n<2>(gwb + i, xb + i, mm, gwb + i);
          }
          scale_n<N>(gwa, gwa, r);
          scale_n<N>(gwb, gwb, r);
          Row<T, INTER> o;
          o.from(gwa, gwb);
          o.store(out + j * sd.o_h, ln.step);
        }
      }
    }
  }
  if (a.want_dw) {
    // the block's groups in ascending order
    if (ln.active) {
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int ch = INTER ? ln.c0 + 2 * i : ln.c0 + i;
        red[gi * LANES * V + ch] = dwa[i];
        red[gi * LANES * V + (INTER ? ch + 1 : ch + ln.step)] = dwb[i];
      }
    }
    __syncthreads();
    for (int d = threadIdx.x; d < a.D; d += kThreads) {
      float sum = 0.f;
#pragma unroll 8
      for (int k = 0; k < kGroups; ++k) sum += red[k * LANES * V + d];
      a.partial[((int64_t)blockIdx.y * gridDim.x + blockIdx.x) * a.D + d] = sum;
    }
  }
}

// Any strides, alignment, D and R: a warp per row, a channel per lane and step.
template <typename T>
__global__ void __launch_bounds__(kThreads) forward_any_kernel(const Args a, int inter) {
  const int lane = threadIdx.x & 31;
  const int heads = a.side[0].heads + a.side[1].heads;
  const int64_t row = (int64_t)blockIdx.x * (kThreads / 32) + threadIdx.x / 32;
  if (row >= a.T * heads) return;
  const int64_t t = row / heads;
  int h = (int)(row - t * heads);
  const int which = h >= a.side[0].heads;
  const Side& sd = a.side[which];
  if (which) h -= a.side[0].heads;
  const T* x = static_cast<const T*>(sd.x) + t * sd.x_t + h * sd.x_h;
  T* out = static_cast<T*>(sd.out) + t * sd.o_t + h * sd.o_h;
  float sq = 0.f;
  for (int i = lane; i < a.D; i += 32) {
    const float v = St<T>::f(x[i]);
    sq = fmaf(v, v, sq);
  }
  sq = group_sum<32>(sq);
  const float r = rsqrtf(fmaf(sq, a.inv_d, a.eps));
  const int64_t tr = table_row(a, t);
  for (int i = lane; i < a.D; i += 32) {
    float z = St<T>::f(x[i]) * r * weight_at(sd.w, a.wtype, i);
    if (i < a.R && tr != -1) {
      const int half = a.R / 2;
      const bool second = inter ? (i & 1) : i >= half;
      const int ip = inter ? (i ^ 1) : (second ? i - half : i + half);
      const int64_t pair = inter ? i >> 1 : (second ? ip : i);
      const float yp = St<T>::f(x[ip]) * r * weight_at(sd.w, a.wtype, ip);
      if (tr == -2) z = __int_as_float(0x7fc00000);
      else z = fmaf(z, a.cos[tr * half + pair], yp * (second ? a.sin[tr * half + pair] : -a.sin[tr * half + pair]));
    }
    out[i] = St<T>::t(z);
  }
}

template <typename T>
__global__ void __launch_bounds__(kThreads) backward_any_kernel(const Args a, int inter) {
  constexpr int kWarps = kThreads / 32;
  constexpr int kPer = UPLIFT_TOK_MAX_NORM_DIM / 32;
  __shared__ float red[kWarps * UPLIFT_TOK_MAX_NORM_DIM];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int half = a.R / 2;
  const Side& sd = a.side[blockIdx.y];
  float dw[kPer];
#pragma unroll
  for (int j = 0; j < kPer; ++j) dw[j] = 0.f;
  const int64_t rows = a.T * sd.heads;
  for (int64_t row = (int64_t)blockIdx.x * kWarps + warp; row < rows; row += (int64_t)gridDim.x * kWarps) {
    const int64_t t = row / sd.heads;
    const int h = (int)(row - t * sd.heads);
    const T* x = static_cast<const T*>(sd.x) + t * sd.x_t + h * sd.x_h;
    const T* gz = static_cast<const T*>(sd.g) + t * sd.g_t + h * sd.g_h;
    T* out = static_cast<T*>(sd.out) + t * sd.o_t + h * sd.o_h;
    const int64_t tr = table_row(a, t);
    float gy[kPer], v[kPer], w[kPer];
    float sq = 0.f, dot = 0.f;
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      const int i = lane + 32 * j;
      gy[j] = v[j] = w[j] = 0.f;
      if (i < a.D) {
        v[j] = St<T>::f(x[i]);
        w[j] = weight_at(sd.w, a.wtype, i);
        float g = St<T>::f(gz[i]);
        if (i < a.R && tr != -1) {
          const bool second = inter ? (i & 1) : i >= half;
          const int ip = inter ? (i ^ 1) : (second ? i - half : i + half);
          const int64_t pair = inter ? i >> 1 : (second ? ip : i);
          const float gp = St<T>::f(gz[ip]);
          if (tr == -2) g = __int_as_float(0x7fc00000);
          else g = fmaf(g, a.cos[tr * half + pair], gp * (second ? -a.sin[tr * half + pair] : a.sin[tr * half + pair]));
        }
        gy[j] = g;
      }
      sq = fmaf(v[j], v[j], sq);
      dot = fmaf(gy[j] * w[j], v[j], dot);
    }
    sq = group_sum<32>(sq);
    dot = group_sum<32>(dot);
    const float r = rsqrtf(fmaf(sq, a.inv_d, a.eps));
    const float m = dot * r * a.inv_d;
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      const int i = lane + 32 * j;
      if (i < a.D) {
        const float hh = v[j] * r;
        out[i] = St<T>::t(r * fmaf(-hh, m, gy[j] * w[j]));
        dw[j] = fmaf(gy[j], hh, dw[j]);
      }
    }
  }
  if (a.want_dw) {
#pragma unroll
    for (int j = 0; j < kPer; ++j) red[warp * UPLIFT_TOK_MAX_NORM_DIM + lane + 32 * j] = dw[j];
    __syncthreads();
    for (int d = threadIdx.x; d < a.D; d += kThreads) {
      float sum = 0.f;
      for (int k = 0; k < kWarps; ++k) sum += red[k * UPLIFT_TOK_MAX_NORM_DIM + d];
      a.partial[((int64_t)blockIdx.y * gridDim.x + blockIdx.x) * a.D + d] = sum;
    }
  }
}

// dweights[which][d] = sum of the side's rows of partials (rows0 of the
// queries, then rows1 of the keys), in a fixed order (32 channels a block, a
// warp every 32nd row) and in 64 bits: the sum runs over all rows of the
// problem.
__global__ void __launch_bounds__(1024) dweights_kernel(const float* partial, void* dweights, int wtype, int rows0, int rows1, int D) {
  __shared__ double red[32][33];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int which = blockIdx.y, d = blockIdx.x * 32 + lane;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  double sum = 0.0;
  if (d < D) {
#pragma unroll 8
    for (int b = warp; b < (which ? rows1 : rows0); b += 32) sum += (double)partial[((int64_t)(which ? rows0 : 0) + b) * D + d];
  }
  red[warp][lane] = sum;
  __syncthreads();
  sum = red[lane][warp];  // channel `warp` of the block, partial sum `lane`
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  const int out = blockIdx.x * 32 + warp;
  if (lane == 0 && out < D) {
    const int64_t at = (int64_t)which * D + out;
    if (wtype == UPLIFT_LA_F32) static_cast<float*>(dweights)[at] = (float)sum;
    else if (wtype == UPLIFT_LA_BF16) static_cast<__nv_bfloat16*>(dweights)[at] = __double2bfloat16(sum);
    else static_cast<__half*>(dweights)[at] = __double2half(sum);
  }
}

template <typename T, int LANES, int HPG>
void launch_vec(const Args& a, bool inter, bool bwd, dim3 blocks, cudaStream_t s) {
  if (bwd) {
    if (inter) backward_kernel<T, LANES, true, HPG><<<blocks, kThreads, 0, s>>>(a);
    else backward_kernel<T, LANES, false, HPG><<<blocks, kThreads, 0, s>>>(a);
  } else {
    if (inter) forward_kernel<T, LANES, true, HPG><<<blocks, kThreads, 0, s>>>(a);
    else forward_kernel<T, LANES, false, HPG><<<blocks, kThreads, 0, s>>>(a);
  }
}

template <typename T, int HPG>
void launch_lanes(const Args& a, int lanes, bool inter, bool bwd, dim3 blocks, cudaStream_t s) {
  switch (lanes) {
    case 4: launch_vec<T, 4, HPG>(a, inter, bwd, blocks, s); break;
    case 8: launch_vec<T, 8, HPG>(a, inter, bwd, blocks, s); break;
    case 16: launch_vec<T, 16, HPG>(a, inter, bwd, blocks, s); break;
    default: launch_vec<T, 32, HPG>(a, inter, bwd, blocks, s); break;
  }
}

// Launches; *rows: rows of partials that the backward writes for each side.
template <typename T>
int run(Args a, int dtype, bool inter, bool bwd, int* partial_rows, cudaStream_t s) {
  constexpr int V = 16 / sizeof(T);  // channels of a lane, in two pieces of 8 bytes
  auto al = [](const void* p) { return (reinterpret_cast<uintptr_t>(p) & 7u) == 0; };
  bool vec = a.D % V == 0 && a.D / V <= 32 && a.R % V == 0 && (a.R == 0 || (al(a.cos) && al(a.sin)));
  for (int i = 0; i < 2; ++i) {
    const Side& d = a.side[i];
    vec = vec && al(d.x) && al(d.out) && d.x_t % (V / 2) == 0 && d.x_h % (V / 2) == 0 && d.o_t % (V / 2) == 0 && d.o_h % (V / 2) == 0;
    if (bwd) vec = vec && al(d.g) && d.g_t % (V / 2) == 0 && d.g_h % (V / 2) == 0;
  }
  a.weight_rows = a.wtype == dtype && al(a.side[0].w) && al(a.side[1].w);
  const int64_t rows = a.T * (a.side[0].heads + a.side[1].heads);
  int lanes = 4;
  while (lanes * V < a.D) lanes *= 2;
  // Heads per group: several amortise the token's angles and the weights and
  // keep more loads in flight; one where several would leave SMs without work.
  // 32 + 8 heads of 128 in bf16, forward and backward, several / one (us): 128
  // tokens 3.2 / 2.5 and 3.7 / 4.1, 512: 4.8 / 4.9 and 6.7 / 7.2, 1024: 6.3 / 8.1
  // and 9.1 / 11.4, 8192: 28 / 50 and 54 / 89.  One threshold serves both, though
  // the backward would gain its 0.4 us below it too.
  const int hpg = vec && rows * lanes >= 148ll * 2048 ? (bwd ? kManyHeadsBwd : kManyHeads) : 1;
  for (int i = 0; i < 2; ++i) a.side[i].chunks = (a.side[i].heads + hpg - 1) / hpg;
  if (bwd) {
    // vec: tokens over x, chunks of heads over y; else rows over x, sides over y
    const int per_block = vec ? kThreads / lanes : kThreads / 32;
    for (int i = 0; i < 2; ++i) a.side[i].blocks_y = vec ? std::min(a.side[i].chunks, kMaxBwdY) : 1;
    const int y = a.side[0].blocks_y + a.side[1].blocks_y;
    const int64_t x = vec ? (a.T + per_block - 1) / per_block : (rows + per_block - 1) / per_block;
    const dim3 blocks((unsigned)std::min<int64_t>(x, std::max(1, kBwdBlocks / y)), y);
    for (int i = 0; i < 2; ++i) partial_rows[i] = (int)blocks.x * a.side[i].blocks_y;
    if (vec && hpg > 1) launch_lanes<T, kManyHeadsBwd>(a, lanes, inter, true, blocks, s);
    else if (vec) launch_lanes<T, 1>(a, lanes, inter, true, blocks, s);
    else backward_any_kernel<T><<<blocks, kThreads, 0, s>>>(a, inter);
    return UPLIFT_LA_OK;
  }
  const int64_t x = vec ? (a.T * lanes + kThreads - 1) / kThreads : (rows + kThreads / 32 - 1) / (kThreads / 32);
  if (x >= (1ll << 31)) return fail(UPLIFT_LA_ERR_SHAPE, "norm_rotate: too many rows");
  const dim3 blocks((unsigned)x, vec ? a.side[0].chunks + a.side[1].chunks : 1);
  if (vec && hpg > 1) launch_lanes<T, kManyHeads>(a, lanes, inter, false, blocks, s);
  else if (vec) launch_lanes<T, 1>(a, lanes, inter, false, blocks, s);
  else forward_any_kernel<T><<<blocks, kThreads, 0, s>>>(a, inter);
  return UPLIFT_LA_OK;
}

// Validates the arguments and fills `a`.
int prepare(const char* what, const uplift_tok_norm_rotate_args* in, bool bwd, Args* a) {
  if (in == nullptr || in->size != (int64_t)sizeof(*in)) return fail(UPLIFT_LA_ERR_ARG, "%s: no arguments, or of another version", what);
  const int dt = in->dtype, wt = in->weight_dtype;
  if (dt != UPLIFT_LA_F32 && dt != UPLIFT_LA_BF16 && dt != UPLIFT_LA_F16)
    return fail(UPLIFT_LA_ERR_ARG, "%s: unknown dtype %d", what, dt);
  if (wt != UPLIFT_LA_F32 && wt != UPLIFT_LA_BF16 && wt != UPLIFT_LA_F16)
    return fail(UPLIFT_LA_ERR_ARG, "%s: unknown weight dtype %d", what, wt);
  if (in->T < 0 || in->T >= (1ll << 31) || in->P < 0 || in->Hq < 1 || in->Hk < 1 || in->Hq > 32767 || in->Hk > 32767)
    return fail(UPLIFT_LA_ERR_SHAPE, "%s: bad sizes T=%lld P=%lld Hq=%d Hk=%d", what, (long long)in->T,
                (long long)in->P, in->Hq, in->Hk);
  if (in->D < 1 || in->D > UPLIFT_TOK_MAX_NORM_DIM)
    return fail(UPLIFT_LA_ERR_SHAPE, "%s: head dimension %d not in 1..%d", what, in->D, UPLIFT_TOK_MAX_NORM_DIM);
  if (in->R < 0 || in->R > in->D || in->R % 2 != 0)
    return fail(UPLIFT_LA_ERR_SHAPE, "%s: %d rotated channels (even, at most D = %d)", what, in->R, in->D);
  if (!(in->eps >= 0.f) || isinf(in->eps)) return fail(UPLIFT_LA_ERR_ARG, "%s: eps must be finite and not negative", what);
  if (in->positions == nullptr && in->R > 0 && in->P < in->T)
    return fail(UPLIFT_LA_ERR_SHAPE, "%s: %lld table rows for %lld tokens without positions", what, (long long)in->P,
                (long long)in->T);
  if (bwd && in->dweights != nullptr && in->partial == nullptr)
    return fail(UPLIFT_LA_ERR_ARG, "%s: weight gradients need the workspace", what);
  if (in->T > 0 && (in->q.data == nullptr || in->k.data == nullptr || in->q_out.data == nullptr ||
                    in->k_out.data == nullptr || (bwd && (in->dq.data == nullptr || in->dk.data == nullptr)) ||
                    (in->R > 0 && in->P > 0 && (in->cos == nullptr || in->sin == nullptr))))
    return fail(UPLIFT_LA_ERR_ARG, "%s: null pointer", what);
  *a = Args{};
  const uplift_tok_rows* x[2] = {&in->q, &in->k};
  const uplift_tok_rows* z[2] = {&in->q_out, &in->k_out};
  const uplift_tok_rows* d[2] = {&in->dq, &in->dk};
  for (int i = 0; i < 2; ++i) {
    Side& sd = a->side[i];
    sd.x = x[i]->data; sd.x_t = x[i]->row; sd.x_h = x[i]->head;
    const uplift_tok_rows* o = bwd ? d[i] : z[i];
    sd.out = o->data; sd.o_t = o->row; sd.o_h = o->head;
    if (bwd) { sd.g = z[i]->data; sd.g_t = z[i]->row; sd.g_h = z[i]->head; }
    sd.w = i == 0 ? in->q_weight : in->k_weight;
    sd.heads = i == 0 ? in->Hq : in->Hk;
  }
  a->cos = in->cos; a->sin = in->sin; a->pos = in->positions; a->pos64 = in->positions64; a->wtype = wt;
  a->T = in->T; a->P = in->P; a->D = in->D; a->R = in->R; a->eps = in->eps; a->inv_d = 1.f / (float)in->D;
  a->partial = in->partial;
  a->want_dw = bwd && in->dweights != nullptr;
  return UPLIFT_LA_OK;
}

int run_dtype(const Args& a, int dtype, bool inter, bool bwd, int* partial_rows, cudaStream_t s) {
  if (dtype == UPLIFT_LA_F32) return run<float>(a, dtype, inter, bwd, partial_rows, s);
  if (dtype == UPLIFT_LA_BF16) return run<__nv_bfloat16>(a, dtype, inter, bwd, partial_rows, s);
  return run<__half>(a, dtype, inter, bwd, partial_rows, s);
}

}  // namespace nr
}  // namespace tok
}  // namespace ula

extern "C" {

int uplift_tok_norm_rotate(const uplift_tok_norm_rotate_args* args, void* stream) {
  using namespace ula;
  using namespace ula::tok::nr;
  Args a;
  int rc = prepare("uplift_tok_norm_rotate", args, false, &a);
  if (rc != UPLIFT_LA_OK || args->T == 0) return rc;
  rc = run_dtype(a, args->dtype, args->interleaved != 0, false, nullptr, static_cast<cudaStream_t>(stream));
  return rc != UPLIFT_LA_OK ? rc : tok::launched("norm_rotate");
}

int64_t uplift_tok_norm_rotate_partial_floats(int D) {
  return D < 1 ? 0 : (int64_t)ula::tok::nr::kBwdBlocks * D;
}

int uplift_tok_norm_rotate_backward(const uplift_tok_norm_rotate_args* args, void* stream) {
  using namespace ula;
  using namespace ula::tok::nr;
  Args a;
  int rc = prepare("uplift_tok_norm_rotate_backward", args, true, &a);
  if (rc != UPLIFT_LA_OK) return rc;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  int partial_rows[2] = {0, 0};
  if (args->T > 0) {
    rc = run_dtype(a, args->dtype, args->interleaved != 0, true, partial_rows, s);
    if (rc != UPLIFT_LA_OK) return rc;
    if ((rc = tok::launched("norm_rotate backward")) != UPLIFT_LA_OK) return rc;
  }
  if (args->dweights != nullptr) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)((args->D + 31) / 32), 2);
    cfg.blockDim = dim3(1024);
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, dweights_kernel, (const float*)args->partial, args->dweights,
                                             (int)args->weight_dtype, partial_rows[0], partial_rows[1], (int)args->D);
    if (e != cudaSuccess) return fail(UPLIFT_LA_ERR_CUDA, "norm_rotate weight gradients launch: %s", cudaGetErrorString(e));
    return tok::launched("norm_rotate weight gradients");
  }
  return UPLIFT_LA_OK;
}

}  // extern "C"
