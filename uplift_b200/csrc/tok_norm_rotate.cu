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
// group of lanes, one 16-byte vector per lane, so the forward reads and
// writes each element once and the backward reads x and dz and writes dx.
// The partner channels of a half-split pair are in another lane of the group
// and come by shuffle, still packed in the storage type.  A group keeps the
// cos / sin row of its token over several heads.

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
constexpr int kBwdBlocks = 148 * 4;  // fixed, so the order of the dw sums does not depend on the problem's size

struct Side {  // queries or keys
  const void* x; int64_t x_t, x_h;
  const void* g; int64_t g_t, g_h;   // backward: gradient of the output
  void* out;     int64_t o_t, o_h;   // forward: the output; backward: dx
  const void* w;
  int heads, chunks;                 // chunks of `hpg` heads
};

struct Args {
  Side side[2];
  const float* cos;
  const float* sin;
  const void* pos;
  int pos64, wtype;
  int64_t T, P;
  int D, R, hpg;  // hpg: heads per group of lanes
  float eps, inv_d;
  float* partial;  // backward: [2][kBwdBlocks][D]
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

template <typename T>
struct Row {  // one lane's 16 bytes of a row
  static constexpr int kVec = 16 / sizeof(T);
  uint4 raw;
  __device__ __forceinline__ void load(const T* p) { raw = __ldg(reinterpret_cast<const uint4*>(p)); }
  __device__ __forceinline__ void store(T* p) const { *reinterpret_cast<uint4*>(p) = raw; }
  __device__ __forceinline__ void to(float* v) const {
    const uint32_t u[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (sizeof(T) == 4) {
        v[i] = __uint_as_float(u[i]);
      } else {
        const float2 f = St<T>::unpack(u[i]);
        v[2 * i] = f.x;
        v[2 * i + 1] = f.y;
      }
    }
  }
  __device__ __forceinline__ void from(const float* v) {
    uint32_t u[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (sizeof(T) == 4) u[i] = __float_as_uint(v[i]);
      else u[i] = St<T>::pack(v[2 * i], v[2 * i + 1]);
    }
    raw = make_uint4(u[0], u[1], u[2], u[3]);
  }
  __device__ __forceinline__ Row shuffled(int src) const {
    Row r;
    r.raw.x = __shfl_sync(0xffffffffu, raw.x, src);
    r.raw.y = __shfl_sync(0xffffffffu, raw.y, src);
    r.raw.z = __shfl_sync(0xffffffffu, raw.z, src);
    r.raw.w = __shfl_sync(0xffffffffu, raw.w, src);
    return r;
  }
};

template <int LANES>
__device__ __forceinline__ float group_sum(float v) {
#pragma unroll
  for (int o = LANES / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// What a lane needs to know of its channels, the same for every row.
template <typename T, int LANES, bool INTER>
struct Lane {
  static constexpr int V = Row<T>::kVec;
  int c0;        // first channel
  bool active;   // it has channels
  bool rotated;  // they are rotated
  bool upper;    // half-split: they are second elements of their pairs
  int partner;   // half-split: lane of the warp that holds the partners
  __device__ __forceinline__ Lane(const Args& a) {
    const int lane = threadIdx.x & 31, l = lane & (LANES - 1);
    c0 = l * V;
    active = c0 < a.D;
    rotated = c0 < a.R;
    upper = !INTER && c0 >= a.R / 2;
    const int shift = (a.R / 2) / V;
    partner = INTER || !rotated ? lane : (upper ? lane - shift : lane + shift);
  }
  // c and s of the lane's channels (s with the sign of the channel's place
  // in its pair: z = y c + y_partner s); false if they are not rotated.
  __device__ __forceinline__ bool angles(const Args& a, int64_t row, float* c, float* s) const {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      c[i] = 1.f;
      s[i] = 0.f;
    }
    if (!rotated || row == -1) return false;
    if (row == -2) {
#pragma unroll
      for (int i = 0; i < V; ++i) c[i] = s[i] = __int_as_float(0x7fc00000);
      return true;
    }
    if constexpr (INTER) {
      const float* pc = a.cos + row * (a.R / 2) + c0 / 2;
      const float* ps = a.sin + row * (a.R / 2) + c0 / 2;
#pragma unroll
      for (int i = 0; i < V / 2; ++i) {
        c[2 * i] = c[2 * i + 1] = __ldg(pc + i);
        s[2 * i + 1] = __ldg(ps + i);
        s[2 * i] = -s[2 * i + 1];
      }
    } else {
      const int i0 = upper ? c0 - a.R / 2 : c0;
      const float4* pc = reinterpret_cast<const float4*>(a.cos + row * (a.R / 2) + i0);
      const float4* ps = reinterpret_cast<const float4*>(a.sin + row * (a.R / 2) + i0);
#pragma unroll
      for (int i = 0; i < V / 4; ++i) {
        const float4 fc = __ldg(pc + i), fs = __ldg(ps + i);
        c[4 * i] = fc.x; c[4 * i + 1] = fc.y; c[4 * i + 2] = fc.z; c[4 * i + 3] = fc.w;
        s[4 * i] = fs.x; s[4 * i + 1] = fs.y; s[4 * i + 2] = fs.z; s[4 * i + 3] = fs.w;
      }
      if (!upper) {
#pragma unroll
        for (int i = 0; i < V; ++i) s[i] = -s[i];
      }
    }
    return true;
  }
};

// Forward.  Group g of LANES lanes: token g / chunks, heads of one chunk.
// Out-of-range groups compute on the last group's rows and store nothing, so
// that every lane of a warp takes part in the shuffles.
template <typename T, int LANES, bool INTER>
__global__ void __launch_bounds__(kThreads) forward_kernel(const Args a) {
  constexpr int V = Row<T>::kVec;
  const Lane<T, LANES, INTER> ln(a);
  const int chunks = a.side[0].chunks + a.side[1].chunks;
  const int64_t groups = a.T * chunks;
  int64_t g = (int64_t)blockIdx.x * (kThreads / LANES) + threadIdx.x / LANES;
  const bool live = g < groups;
  g = min(g, groups - 1);
  const int64_t t = g / chunks;
  int ch = (int)(g - t * chunks);
  const int which = ch >= a.side[0].chunks;
  const Side& sd = a.side[which];
  if (which) ch -= a.side[0].chunks;
  const int h0 = ch * a.hpg;
  const T* x = static_cast<const T*>(sd.x) + t * sd.x_t + ln.c0;
  T* out = static_cast<T*>(sd.out) + t * sd.o_t + ln.c0;
  float c[V], s[V], w[V], wp[V];
  const bool turn = ln.angles(a, table_row(a, t), c, s);
#pragma unroll
  for (int i = 0; i < V; ++i) {
    w[i] = wp[i] = 0.f;
    if (ln.active) {
      w[i] = weight_at(sd.w, a.wtype, ln.c0 + i);
      if (!INTER && ln.rotated) wp[i] = weight_at(sd.w, a.wtype, ln.upper ? ln.c0 + i - a.R / 2 : ln.c0 + i + a.R / 2);
    }
  }
  // the loop count is that of the kernel, not of the chunk: uniform over the warp
  Row<T> next{};
  if (ln.active) next.load(x + min(h0, sd.heads - 1) * sd.x_h);
  for (int j = 0; j < a.hpg; ++j) {
    const int h = h0 + j;
    const Row<T> cur = next;
    if (ln.active && j + 1 < a.hpg) next.load(x + min(h + 1, sd.heads - 1) * sd.x_h);
    float v[V];
    cur.to(v);
    float sq = 0.f;
#pragma unroll
    for (int i = 0; i < V; ++i) sq = fmaf(v[i], v[i], sq);
    sq = group_sum<LANES>(sq);
    const float r = 1.f / sqrtf(fmaf(sq, a.inv_d, a.eps));
    float z[V];
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = v[i] * r * w[i];
    if constexpr (INTER) {
#pragma unroll
      for (int i = 0; i < V; ++i) z[i] = fmaf(v[i], c[i], v[i ^ 1] * s[i]);
    } else {
      float vp[V];
      cur.shuffled(ln.partner).to(vp);
#pragma unroll
      for (int i = 0; i < V; ++i) z[i] = fmaf(v[i], c[i], vp[i] * r * wp[i] * s[i]);
    }
    if (live && ln.active && h < sd.heads) {
      // a partner's infinity must not reach channels that are not rotated
#pragma unroll
      for (int i = 0; i < V; ++i) z[i] = turn ? z[i] : v[i];
      Row<T> o;
      o.from(z);
      o.store(out + h * sd.o_h);
    }
  }
}

// Backward.  Blocks stride over the groups; each lane sums its channels' dw
// over its rows, first of all query rows, then of all key rows.
template <typename T, int LANES, bool INTER>
__global__ void __launch_bounds__(kThreads) backward_kernel(const Args a) {
  constexpr int V = Row<T>::kVec;
  constexpr int kGroups = kThreads / LANES;
  __shared__ float red[kGroups * LANES * V];
  const Lane<T, LANES, INTER> ln(a);
  const int gi = threadIdx.x / LANES;
#pragma unroll 1
  for (int which = 0; which < 2; ++which) {
    const Side& sd = a.side[which];
    float w[V], dw[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
      w[i] = ln.active ? weight_at(sd.w, a.wtype, ln.c0 + i) : 0.f;
      dw[i] = 0.f;
    }
    const int64_t groups = a.T * sd.chunks;
    const int64_t rounds = (groups + (int64_t)gridDim.x * kGroups - 1) / ((int64_t)gridDim.x * kGroups);
    for (int64_t n = 0; n < rounds; ++n) {
      int64_t g = (n * gridDim.x + blockIdx.x) * kGroups + gi;
      const bool live = g < groups;
      g = min(g, groups - 1);
      const int64_t t = g / sd.chunks;
      const int h0 = (int)(g - t * sd.chunks) * a.hpg;
      const T* x = static_cast<const T*>(sd.x) + t * sd.x_t + ln.c0;
      const T* gz = static_cast<const T*>(sd.g) + t * sd.g_t + ln.c0;
      T* out = static_cast<T*>(sd.out) + t * sd.o_t + ln.c0;
      float c[V], s[V];
      const bool turn = ln.angles(a, table_row(a, t), c, s);
      Row<T> nx{}, ng{};
      if (ln.active) {
        nx.load(x + min(h0, sd.heads - 1) * sd.x_h);
        ng.load(gz + min(h0, sd.heads - 1) * sd.g_h);
      }
      for (int j = 0; j < a.hpg; ++j) {
        const int h = h0 + j;
        const Row<T> cx = nx, cg = ng;
        if (ln.active && j + 1 < a.hpg) {
          nx.load(x + min(h + 1, sd.heads - 1) * sd.x_h);
          ng.load(gz + min(h + 1, sd.heads - 1) * sd.g_h);
        }
        float v[V], gy[V];
        cx.to(v);
        cg.to(gy);
        // transpose of the rotation: the signs of s swap
        if constexpr (INTER) {
          float gr[V];
#pragma unroll
          for (int i = 0; i < V; ++i) gr[i] = fmaf(gy[i], c[i], -gy[i ^ 1] * s[i]);
#pragma unroll
          for (int i = 0; i < V; ++i) gy[i] = turn ? gr[i] : gy[i];
        } else {
          float gp[V];
          cg.shuffled(ln.partner).to(gp);
          if (turn) {
#pragma unroll
            for (int i = 0; i < V; ++i) gy[i] = fmaf(gy[i], c[i], -gp[i] * s[i]);
          }
        }
        float sq = 0.f, dot = 0.f;
#pragma unroll
        for (int i = 0; i < V; ++i) {
          sq = fmaf(v[i], v[i], sq);
          dot = fmaf(gy[i] * w[i], v[i], dot);
        }
        sq = group_sum<LANES>(sq);
        dot = group_sum<LANES>(dot);
        const float r = 1.f / sqrtf(fmaf(sq, a.inv_d, a.eps));
        const float m = dot * r * a.inv_d;  // mean(g w h)
        if (live && ln.active && h < sd.heads) {
          float d[V];
#pragma unroll
          for (int i = 0; i < V; ++i) {
            const float hh = v[i] * r;
            d[i] = r * fmaf(-hh, m, gy[i] * w[i]);
            dw[i] = fmaf(gy[i], hh, dw[i]);
          }
          Row<T> o;
          o.from(d);
          o.store(out + h * sd.o_h);
        }
      }
    }
    if (a.want_dw) {
      // the block's groups in ascending order
      __syncthreads();
#pragma unroll
      for (int i = 0; i < V; ++i) red[gi * LANES * V + ln.c0 + i] = dw[i];
      __syncthreads();
      for (int d = threadIdx.x; d < a.D; d += kThreads) {
        float sum = 0.f;
#pragma unroll 8
        for (int k = 0; k < kGroups; ++k) sum += red[k * LANES * V + d];
        a.partial[((int64_t)which * gridDim.x + blockIdx.x) * a.D + d] = sum;
      }
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
  const float r = 1.f / sqrtf(fmaf(sq, a.inv_d, a.eps));
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
#pragma unroll 1
  for (int which = 0; which < 2; ++which) {
    const Side& sd = a.side[which];
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
      const float r = 1.f / sqrtf(fmaf(sq, a.inv_d, a.eps));
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
      __syncthreads();
#pragma unroll
      for (int j = 0; j < kPer; ++j) red[warp * UPLIFT_TOK_MAX_NORM_DIM + lane + 32 * j] = dw[j];
      __syncthreads();
      for (int d = threadIdx.x; d < a.D; d += kThreads) {
        float sum = 0.f;
        for (int k = 0; k < kWarps; ++k) sum += red[k * UPLIFT_TOK_MAX_NORM_DIM + d];
        a.partial[((int64_t)which * gridDim.x + blockIdx.x) * a.D + d] = sum;
      }
    }
  }
}

// dweights[which][d] = sum over blocks of partial[which][block][d], in a
// fixed order (a warp per output, lanes over blocks) and in 64 bits: the sum
// runs over all rows of the problem.
__global__ void __launch_bounds__(kThreads) dweights_kernel(const float* partial, float* dweights, int blocks, int D) {
  const int out = blockIdx.x * (kThreads / 32) + threadIdx.x / 32, lane = threadIdx.x & 31;
  if (out >= 2 * D) return;
  const int which = out / D, d = out - which * D;
  double sum = 0.0;
  for (int b = lane; b < blocks; b += 32) sum += (double)partial[((int64_t)which * blocks + b) * D + d];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if (lane == 0) dweights[out] = (float)sum;
}

template <typename T, int LANES>
void launch_vec(const Args& a, bool inter, bool bwd, int blocks, cudaStream_t s) {
  if (bwd) {
    if (inter) backward_kernel<T, LANES, true><<<blocks, kThreads, 0, s>>>(a);
    else backward_kernel<T, LANES, false><<<blocks, kThreads, 0, s>>>(a);
  } else {
    if (inter) forward_kernel<T, LANES, true><<<blocks, kThreads, 0, s>>>(a);
    else forward_kernel<T, LANES, false><<<blocks, kThreads, 0, s>>>(a);
  }
}

template <typename T>
int run(Args a, bool inter, bool bwd, cudaStream_t s) {
  constexpr int V = Row<T>::kVec;
  auto al = [](const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; };
  const int half = a.R / 2;
  bool vec = a.D % V == 0 && a.D / V <= 32 && (inter ? a.R % V == 0 : half % V == 0);
  if (!inter && a.R > 0) vec = vec && al(a.cos) && al(a.sin);
  for (int i = 0; i < 2; ++i) {
    const Side& d = a.side[i];
    vec = vec && al(d.x) && al(d.out) && d.x_t % V == 0 && d.x_h % V == 0 && d.o_t % V == 0 && d.o_h % V == 0;
    if (bwd) vec = vec && al(d.g) && d.g_t % V == 0 && d.g_h % V == 0;
  }
  int blocks = 0;
  if (vec) {
    int lanes = 4;
    while (lanes * V < a.D) lanes *= 2;
    // Heads per group: 4 amortise the token's angles, the weights and the
    // latency of the first load; 1 where 4 would leave SMs without work.
    const int64_t rows = a.T * (a.side[0].heads + a.side[1].heads);
    a.hpg = rows * lanes >= 4ll * 148 * 2048 ? 4 : 1;
    for (int i = 0; i < 2; ++i) a.side[i].chunks = (a.side[i].heads + a.hpg - 1) / a.hpg;
    const int64_t groups = a.T * (a.side[0].chunks + a.side[1].chunks);
    const int64_t need = (groups * lanes + kThreads - 1) / kThreads;
    if (!bwd && need >= (1ll << 31)) return fail(UPLIFT_LA_ERR_SHAPE, "norm_rotate: too many rows");
    blocks = bwd ? (int)std::min<int64_t>(need, kBwdBlocks) : (int)need;
    switch (lanes) {
      case 4: launch_vec<T, 4>(a, inter, bwd, blocks, s); break;
      case 8: launch_vec<T, 8>(a, inter, bwd, blocks, s); break;
      case 16: launch_vec<T, 16>(a, inter, bwd, blocks, s); break;
      default: launch_vec<T, 32>(a, inter, bwd, blocks, s); break;
    }
  } else {
    const int64_t rows = a.T * (a.side[0].heads + a.side[1].heads);
    const int64_t need = (rows + kThreads / 32 - 1) / (kThreads / 32);
    if (!bwd && need >= (1ll << 31)) return fail(UPLIFT_LA_ERR_SHAPE, "norm_rotate: too many rows");
    blocks = bwd ? (int)std::min<int64_t>(need, kBwdBlocks) : (int)need;
    if (bwd) backward_any_kernel<T><<<blocks, kThreads, 0, s>>>(a, inter);
    else forward_any_kernel<T><<<blocks, kThreads, 0, s>>>(a, inter);
  }
  return bwd ? -blocks : UPLIFT_LA_OK;
}

// Validates the arguments and fills `a`.
int prepare(const char* what, const uplift_tok_norm_rotate_args* in, bool bwd, Args* a) {
  if (in == nullptr || in->size != (int64_t)sizeof(*in)) return fail(UPLIFT_LA_ERR_ARG, "%s: no arguments, or of another version", what);
  const int dt = in->dtype, wt = in->weight_dtype;
  if (dt != UPLIFT_LA_F32 && dt != UPLIFT_LA_BF16 && dt != UPLIFT_LA_F16)
    return fail(UPLIFT_LA_ERR_ARG, "%s: unknown dtype %d", what, dt);
  if (wt != UPLIFT_LA_F32 && wt != UPLIFT_LA_BF16 && wt != UPLIFT_LA_F16)
    return fail(UPLIFT_LA_ERR_ARG, "%s: unknown weight dtype %d", what, wt);
  if (in->T < 0 || in->T >= (1ll << 31) || in->P < 0 || in->Hq < 1 || in->Hk < 1 || in->Hq > 65536 || in->Hk > 65536)
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

int run_dtype(const Args& a, int dtype, bool inter, bool bwd, cudaStream_t s) {
  if (dtype == UPLIFT_LA_F32) return run<float>(a, inter, bwd, s);
  if (dtype == UPLIFT_LA_BF16) return run<__nv_bfloat16>(a, inter, bwd, s);
  return run<__half>(a, inter, bwd, s);
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
  rc = run_dtype(a, args->dtype, args->interleaved != 0, false, static_cast<cudaStream_t>(stream));
  return rc != UPLIFT_LA_OK ? rc : tok::launched("norm_rotate");
}

int64_t uplift_tok_norm_rotate_partial_floats(int D) {
  return D < 1 ? 0 : 2ll * ula::tok::nr::kBwdBlocks * D;
}

int uplift_tok_norm_rotate_backward(const uplift_tok_norm_rotate_args* args, void* stream) {
  using namespace ula;
  using namespace ula::tok::nr;
  Args a;
  int rc = prepare("uplift_tok_norm_rotate_backward", args, true, &a);
  if (rc != UPLIFT_LA_OK) return rc;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  int blocks = 0;
  if (args->T > 0) {
    rc = run_dtype(a, args->dtype, args->interleaved != 0, true, s);
    if (rc > 0) return rc;
    blocks = -rc;
    if ((rc = tok::launched("norm_rotate backward")) != UPLIFT_LA_OK) return rc;
  }
  if (args->dweights != nullptr) {
    dweights_kernel<<<(2 * args->D + kThreads / 32 - 1) / (kThreads / 32), kThreads, 0, s>>>(args->partial, args->dweights,
                                                                                            blocks, args->D);
    return tok::launched("norm_rotate weight gradients");
  }
  return UPLIFT_LA_OK;
}

}  // extern "C"
