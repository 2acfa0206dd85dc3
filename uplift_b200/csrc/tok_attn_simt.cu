// Attention over packed sequences in fp32 on CUDA cores, forward and backward,
// D <= 128, any strides.  (The tensor cores would round the operands to 11
// bits.)  The formulas and the passes are those of the 16-bit kernels
// (tok_attn_fwd.cu, tok_attn_bwd.cu); tiles of 64 x 64 meet in shared memory
// and the 256 threads hold 4 x 4 scores and 4 rows of the result each.
//
// Bound by the fp32 units.  4 images of 1025 tokens, 6 heads of 64: forward
// 269 us (24 TFLOP/s), gradients 402 + 522 us (24, 25), a third of what the
// units could do; a warp per row with its keys 32 at a time, as it was before,
// took 6606, 12460 and 12988 us.  D = 128 runs at 30 TFLOP/s (2 CTAs per SM;
// with 1, 22 % slower).  Few queries on many keys are bound by latency instead:
// a token walks its 1000 keys in 240 us (a warp per row: 697), without a form
// that splits the keys, since decoding runs in 16 bits.

#include <math.h>

#include <algorithm>
#include <atomic>

#include "tok_attn_tc.h"

namespace ula {
namespace tok {
namespace simt {

constexpr int kWarps = 4;

__device__ __forceinline__ const float* row_of(const Rows& r, int64_t t, int h) {
  return static_cast<const float*>(r.p) + t * r.t + h * r.h;
}
__device__ __forceinline__ float* out_row(const Rows& r, int64_t t, int h) {
  return static_cast<float*>(const_cast<void*>(r.p)) + t * r.t + h * r.h;
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// delta_i = dO_i . O_i
__global__ void __launch_bounds__(kWarps * 32) delta_kernel(const AttnArgs a) {
  const int lane = threadIdx.x & 31;
  const int64_t item = (int64_t)blockIdx.x * kWarps + (threadIdx.x >> 5);
  if (item >= (int64_t)a.pk.T * a.Hq) return;
  const int t = (int)(item / a.Hq), h = (int)(item % a.Hq);
  const float* o = row_of(a.out, t, h);
  const float* g = row_of(a.dout, t, h);
  float s = 0.f;
  for (int c = lane; c < a.D; c += 32) s = fmaf(o[c], g[c], s);
  s = warp_sum(s);
  if (lane == 0) a.delta[(int64_t)h * a.pk.T + t] = s;
}

// ------------------------------------------------------------ tiles
// Two tiles of 64 rows meet in shared memory.  A tile is stored by channels,
// [DP][kPitch] with the rows along the line, so that both kinds of product
// read float4 without bank conflicts:
//   S[64 x 64] = X Y^T:  thread (ty, tx) owns rows 4 ty .. + 3 and columns
//     4 tx .. + 3 (a line of X, shared by the lanes of a ty, and of Y per channel);
//   A[64 x D] += P Y:    rows 4 ty .. + 3, channels tx + 16 i (P by rows).
constexpr int kTile = 64, kPitch = 68, kTileThreads = 256;

template <int DP>
__device__ __forceinline__ void load_tile(float* dst, const Rows& src, int64_t row0, int h, int n, int D, float scale) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const float* p = static_cast<const float*>(src.p) + row0 * src.t + (int64_t)h * src.h;
  // a warp takes 4 rows x 8 channels: whole sectors, and 32 different banks
#pragma unroll 8
  for (int i = warp; i < 2 * DP; i += kTileThreads / 32) {
    const int r = 4 * (i & 15) + (lane >> 3), d = 8 * (i >> 4) + (lane & 7);
    dst[d * kPitch + r] = r < n && d < D ? p[r * src.t + d] * scale : 0.f;
  }
}

__device__ __forceinline__ float4 ld4(const float* p) { return *reinterpret_cast<const float4*>(p); }

__device__ __forceinline__ void product(const float* x, const float* y, int D, float (&s)[4][4]) {
  const int ty = threadIdx.x >> 4, tx = threadIdx.x & 15;
#pragma unroll
  for (int r = 0; r < 4; ++r)
#pragma unroll
    for (int c = 0; c < 4; ++c) s[r][c] = 0.f;
#pragma unroll 8
  for (int d = 0; d < D; ++d) {
    const float4 a4 = ld4(x + d * kPitch + 4 * ty), b4 = ld4(y + d * kPitch + 4 * tx);
    const float a[4] = {a4.x, a4.y, a4.z, a4.w}, b[4] = {b4.x, b4.y, b4.z, b4.w};
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
      for (int c = 0; c < 4; ++c) s[r][c] = fmaf(a[r], b[c], s[r][c]);
  }
}

// EDGE: row r only takes the columns lo[r] .. hi[r] - 1: an infinity or NaN
// in a row of Y that it does not see must not meet its weight of zero.
template <int DP, bool EDGE>
__device__ __forceinline__ void accumulate(const float* w, const float* y, const int (&lo)[4], const int (&hi)[4],
                                           float (&acc)[4][DP / 16]) {
  const int ty = threadIdx.x >> 4, tx = threadIdx.x & 15;
#pragma unroll 2
  for (int k = 0; k < kTile; k += 4) {
    float a[4][4];
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const float4 v = ld4(w + (4 * ty + r) * kPitch + k);
      a[r][0] = v.x; a[r][1] = v.y; a[r][2] = v.z; a[r][3] = v.w;
    }
#pragma unroll
    for (int i = 0; i < DP / 16; ++i) {
      const float4 v = ld4(y + (tx + 16 * i) * kPitch + k);
      const float b[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (!EDGE || (k + e >= lo[r] && k + e < hi[r])) acc[r][i] = fmaf(a[r][e], b[e], acc[r][i]);
    }
  }
}

__device__ __forceinline__ void store4(float* w, int r, const float (&x)[4]) {
  const int ty = threadIdx.x >> 4, tx = threadIdx.x & 15;
  *reinterpret_cast<float4*>(w + (4 * ty + r) * kPitch + 4 * tx) = make_float4(x[0], x[1], x[2], x[3]);
}

// The next item of this CTA: sequence and tile (threads of the CTA agree).
struct Items {
  TileWalk walk;
  int n = 0;
  __device__ __forceinline__ bool next(const Packing& pk, bool by_keys, int heads, int* shared, int* b, int* local, int* h) {
    const int64_t i = dealt(n++);
    const int64_t tile = i / heads;
    __syncthreads();  // the shared words and tiles of the last item have been read
    if (threadIdx.x < 32) {
      int tiles;
      const bool more = tile < (1ll << 31) && walk.find(pk, by_keys, kTile, (int)tile, b, local, &tiles);
      if (threadIdx.x == 0) {
        shared[0] = more ? *b : -1;
        shared[1] = *local;
      }
    }
    __syncthreads();
    *b = shared[0];
    *local = shared[1];
    *h = (int)(i - tile * heads);
    return *b >= 0;
  }
};

// Zeros (and lse = -inf) for the rows of no sequence.
__device__ __forceinline__ void clear_gaps(const int32_t* cu, int B, int rows, int heads, int D, const Rows& o, const Rows* o2, float* lse) {
  int lo = 0, hi = 0;
  if (B > 0) {
    lo = segment(cu, 0, rows).x;
    const int2 e = segment(cu, B - 1, rows);
    hi = max(lo, e.x + e.y);
  }
  const int lane = threadIdx.x & 31;
  const int64_t gap = (int64_t)lo + (rows - hi);
  constexpr int kW = kTileThreads / 32;
  for (int64_t i = (int64_t)blockIdx.x * kW + (threadIdx.x >> 5); i < gap * heads; i += (int64_t)gridDim.x * kW) {
    const int64_t k = i / heads;
    const int h = (int)(i - k * heads);
    const int64_t row = k < lo ? k : hi + (k - lo);
    for (int c = lane; c < D; c += 32) {
      out_row(o, row, h)[c] = 0.f;
      if (o2 != nullptr) out_row(*o2, row, h)[c] = 0.f;
    }
    if (lse != nullptr && lane == 0) lse[(int64_t)h * rows + row] = -INFINITY;
  }
}

template <int DP> constexpr int kFwdSmem = 3 * DP * kPitch * 4;
template <int DP, bool KEYS> constexpr int kBwdSmem = (4 * DP + (KEYS ? 2 : 1) * kTile) * kPitch * 4;
template <int DP> constexpr int kFwdCtas = DP == 64 ? 3 : 2;
template <int DP> constexpr int kBwdCtas = DP == 64 ? 2 : 1;

// One pass over the keys with the running maximum and sum of the softmax.
template <int DP>
__global__ void __launch_bounds__(kTileThreads, kFwdCtas<DP>) forward_tile_kernel(const AttnArgs a) {
  extern __shared__ __align__(16) float tiles[];
  __shared__ int shared[2];
  float *sq = tiles, *sk = sq + DP * kPitch, *sv = sk + DP * kPitch;  // the weights overwrite K
  const int ty = threadIdx.x >> 4, tx = threadIdx.x & 15;
  Items items;
  int b, local, h;
  while (items.next(a.pk, false, a.Hq, shared, &b, &local, &h)) {
    const Seq s = sequence(a.pk, b);
    const int i0 = local * kTile, n = min(kTile, s.nq - i0), hk = h / (a.Hq / a.Hk);
    int see[4], lo[4] = {0, 0, 0, 0}, hi[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) see[r] = 4 * ty + r < n ? keys_seen(s, i0 + 4 * ty + r, a.pk.causal) : 0;
    const int all = keys_seen(s, i0 + n - 1, a.pk.causal);          // keys that some row sees
    const int every = n == kTile ? keys_seen(s, i0, a.pk.causal) : 0;  // .. that every row does
    load_tile<DP>(sq, a.q, s.q0 + i0, h, n, a.D, a.scale);
    float m[4], l[4], acc[4][DP / 16];
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      m[r] = -INFINITY;
      l[r] = 0.f;
#pragma unroll
      for (int i = 0; i < DP / 16; ++i) acc[r][i] = 0.f;
    }
    for (int j = 0; j < all; j += kTile) {
      __syncthreads();
      load_tile<DP>(sk, a.k, s.k0 + j, hk, min(kTile, all - j), a.D, 1.f);
      load_tile<DP>(sv, a.v, s.k0 + j, hk, min(kTile, all - j), a.D, 1.f);
      __syncthreads();
      float x[4][4];
      product(sq, sk, a.D, x);
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        hi[r] = see[r] - j;
        float mx = -INFINITY;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          if (4 * tx + c >= hi[r]) x[r][c] = -INFINITY;
          mx = fmaxf(mx, x[r][c]);
        }
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
        const float mn = fmaxf(m[r], mx), ms = mn == -INFINITY ? 0.f : mn, f = expf(m[r] - ms);
        m[r] = mn;
        float sum = 0.f;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          x[r][c] = expf(x[r][c] - ms);
          sum += x[r][c];
        }
        l[r] = fmaf(l[r], f, sum);
#pragma unroll
        for (int i = 0; i < DP / 16; ++i) acc[r][i] *= f;
      }
      __syncthreads();
#pragma unroll
      for (int r = 0; r < 4; ++r) store4(sk, r, x[r]);
      __syncthreads();
      if (j + kTile <= every) accumulate<DP, false>(sk, sv, lo, hi, acc);
      else accumulate<DP, true>(sk, sv, lo, hi, acc);
    }
#pragma unroll
    for (int r = 0; r < 4; ++r) {
#pragma unroll
      for (int o = 8; o > 0; o >>= 1) l[r] += __shfl_xor_sync(0xffffffffu, l[r], o);
      if (4 * ty + r >= n) continue;
      const bool none = l[r] == 0.f;  // no key seen, or all scores -inf
      const int64_t row = s.q0 + i0 + 4 * ty + r;
#pragma unroll
      for (int i = 0; i < DP / 16; ++i)
        if (tx + 16 * i < a.D) out_row(a.out, row, h)[tx + 16 * i] = none ? 0.f : acc[r][i] / l[r];
      if (a.lse != nullptr && tx == 0) a.lse[(int64_t)h * a.pk.T + row] = none ? -INFINITY : m[r] + logf(l[r]);
    }
  }
  clear_gaps(a.pk.cu_q, a.pk.B, a.pk.T, a.Hq, a.D, a.out, nullptr, a.lse);
}

// Gradients: the rows of one side stay (X0, X1), the other's go by (Y0, Y1).
//   !KEYS: X = Q, dO of 64 queries of a head, Y = K, V:  dQ = dS Y0;
//   KEYS:  X = K, V of 64 keys of a key head, Y = Q, dO of all heads of its
//          group:  dK = dS^T Y0, dV = P^T Y1.
// Each CTA owns the rows that it writes: no atomics, one order of summation.
template <int DP, bool KEYS>
__global__ void __launch_bounds__(kTileThreads, kBwdCtas<DP>) gradient_tile_kernel(const AttnArgs a) {
  extern __shared__ __align__(16) float tiles[];
  __shared__ int shared[2];
  float *x0 = tiles, *x1 = x0 + DP * kPitch, *y0 = x1 + DP * kPitch, *y1 = y0 + DP * kPitch;
  float *sds = y1 + DP * kPitch, *sp = sds + kTile * kPitch;
  const int ty = threadIdx.x >> 4, tx = threadIdx.x & 15;
  const int group = a.Hq / a.Hk;
  Items items;
  int b, local, h;
  while (items.next(a.pk, KEYS, KEYS ? a.Hk : a.Hq, shared, &b, &local, &h)) {
    const Seq s = sequence(a.pk, b);
    const int t0 = local * kTile;
    const int n = min(kTile, (KEYS ? segment(a.pk.cu_k, b, a.pk.S).y : s.nq) - t0);
    const int live = KEYS ? max(0, min(n, s.nk - t0)) : n;  // behind them: room of the cache
    const int64_t row0 = (KEYS ? s.k0 : s.q0) + t0;
    // the rows of the other side that go by
    const int first = KEYS && a.pk.causal ? max(0, t0 - s.nk + s.nq) : 0;
    const int end = live == 0 ? 0 : KEYS ? s.nq : keys_seen(s, t0 + n - 1, a.pk.causal);
    load_tile<DP>(x0, KEYS ? a.k : a.q, row0, h, live, a.D, a.scale);
    load_tile<DP>(x1, KEYS ? a.v : a.dout, row0, h, live, a.D, 1.f);
    float lse[4], delta[4], acc0[4][DP / 16], acc1[4][DP / 16];
    int from[4], to[4];  // that row r takes part in
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int i = 4 * ty + r;
      from[r] = KEYS && a.pk.causal ? t0 + i - s.nk + s.nq : 0;
      to[r] = i >= live ? 0 : KEYS ? s.nq : keys_seen(s, t0 + i, a.pk.causal);
      if (!KEYS && i < live) {
        lse[r] = a.lse[(int64_t)h * a.pk.T + row0 + i];
        delta[r] = a.delta[(int64_t)h * a.pk.T + row0 + i];
        if (lse[r] == -INFINITY) to[r] = 0;
      }
#pragma unroll
      for (int c = 0; c < DP / 16; ++c) acc0[r][c] = acc1[r][c] = 0.f;
    }
    for (int g = 0; g < (KEYS ? group : 1); ++g) {
      const int hy = KEYS ? h * group + g : h / group;
      for (int y = first; y < end; y += kTile) {
        const int ny = min(kTile, end - y);
        __syncthreads();
        load_tile<DP>(y0, KEYS ? a.q : a.k, (KEYS ? s.q0 : s.k0) + y, hy, ny, a.D, 1.f);
        load_tile<DP>(y1, KEYS ? a.dout : a.v, (KEYS ? s.q0 : s.k0) + y, hy, ny, a.D, 1.f);
        __syncthreads();
        float p[4][4], ds[4][4];
        product(x0, y0, a.D, p);
        product(x1, y1, a.D, ds);
        int lo[4], hi[4];
        bool whole = true;  // every row takes part in every column
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          lo[r] = from[r] - y;
          hi[r] = to[r] - y;
          whole = whole && lo[r] <= 0 && hi[r] >= kTile;
        }
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const int col = 4 * tx + c;
          float ls = 0.f, de = 0.f;
          if (KEYS && col < ny) {
            const int64_t at = (int64_t)hy * a.pk.T + s.q0 + y + col;
            ls = a.lse[at];
            de = a.delta[at];
          }
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const float le = KEYS ? ls : lse[r];
            const bool seen = col >= lo[r] && col < hi[r] && le != -INFINITY;
            p[r][c] = seen ? expf(p[r][c] - le) : 0.f;
            ds[r][c] = seen ? p[r][c] * (ds[r][c] - (KEYS ? de : delta[r])) * a.scale : 0.f;
          }
        }
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          store4(sds, r, ds[r]);
          if (KEYS) store4(sp, r, p[r]);
        }
        whole = __syncthreads_and(whole) != 0;
        if (whole) {
          accumulate<DP, false>(sds, y0, lo, hi, acc0);
          if (KEYS) accumulate<DP, false>(sp, y1, lo, hi, acc1);
        } else {
          accumulate<DP, true>(sds, y0, lo, hi, acc0);
          if (KEYS) accumulate<DP, true>(sp, y1, lo, hi, acc1);
        }
      }
    }
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      if (4 * ty + r >= n) continue;
      const int64_t row = row0 + 4 * ty + r;
#pragma unroll
      for (int i = 0; i < DP / 16; ++i) {
        if (tx + 16 * i >= a.D) continue;
        out_row(KEYS ? a.dk : a.dq, row, h)[tx + 16 * i] = acc0[r][i];
        if (KEYS) out_row(a.dv, row, h)[tx + 16 * i] = acc1[r][i];
      }
    }
  }
  if (KEYS) clear_gaps(a.pk.cu_k, a.pk.B, a.pk.S, a.Hk, a.D, a.dk, &a.dv, nullptr);
  else clear_gaps(a.pk.cu_q, a.pk.B, a.pk.T, a.Hq, a.D, a.dq, nullptr, nullptr);
}

// One CTA per item, as many as the SMs hold.
int grid_for(int64_t rows, int B, int heads, int ctas, int sms) {
  const int64_t most = (rows / kTile + std::min<int64_t>(rows, B)) * heads;
  return (int)std::min<int64_t>(std::max<int64_t>(most, 1), (int64_t)sms * ctas);
}

template <int DP>
int forward_tiles(const AttnArgs& a, int dev, int sms, cudaStream_t s) {
  static std::atomic<bool> configured[64] = {};
  const int rc = opt_in_smem(forward_tile_kernel<DP>, kFwdSmem<DP>, configured, dev);
  if (rc != UPLIFT_LA_OK) return rc;
  forward_tile_kernel<DP><<<grid_for(a.pk.T, a.pk.B, a.Hq, kFwdCtas<DP>, sms), kTileThreads, kFwdSmem<DP>, s>>>(a);
  return launched("attention");
}

template <int DP, bool KEYS>
int gradient_tiles(const AttnArgs& a, int dev, int sms, cudaStream_t s) {
  static std::atomic<bool> configured[64] = {};
  const int rc = opt_in_smem(gradient_tile_kernel<DP, KEYS>, kBwdSmem<DP, KEYS>, configured, dev);
  if (rc != UPLIFT_LA_OK) return rc;
  const int grid = grid_for(KEYS ? a.pk.S : a.pk.T, a.pk.B, KEYS ? a.Hk : a.Hq, kBwdCtas<DP>, sms);
  gradient_tile_kernel<DP, KEYS><<<grid, kTileThreads, kBwdSmem<DP, KEYS>, s>>>(a);
  return launched("attention backward");
}

int blocks_for(int64_t items, int* blocks) {
  const int64_t n = (items + kWarps - 1) / kWarps;
  if (n >= (1ll << 31)) return fail(UPLIFT_LA_ERR_SHAPE, "attention: too many rows");
  *blocks = (int)n;
  return UPLIFT_LA_OK;
}

}  // namespace simt

int attn_simt_forward(const AttnArgs& a, cudaStream_t s) {
  using namespace simt;
  int dev = 0, sms = 0;
  const int rc = sm_count(&dev, &sms);
  if (rc != UPLIFT_LA_OK) return rc;
  return a.D <= 64 ? forward_tiles<64>(a, dev, sms, s) : forward_tiles<128>(a, dev, sms, s);
}

int attn_simt_backward(const AttnArgs& a, cudaStream_t s) {
  using namespace simt;
  int dev = 0, sms = 0, blocks = 0;
  int rc = sm_count(&dev, &sms);
  if (rc == UPLIFT_LA_OK) rc = blocks_for((int64_t)a.pk.T * a.Hq, &blocks);
  if (rc != UPLIFT_LA_OK) return rc;
  if (blocks > 0) {
    delta_kernel<<<blocks, kWarps * 32, 0, s>>>(a);
    rc = a.D <= 64 ? gradient_tiles<64, false>(a, dev, sms, s) : gradient_tiles<128, false>(a, dev, sms, s);
    if (rc != UPLIFT_LA_OK) return rc;
  }
  if (a.pk.S == 0) return UPLIFT_LA_OK;
  return a.D <= 64 ? gradient_tiles<64, true>(a, dev, sms, s) : gradient_tiles<128, true>(a, dev, sms, s);
}

}  // namespace tok
}  // namespace ula
