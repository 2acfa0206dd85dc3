// Attention of few queries per sequence on long key ranges -- the step of
// one new token per sequence -- for bf16 / fp16, D <= 128.
//
// Each key and value is read once and meets only the Hq / Hk queries of its
// group, so HBM bounds it: the kernel is built to keep loads in flight.  The
// keys of a query token are cut into chunks; an item is one chunk for one
// token and key head, and its group's query heads are the 16 rows of
// mma.m16n8k16 (fewer are padded, more make further items).  The CTA's four
// warps take 16 keys in turn, each with its own running maximum and sum:
//
//   S[16 x 16] = Q K^T,  P = exp2((S - m) scale log2 e),  O[16 x D] += P V
//
// K and V go from global memory straight into the registers of the MMA
// fragments, 16 bytes per load: the order of the channels in a product does
// not matter, so a lane takes 8 neighbouring channels of a key as its part of
// two k-steps (Q is laid out alike), and 8 neighbouring channels of four keys
// of V as its columns of eight n-tiles (pairs of keys are merged by byte
// permutes).  The next K is loaded while the weights are formed, V while the
// scores are.  The warps' results are joined in shared memory; the chunks'
// results go to a workspace and a second kernel joins them, unless the
// token has one chunk only.

#include <math.h>

#include <algorithm>
#include <atomic>

#include "tok_attn_tc.h"

namespace ula {
namespace tok {
namespace step {

constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
constexpr int kKeys = 16;          // keys of a warp at a time
constexpr int kRows = 16;          // query heads of an item
constexpr int kMinChunk = kWarps * kKeys;
constexpr int kMaxChunks = 128;    // of one token
constexpr int kCtasPerSm = 3;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kRescale = 8.f;    // see tok_attn_fwd.cu

struct Params {
  Rows q, k, v, out;
  float* lse;
  float* part_o;   // [T][chunks][Hq][D]
  float2* part_ml; // [T][chunks][Hq]: maximum (of scale S log2 e) and sum
  Packing pk;
  int Hq, Hk, group, D;
  int row_tiles;   // ceil(group / 16)
  int chunks;      // at most, per token
  int min_len;     // least keys of a chunk
  float scale;
};

// Keys of a chunk of a sequence, a multiple of kMinChunk.
__device__ __forceinline__ int chunk_len(const Params& p, int nk) {
  const int even = (nk + p.chunks - 1) / p.chunks;
  return max(p.min_len, (even + kMinChunk - 1) / kMinChunk * kMinChunk);
}

template <typename T> struct Mma;
template <> struct Mma<__nv_bfloat16> {
  __device__ __forceinline__ static void run(float* c, const uint32_t* a, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
};
template <> struct Mma<__half> {
  __device__ __forceinline__ static void run(float* c, const uint32_t* a, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
};

__device__ __forceinline__ float quad_max(float v) {
  v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 1));
  return fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 2));
}
__device__ __forceinline__ float quad_sum(float v) {
  v += __shfl_xor_sync(0xffffffffu, v, 1);
  return v + __shfl_xor_sync(0xffffffffu, v, 2);
}
// Loads that are not kept in L1: every byte is used once.
__device__ __forceinline__ uint4 load16(const void* p, bool there) {
  uint4 v = make_uint4(0, 0, 0, 0);
  if (there) asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}

// Units of a sequence: one per query token and chunk of its keys.
struct UnitWalk {
  int b0 = 0;
  int64_t before = 0;
  __device__ __forceinline__ bool find(const Params& p, int64_t unit, Seq* s, int* len, int* local) {
    const int lane = threadIdx.x & 31;
    while (b0 < p.pk.B) {
      Seq mine{};
      int l = kMinChunk;
      int64_t n = 0;
      if (b0 + lane < p.pk.B) {
        mine = sequence(p.pk, b0 + lane);
        l = chunk_len(p, mine.nk);
        n = (int64_t)mine.nq * ((mine.nk + l - 1) / l);
      }
      int64_t sum = n;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int64_t v = __shfl_up_sync(0xffffffffu, sum, o);
        if (lane >= o) sum += v;
      }
      const int64_t total = __shfl_sync(0xffffffffu, sum, 31);
      if (unit < before + total) {
        const int src = __ffs(__ballot_sync(0xffffffffu, unit < before + sum)) - 1;
        s->q0 = __shfl_sync(0xffffffffu, mine.q0, src);
        s->nq = __shfl_sync(0xffffffffu, mine.nq, src);
        s->k0 = __shfl_sync(0xffffffffu, mine.k0, src);
        s->nk = __shfl_sync(0xffffffffu, mine.nk, src);
        *len = __shfl_sync(0xffffffffu, l, src);
        *local = (int)(unit - before - __shfl_sync(0xffffffffu, sum - n, src));
        return true;
      }
      before += total;
      b0 += 32;
    }
    return false;
  }
};

template <typename T, int DP>
__global__ void __launch_bounds__(kThreads, kCtasPerSm) chunk_kernel(const Params p) {
  constexpr int KB = DP / 32;  // blocks of 32 channels of Q and K
  constexpr int VB = DP / 64;  // blocks of 64 channels of V
  constexpr int kPad = DP + 4;
  __shared__ float s_m[kWarps][kRows], s_l[kWarps][kRows];
  __shared__ __align__(16) float s_o[kWarps][kRows][kPad];
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, t = lane & 3;
  const float c2 = p.scale * kLog2e;
  UnitWalk walk;
  const int per_unit = p.Hk * p.row_tiles;
  for (int64_t i = blockIdx.x;; i += gridDim.x) {
    Seq s;
    int len, local;
    const int64_t unit = i / per_unit;
    if (!walk.find(p, unit, &s, &len, &local)) break;
    const int sub = (int)(i - unit * per_unit);
    const int hk = sub / p.row_tiles, h0 = hk * p.group + (sub - hk * p.row_tiles) * kRows;
    const int rows = min(kRows, (hk + 1) * p.group - h0);
    const int chunks = (s.nk + len - 1) / len;
    const int tok = local / chunks, chunk = local - tok * chunks;
    const int see = keys_seen(s, tok, p.pk.causal);
    const int j0 = chunk * len, j1 = min(see, j0 + len);
    if (j0 >= j1) continue;  // this token sees none of the chunk (the whole CTA skips it)
    const int64_t row = s.q0 + tok;
    // Q: rows g and g + 8, 8 channels of each block of 32
    uint32_t qa[KB][2][4];
#pragma unroll
    for (int b = 0; b < KB; ++b) {
      const int c = 32 * b + 8 * t;
      const T* q = static_cast<const T*>(p.q.p) + row * p.q.t + (int64_t)h0 * p.q.h + c;
      const uint4 lo = load16(q + g * p.q.h, g < rows && c < p.D);
      const uint4 hi = load16(q + (g + 8) * p.q.h, g + 8 < rows && c < p.D);
      qa[b][0][0] = lo.x; qa[b][0][1] = hi.x; qa[b][0][2] = lo.y; qa[b][0][3] = hi.y;
      qa[b][1][0] = lo.z; qa[b][1][1] = hi.z; qa[b][1][2] = lo.w; qa[b][1][3] = hi.w;
    }
    const T* kb = static_cast<const T*>(p.k.p) + (int64_t)s.k0 * p.k.t + (int64_t)hk * p.k.h + 8 * t;
    const T* vb = static_cast<const T*>(p.v.p) + (int64_t)s.k0 * p.v.t + (int64_t)hk * p.v.h + 8 * g;
    uint4 kr[KB][2];
    auto load_k = [&](int j) {  // keys j + g, j + 8 + g
#pragma unroll
      for (int b = 0; b < KB; ++b) {
#pragma unroll
        for (int u = 0; u < 2; ++u)
          kr[b][u] = load16(kb + (int64_t)(j + 8 * u + g) * p.k.t + 32 * b, j + 8 * u + g < j1 && 32 * b + 8 * t < p.D);
      }
    };
    float acc[VB][8][4], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
#pragma unroll
    for (int b = 0; b < VB; ++b) {
#pragma unroll
      for (int e = 0; e < 8; ++e) acc[b][e][0] = acc[b][e][1] = acc[b][e][2] = acc[b][e][3] = 0.f;
    }
    int j = j0 + warp * kKeys;
    if (j < j1) load_k(j);
    for (; j < j1; j += kMinChunk) {
      uint4 vr[VB][4];  // keys j + 2t, + 2t + 1, + 2t + 8, + 2t + 9
#pragma unroll
      for (int b = 0; b < VB; ++b) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int key = j + 2 * t + (e & 1) + 8 * (e >> 1);
          vr[b][e] = load16(vb + (int64_t)key * p.v.t + 64 * b, key < j1 && 64 * b + 8 * g < p.D);
        }
      }
      float sc[2][4] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
      for (int b = 0; b < KB; ++b) {
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          Mma<T>::run(sc[u], qa[b][0], kr[b][u].x, kr[b][u].y);
          Mma<T>::run(sc[u], qa[b][1], kr[b][u].z, kr[b][u].w);
        }
      }
      if (j + kMinChunk < j1) load_k(j + kMinChunk);
      if (j + kKeys > j1) {
#pragma unroll
        for (int u = 0; u < 2; ++u) {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (j + 8 * u + 2 * t + (e & 1) >= j1) sc[u][e] = -INFINITY;
        }
      }
      uint32_t pa[4];
#pragma unroll
      for (int h = 0; h < 2; ++h) {  // rows g, g + 8
        const float mx = quad_max(fmaxf(fmaxf(sc[0][2 * h], sc[0][2 * h + 1]), fmaxf(sc[1][2 * h], sc[1][2 * h + 1]))) * c2;
        const bool grow = mx - m[h] > kRescale || (m[h] == -INFINITY && mx > m[h]);
        if (__any_sync(0xffffffffu, grow)) {
          const float f = grow ? ex2(m[h] - mx) : 1.f;  // exp2(-inf) = 0 at the first keys
          if (grow) m[h] = mx;
          l[h] *= f;
#pragma unroll
          for (int b = 0; b < VB; ++b) {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              acc[b][e][2 * h] *= f;
              acc[b][e][2 * h + 1] *= f;
            }
          }
        }
        const float mm = m[h] == -INFINITY ? 0.f : m[h];
        float w[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) w[e] = ex2(fmaf(sc[e >> 1][2 * h + (e & 1)], c2, -mm));
        l[h] += (w[0] + w[1]) + (w[2] + w[3]);
        pa[h] = St<T>::pack(w[0], w[1]);
        pa[2 + h] = St<T>::pack(w[2], w[3]);
      }
#pragma unroll
      for (int b = 0; b < VB; ++b) {
        const uint32_t* x[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = &vr[b][e].x;
#pragma unroll
        for (int e = 0; e < 4; ++e) {  // channels 8g + 2e, 8g + 2e + 1
          Mma<T>::run(acc[b][2 * e], pa, __byte_perm(x[0][e], x[1][e], 0x5410), __byte_perm(x[2][e], x[3][e], 0x5410));
          Mma<T>::run(acc[b][2 * e + 1], pa, __byte_perm(x[0][e], x[1][e], 0x7632), __byte_perm(x[2][e], x[3][e], 0x7632));
        }
      }
    }
    // join the warps
#pragma unroll
    for (int h = 0; h < 2; ++h) l[h] = quad_sum(l[h]);
    if (t == 0) {
      s_m[warp][g] = m[0];
      s_m[warp][g + 8] = m[1];
      s_l[warp][g] = l[0];
      s_l[warp][g + 8] = l[1];
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      if (g + 8 * h < rows) {
#pragma unroll
        for (int b = 0; b < VB; ++b) {
#pragma unroll
          for (int n = 0; n < 2; ++n) {  // accumulator columns 2t, 2t + 1: channels 8 (2t + n) + e
            float* o = &s_o[warp][g + 8 * h][64 * b + 8 * (2 * t + n)];
            *reinterpret_cast<float4*>(o) = make_float4(acc[b][0][2 * h + n], acc[b][1][2 * h + n], acc[b][2][2 * h + n], acc[b][3][2 * h + n]);
            *reinterpret_cast<float4*>(o + 4) = make_float4(acc[b][4][2 * h + n], acc[b][5][2 * h + n], acc[b][6][2 * h + n], acc[b][7][2 * h + n]);
          }
        }
      }
    }
    __syncthreads();
    const bool last = see <= len;  // the token's only chunk
    for (int e = threadIdx.x; e < rows * (DP / 4); e += kThreads) {
      const int rr = e / (DP / 4), c = (e - rr * (DP / 4)) * 4;
      if (c >= p.D) continue;
      float mm = -INFINITY;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) mm = fmaxf(mm, s_m[w][rr]);
      float sum = 0.f;
      float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const float f = s_m[w][rr] == -INFINITY ? 0.f : ex2(s_m[w][rr] - mm);
        // a warp that saw NaN scores only still has m = -inf
        const float lw = s_l[w][rr];
        const float4 x = *reinterpret_cast<const float4*>(&s_o[w][rr][c]);
        const float ff = lw == lw ? f : lw;
        sum = fmaf(lw, ff, sum);
        o.x = fmaf(x.x, ff, o.x); o.y = fmaf(x.y, ff, o.y); o.z = fmaf(x.z, ff, o.z); o.w = fmaf(x.w, ff, o.w);
      }
      const int h = h0 + rr;
      if (last) {
        const float inv = sum == 0.f ? 0.f : 1.f / sum;
        if (sum == 0.f) o = make_float4(0.f, 0.f, 0.f, 0.f);
        *reinterpret_cast<uint2*>(static_cast<T*>(const_cast<void*>(p.out.p)) + row * p.out.t + (int64_t)h * p.out.h + c) =
            make_uint2(St<T>::pack(o.x * inv, o.y * inv), St<T>::pack(o.z * inv, o.w * inv));
        if (c == 0 && p.lse != nullptr)
          p.lse[(int64_t)h * p.pk.T + row] = sum == 0.f ? -INFINITY : mm / kLog2e + logf(sum);
      } else {
        const int64_t at = (row * p.chunks + chunk) * p.Hq + h;
        *reinterpret_cast<float4*>(p.part_o + at * p.D + c) = o;
        if (c == 0) p.part_ml[at] = make_float2(mm, sum);
      }
    }
    __syncthreads();
  }
}

// Sequence of row t (the last one that starts at or before it).
__device__ __forceinline__ int sequence_of(const int32_t* cu, int B, int t) {
  int lo = 0, hi = B;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (__ldg(cu + mid) <= t) lo = mid;
    else hi = mid;
  }
  return lo;
}

// Joins the chunks of each token and head (a warp each); also writes the
// rows that see no key or belong to no sequence.
template <typename T>
__global__ void __launch_bounds__(256) join_kernel(const Params p) {
  const int lane = threadIdx.x & 31;
  const int64_t item = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  // the sequences were there before the first kernel began
  int chunks = 0;
  const bool live = item < (int64_t)p.pk.T * p.Hq;
  const int64_t row = live ? item / p.Hq : 0;
  const int h = (int)(item - row * p.Hq);
  if (live && p.pk.B > 0) {
    const Seq s = sequence(p.pk, sequence_of(p.pk.cu_q, p.pk.B, (int)row));
    if (row >= s.q0 && row < s.q0 + s.nq) {
      const int see = keys_seen(s, (int)row - s.q0, p.pk.causal), len = chunk_len(p, s.nk);
      chunks = (see + len - 1) / len;
    }
  }
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (!live || chunks == 1) return;
  const int64_t base = row * p.chunks * p.Hq + h;
  float mm = -INFINITY, ml[kMaxChunks / 32], ll[kMaxChunks / 32];
#pragma unroll
  for (int i = 0; i < kMaxChunks / 32; ++i) {
    const int c = lane + 32 * i;
    ml[i] = -INFINITY;
    ll[i] = 0.f;
    if (c < chunks) {
      const float2 v = p.part_ml[base + (int64_t)c * p.Hq];
      ml[i] = v.x;
      ll[i] = v.y;
    }
    mm = fmaxf(mm, ml[i]);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) mm = fmaxf(mm, __shfl_xor_sync(0xffffffffu, mm, o));
  float sum = 0.f;
#pragma unroll
  for (int i = 0; i < kMaxChunks / 32; ++i) {
    const float f = ml[i] == -INFINITY ? 0.f : ex2(ml[i] - mm);
    ml[i] = ll[i] == ll[i] ? f : ll[i];  // weight of the chunk; NaN stays NaN
    sum = fmaf(ll[i], ml[i], sum);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  const int c = lane * 4;
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
  for (int i = 0; i < kMaxChunks / 32; ++i) {
    const int cnt = min(32, chunks - 32 * i);
    for (int e = 0; e < cnt; ++e) {
      const float f = __shfl_sync(0xffffffffu, ml[i], e);
      if (c < p.D) {
        const float4 x = *reinterpret_cast<const float4*>(p.part_o + (base + (int64_t)(32 * i + e) * p.Hq) * p.D + c);
        o.x = fmaf(x.x, f, o.x); o.y = fmaf(x.y, f, o.y); o.z = fmaf(x.z, f, o.z); o.w = fmaf(x.w, f, o.w);
      }
    }
  }
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  if (sum == 0.f) o = make_float4(0.f, 0.f, 0.f, 0.f);
  if (c < p.D)
    *reinterpret_cast<uint2*>(static_cast<T*>(const_cast<void*>(p.out.p)) + row * p.out.t + (int64_t)h * p.out.h + c) =
        make_uint2(St<T>::pack(o.x * inv, o.y * inv), St<T>::pack(o.z * inv, o.w * inv));
  if (lane == 0 && p.lse != nullptr)
    p.lse[(int64_t)h * p.pk.T + row] = sum == 0.f ? -INFINITY : mm / kLog2e + logf(sum);
}

// Chunks per token, at most: enough that the items fill the SMs several
// times over, so that sequences of different lengths even out.
int chunks_for(int64_t T, int group, int Hk) {
  const int64_t per_chunk = T * Hk * ((group + kRows - 1) / kRows);
  return (int)std::min<int64_t>(kMaxChunks, std::max<int64_t>(1, (148 * 24 + per_chunk - 1) / per_chunk));
}

template <typename T, int DP>
int run(const Params& p, int sms, cudaStream_t s) {
  const int64_t most = (int64_t)p.pk.T * p.chunks * p.Hk * p.row_tiles;
  const int grid = (int)std::min<int64_t>(most, (int64_t)sms * kCtasPerSm);
  chunk_kernel<T, DP><<<grid, kThreads, 0, s>>>(p);
  int rc = launched("attention");
  if (rc != UPLIFT_LA_OK) return rc;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(((int64_t)p.pk.T * p.Hq + 7) / 8));
  cfg.blockDim = dim3(256);
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, join_kernel<T>, p);
  if (e != cudaSuccess) return fail(UPLIFT_LA_ERR_CUDA, "attention launch: %s", cudaGetErrorString(e));
  return launched("attention");
}

}  // namespace step

// Few queries per sequence: the keys are read for each query token, so this
// form is for batches with at most a few tokens per sequence.
bool attn_step_applies(int B, int64_t T, int dtype) { return dtype != UPLIFT_LA_F32 && T <= 4ll * B && T <= 65536; }

int64_t attn_step_workspace(int64_t T, int Hq, int Hk, int D) {
  return T * step::chunks_for(T, Hq / Hk, Hk) * Hq * (D + 2) * 4;
}

int attn_step_forward(const AttnArgs& a, void* workspace, cudaStream_t s) {
  using namespace step;
  int dev = 0, sms = 0;
  const int rc = sm_count(&dev, &sms);
  if (rc != UPLIFT_LA_OK) return rc;
  Params p = {};
  p.q = a.q; p.k = a.k; p.v = a.v; p.out = a.out;
  p.lse = a.lse;
  p.pk = a.pk;
  p.Hq = a.Hq; p.Hk = a.Hk; p.group = a.Hq / a.Hk; p.D = a.D;
  p.row_tiles = (p.group + kRows - 1) / kRows;
  p.chunks = chunks_for(a.pk.T, p.group, a.Hk);
  p.part_o = static_cast<float*>(workspace);
  p.part_ml = reinterpret_cast<float2*>(p.part_o + (int64_t)a.pk.T * p.chunks * a.Hq * a.D);
  p.scale = a.scale;
  // Keys per item so that the items fill the SMs about four times, within 64
  // (the four warps once) and 512 (where the join costs 3 % of the reads).
  const int64_t pairs = a.pk.B > 0 ? (int64_t)a.pk.T * a.pk.S / a.pk.B * a.Hk * p.row_tiles : 0;
  const int64_t len = pairs / ((int64_t)sms * kCtasPerSm * 4);
  p.min_len = (int)std::min<int64_t>(512, std::max<int64_t>(kMinChunk, (len + kMinChunk - 1) / kMinChunk * kMinChunk));
  if (a.dtype == UPLIFT_LA_BF16)
    return a.D <= 64 ? run<__nv_bfloat16, 64>(p, sms, s) : run<__nv_bfloat16, 128>(p, sms, s);
  return a.D <= 64 ? run<__half, 64>(p, sms, s) : run<__half, 128>(p, sms, s);
}

}  // namespace tok
}  // namespace ula
