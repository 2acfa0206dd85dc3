// Attention of few queries per sequence on long key ranges -- the step of
// one new token per sequence -- for bf16 / fp16, D <= 128.
//
// Each key and value is read once and meets only the Hq / Hk queries of its
// group, so HBM bounds it: the kernel is built to keep loads in flight with
// few instructions.  The keys of a sequence are cut into chunks; an item is
// one chunk for (up to) eight query rows -- the heads of a group, token after
// token -- which are the N of mma.m16n8k16 (fewer are padded, more make
// further items, so several tokens read the keys once as long as they and
// their heads are eight).  The
// CTA's four warps take 16 keys in turn, each with its own running maximum
// and sum, and everything is transposed, so that the few heads are the short
// side of the products:
//
//   S^T[16 keys x 8] = K Q^T,  P = exp2((S - m) scale log2 e),
//   O^T[D x 8] += V^T P^T
//
// K and V go from global memory straight into the registers of the MMA
// fragments, 16 bytes per load: the order of the channels in a product does
// not matter, so a lane takes 8 neighbouring channels of a key as its part of
// two k-steps of K (Q is laid out alike), and 8 neighbouring channels of four
// keys of V as its rows of four m-tiles (pairs of keys are merged by byte
// permutes).  P^T changes from accumulator to operand layout with movmatrix.
// V is loaded while the scores are formed, the next K while the weights are.
// The maximum is shared between a warp's lanes only when one of them saw it
// grow by more than 2^8.  The warps' results are joined in shared memory; the
// chunks' results go to a workspace and a second kernel joins them, unless
// the token has one chunk only.
//
// 64 tokens on up to 8192 keys each (762 MB), 32 heads on 8 of 128, bf16: 135
// us, 5.6 TB/s, 0.86 of a copy; on 8192 keys each 333 us, 6.45 TB/s, 0.99.  4
// tokens on up to 1500 keys: 13 us on the device for both kernels, where the
// reads take 3: launches and the length of one chunk.

#include <math.h>

#include <algorithm>
#include <atomic>
#include <type_traits>

#include "tok_attn_tc.h"

namespace ula {
namespace tok {
namespace step {

constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
constexpr int kKeys = 16;          // keys of a warp at a time
constexpr int kRows = 8;           // query rows of an item
constexpr int kMinChunk = kWarps * kKeys;
constexpr int kMaxChunks = 128;    // of one token
constexpr int kCtasPerSm = 3;      // 168 registers a thread; with 4 (128) or 2 the large steps are 1.5 and 1.2 times slower
constexpr int kManyKeys = 1024;    // keys of an item of a large problem
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kRescale = 8.f;    // see tok_attn_fwd.cu

struct Params {
  Rows q, k, v, out, out_lo;  // out_lo.p: null if not wanted
  float* lse;
  float* part_o;   // [T][chunks][Hq][D]
  float2* part_ml; // [T][chunks][Hq]: maximum (of scale S log2 e) and sum
  Packing pk;
  int Hq, Hk, group, D;
  float units;     // row tiles of a key head over all sequences, about
  int chunks;      // at most, per token
  float share;     // of the pairs of one head, that an item takes to fill the SMs once; 0: items of kManyKeys
  float scale;
};

__device__ __forceinline__ int row_tiles(const Params& p, int nq) { return (nq * p.group + kRows - 1) / kRows; }

// Row tiles times keys of a small batch (whole warp); 0 for a large one.
__device__ __forceinline__ float pairs_of(const Params& p) {
  if (p.pk.B > 32 || p.share == 0.f) return 0.f;
  float n = 0.f;
  if ((int)(threadIdx.x & 31) < p.pk.B) {
    const Seq s = sequence(p.pk, threadIdx.x & 31);
    n = (float)row_tiles(p, s.nq) * (float)s.nk;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) n += __shfl_xor_sync(0xffffffffu, n, o);
  return n;
}

// Keys of a chunk of a sequence, a multiple of kMinChunk.  The items of a
// small problem fill the SMs once, those of a large one (half as many tokens
// times key heads as CTAs) have 1024 keys: the join costs 2 % of the reads
// (512: 8 % slower).  What counts are the keys there are, not the cache's
// room (4 tokens with 1000 keys each, 32 on 8 heads of 128, in room for 32768:
// 14.4 us, by the room 26.8; in room for 1000: 13.0 and 12.4).  Batches of
// more than 32 sequences are taken to be like the one at hand.
__device__ __forceinline__ int chunk_len(const Params& p, float pairs, int nk) {
  if (p.pk.B > 32) pairs = p.units * (float)nk;
  const int fill = p.share == 0.f ? kManyKeys : (int)fminf((float)kManyKeys, pairs * p.share);
  const int even = (nk + p.chunks - 1) / p.chunks;  // the workspace holds that many
  return (max(max(fill, even), 1) + kMinChunk - 1) / kMinChunk * kMinChunk;
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

// Lanes with the same t (lane & 3): the keys of two heads.
__device__ __forceinline__ float keys_max(float v) {
  v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 4));
  v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 8));
  return fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 16));
}
__device__ __forceinline__ float keys_sum(float v) {
  v += __shfl_xor_sync(0xffffffffu, v, 4);
  v += __shfl_xor_sync(0xffffffffu, v, 8);
  return v + __shfl_xor_sync(0xffffffffu, v, 16);
}
// Four channels of a result; out_lo: what the rounding left.
template <typename T>
__device__ __forceinline__ void store_out(const Params& p, int64_t row, int h, int c, float4 x) {
  const uint32_t y[2] = {St<T>::pack(x.x, x.y), St<T>::pack(x.z, x.w)};
  *reinterpret_cast<uint2*>(static_cast<T*>(const_cast<void*>(p.out.p)) + row * p.out.t + (int64_t)h * p.out.h + c) =
      make_uint2(y[0], y[1]);
  if (p.out_lo.p == nullptr) return;
  const float2 a = St<T>::unpack(y[0]), b = St<T>::unpack(y[1]);
  *reinterpret_cast<uint2*>(static_cast<T*>(const_cast<void*>(p.out_lo.p)) + row * p.out_lo.t + (int64_t)h * p.out_lo.h + c) =
      make_uint2(St<T>::pack(isfinite(a.x) ? x.x - a.x : 0.f, isfinite(a.y) ? x.y - a.y : 0.f),
                 St<T>::pack(isfinite(b.x) ? x.z - b.x : 0.f, isfinite(b.y) ? x.w - b.y : 0.f));
}

// Loads that are not kept in L1: every byte is used once.
__device__ __forceinline__ uint4 load16(const void* p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}
__device__ __forceinline__ uint4 load16_if(const void* p, bool there) {  // zeros if not there; no branch
  uint4 v;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.u32 p, %5, 0;\n\t"
      "mov.u32 %0, 0;\n\tmov.u32 %1, 0;\n\tmov.u32 %2, 0;\n\tmov.u32 %3, 0;\n\t"
      "@p ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];\n\t}\n"
      : "=&r"(v.x), "=&r"(v.y), "=&r"(v.z), "=&r"(v.w)
      : "l"(p), "r"((uint32_t)there));
  return v;
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t v) {
  uint32_t d;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(v));
  return d;
}

// Units of a sequence: one per row tile and chunk of its keys.
struct UnitWalk {
  float pairs;
  int b0 = 0;
  int64_t before = 0;
  __device__ __forceinline__ explicit UnitWalk(const Params& p) : pairs(pairs_of(p)) {}
  __device__ __forceinline__ bool find(const Params& p, int64_t unit, Seq* s, int* len, int* local) {
    const int lane = threadIdx.x & 31;
    while (b0 < p.pk.B) {
      Seq mine{};
      int l = kMinChunk;
      int64_t n = 0;
      if (b0 + lane < p.pk.B) {
        mine = sequence(p.pk, b0 + lane);
        l = chunk_len(p, pairs, mine.nk);
        n = (int64_t)row_tiles(p, mine.nq) * ((mine.nk + l - 1) / l);
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

// FULL: D == DP, no channel is missing.
template <typename T, int DP, bool FULL>
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
  UnitWalk walk(p);
  for (int64_t i = blockIdx.x;; i += gridDim.x) {
    Seq s;
    int len, local;
    const int64_t unit = i / p.Hk;
    if (!walk.find(p, unit, &s, &len, &local)) break;
    const int hk = (int)(i - unit * p.Hk);
    const int chunks = (s.nk + len - 1) / len;
    const int tile = local / chunks, chunk = local - tile * chunks;
    // rows f0 .. of the nq x group of the sequence: token f / group, head f % group
    const int f0 = tile * kRows, rows = min(kRows, s.nq * p.group - f0);
    auto token = [&](int r) { return (f0 + min(r, rows - 1)) / p.group; };
    auto head = [&](int r) { return hk * p.group + (f0 + r) % p.group; };
    const int first_tok = token(0), last_tok = token(rows - 1);
    const int j0 = chunk * len, j1 = min(keys_seen(s, last_tok, p.pk.causal), j0 + len);
    if (j0 >= j1) continue;  // these rows see none of the chunk (the whole CTA skips it)
    // keys that all of the rows see, and those of rows 2t, 2t + 1
    const int every = min(keys_seen(s, first_tok, p.pk.causal), j1);
    const int lim[2] = {min(keys_seen(s, token(2 * t), p.pk.causal), j1), min(keys_seen(s, token(2 * t + 1), p.pk.causal), j1)};
    const int gtok = token(g);
    // Q^T: row g, 8 channels of each block of 32
    uint32_t qb[KB][4];
#pragma unroll
    for (int b = 0; b < KB; ++b) {
      const int c = 32 * b + 8 * t;
      const uint4 v = load16_if(static_cast<const T*>(p.q.p) + (int64_t)(s.q0 + gtok) * p.q.t + (int64_t)head(g) * p.q.h + c, g < rows && c < p.D);
      qb[b][0] = v.x; qb[b][1] = v.y; qb[b][2] = v.z; qb[b][3] = v.w;
    }
    // keys j + g, j + 8 + g of K, and j + 2t, + 2t + 1, + 2t + 8, + 2t + 9 of V
    int j = j0 + warp * kKeys;
    const int64_t k8 = 8 * p.k.t, k_step = (int64_t)kMinChunk * p.k.t, v_step = (int64_t)kMinChunk * p.v.t;
    const T* kp = static_cast<const T*>(p.k.p) + (int64_t)(s.k0 + j + g) * p.k.t + (int64_t)hk * p.k.h + 8 * t;
    const T* vp = static_cast<const T*>(p.v.p) + (int64_t)(s.k0 + j + 2 * t) * p.v.t + (int64_t)hk * p.v.h + 8 * g;
    uint4 kr[KB][2], vr[VB][4];
    auto load_k = [&](int jj) {
      const bool whole = jj + kKeys <= j1;
#pragma unroll
      for (int u = 0; u < 2; ++u) {
#pragma unroll
        for (int b = 0; b < KB; ++b) {
          const T* at = kp + u * k8 + 32 * b;
          if (FULL && whole) kr[b][u] = load16(at);
          else kr[b][u] = load16_if(at, jj + 8 * u + g < j1 && (FULL || 32 * b + 8 * t < p.D));
        }
      }
      kp += k_step;
    };
    auto load_v = [&](int jj) {
      const bool whole = jj + kKeys <= j1;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int key = (e & 1) + 8 * (e >> 1);
#pragma unroll
        for (int b = 0; b < VB; ++b) {
          const T* at = vp + key * p.v.t + 64 * b;
          if (FULL && whole) vr[b][e] = load16(at);
          else vr[b][e] = load16_if(at, jj + 2 * t + key < j1 && (FULL || 64 * b + 8 * g < p.D));
        }
      }
      vp += v_step;
    };
    float acc[VB][4][4], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};  // rows 2t, 2t + 1
#pragma unroll
    for (int b = 0; b < VB; ++b) {
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[b][e][0] = acc[b][e][1] = acc[b][e][2] = acc[b][e][3] = 0.f;
    }
    if (j < j1) load_k(j);
#pragma unroll 1
    for (; j < j1; j += kMinChunk) {
      load_v(j);
      float sc[4] = {0.f, 0.f, 0.f, 0.f};  // key g: rows 2t, 2t + 1; key g + 8: the same
#pragma unroll
      for (int b = 0; b < KB; ++b) {
        const uint32_t a0[4] = {kr[b][0].x, kr[b][1].x, kr[b][0].y, kr[b][1].y};
        const uint32_t a1[4] = {kr[b][0].z, kr[b][1].z, kr[b][0].w, kr[b][1].w};
        Mma<T>::run(sc, a0, qb[b][0], qb[b][1]);
        Mma<T>::run(sc, a1, qb[b][2], qb[b][3]);
      }
      if (j + kMinChunk < j1) load_k(j + kMinChunk);
      const bool part = j + kKeys > every;
      if (part) {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (j + g + 8 * (e >> 1) >= lim[e & 1]) sc[e] = -INFINITY;
      }
      const float mx[2] = {fmaxf(sc[0], sc[2]) * c2, fmaxf(sc[1], sc[3]) * c2};
      if (__any_sync(0xffffffffu, mx[0] - m[0] > kRescale || mx[1] - m[1] > kRescale)) {  // also from m = -inf
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const float mn = fmaxf(m[h], keys_max(mx[h]));
          const float f = mn == -INFINITY ? 1.f : ex2(m[h] - mn);
          m[h] = mn;
          l[h] *= f;
#pragma unroll
          for (int b = 0; b < VB; ++b) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              acc[b][e][h] *= f;
              acc[b][e][2 + h] *= f;
            }
          }
        }
      }
      const float mm[2] = {m[0] == -INFINITY ? 0.f : -m[0], m[1] == -INFINITY ? 0.f : -m[1]};
      float w[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) w[e] = ex2(fmaf(sc[e], c2, mm[e & 1]));
      l[0] += w[0] + w[2];
      l[1] += w[1] + w[3];
      const uint32_t p0 = transpose8x8(St<T>::pack(w[0], w[1]));  // row g, keys 2t, 2t + 1
      const uint32_t p1 = transpose8x8(St<T>::pack(w[2], w[3]));  // keys 2t + 8, 2t + 9
      auto add = [&](auto all, bool keep0, bool keep1) {  // to all rows, or to those of 2t, 2t + 1 that are kept
#pragma unroll
        for (int b = 0; b < VB; ++b) {
          const uint32_t x[4][4] = {{vr[b][0].x, vr[b][0].y, vr[b][0].z, vr[b][0].w}, {vr[b][1].x, vr[b][1].y, vr[b][1].z, vr[b][1].w},
                                    {vr[b][2].x, vr[b][2].y, vr[b][2].z, vr[b][2].w}, {vr[b][3].x, vr[b][3].y, vr[b][3].z, vr[b][3].w}};
#pragma unroll
          for (int e = 0; e < 4; ++e) {  // rows g, g + 8 of the tile: channels 8g + 2e, 8g + 2e + 1
            const uint32_t a[4] = {__byte_perm(x[0][e], x[1][e], 0x5410), __byte_perm(x[0][e], x[1][e], 0x7632),
                                   __byte_perm(x[2][e], x[3][e], 0x5410), __byte_perm(x[2][e], x[3][e], 0x7632)};
            if constexpr (decltype(all)::value) {
              Mma<T>::run(acc[b][e], a, p0, p1);
            } else {
              float d[4] = {acc[b][e][0], acc[b][e][1], acc[b][e][2], acc[b][e][3]};
              Mma<T>::run(d, a, p0, p1);
#pragma unroll
              for (int u = 0; u < 4; ++u)
                if (u & 1 ? keep1 : keep0) acc[b][e][u] = d[u];
            }
          }
        }
      };
      if (part && every < j1) {
        // A value that a token does not see may be an infinity or NaN: from
        // the last token back, each with the values that it sees.
#pragma unroll 1
        for (int tok = last_tok; tok >= first_tok; --tok) {
          const int see = keys_seen(s, tok, p.pk.causal);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            if (j + 2 * t + (e & 1) + 8 * (e >> 1) < see) continue;
#pragma unroll
            for (int b = 0; b < VB; ++b) vr[b][e] = make_uint4(0, 0, 0, 0);
          }
          add(std::false_type{}, token(2 * t) == tok, token(2 * t + 1) == tok);
        }
      } else {
        add(std::true_type{}, true, true);
      }
    }
    // join the warps
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      l[h] = keys_sum(l[h]);
      if (g == 0) {
        s_m[warp][2 * t + h] = m[h];
        s_l[warp][2 * t + h] = l[h];
      }
      if (2 * t + h < rows) {
#pragma unroll
        for (int b = 0; b < VB; ++b) {
          float* o = &s_o[warp][2 * t + h][64 * b + 8 * g];
          *reinterpret_cast<float4*>(o) = make_float4(acc[b][0][h], acc[b][0][2 + h], acc[b][1][h], acc[b][1][2 + h]);
          *reinterpret_cast<float4*>(o + 4) = make_float4(acc[b][2][h], acc[b][2][2 + h], acc[b][3][h], acc[b][3][2 + h]);
        }
      }
    }
    __syncthreads();
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
      const int h = head(rr), tok = token(rr);
      const int64_t row = s.q0 + tok;
      const int see = keys_seen(s, tok, p.pk.causal);
      if (j0 >= see) continue;  // the join does not look for it
      if (see <= len) {  // the token's only chunk
        const float inv = sum == 0.f ? 0.f : 1.f / sum;
        if (sum == 0.f) o = make_float4(0.f, 0.f, 0.f, 0.f);
        store_out<T>(p, row, h, c, make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv));
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
  const float pairs = pairs_of(p);
  if (live && p.pk.B > 0) {
    const Seq s = sequence(p.pk, sequence_of(p.pk.cu_q, p.pk.B, (int)row));
    if (row >= s.q0 && row < s.q0 + s.nq) {
      const int see = keys_seen(s, (int)row - s.q0, p.pk.causal), len = chunk_len(p, pairs, s.nk);
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
    store_out<T>(p, row, h, c, make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv));
  if (lane == 0 && p.lse != nullptr)
    p.lse[(int64_t)h * p.pk.T + row] = sum == 0.f ? -INFINITY : mm / kLog2e + logf(sum);
}

// Chunks per token, at most: enough that the items fill the SMs several
// times over, so that sequences of different lengths even out.  Many tokens do
// that with a chunk each; one history far longer than the others is then walked
// by a CTA per key head (500 tokens on 500 keys and one on 65536: 1547 us, apart
// 206 and 87).
int chunks_for(int64_t T, int group, int Hk) {
  const int64_t per_chunk = T * Hk * ((group + kRows - 1) / kRows);
  return (int)std::min<int64_t>(kMaxChunks, std::max<int64_t>(1, (148 * 24 + per_chunk - 1) / per_chunk));
}

template <typename T, int DP>
int run(const Params& p, int sms, cudaStream_t s) {
  const int64_t most = ((int64_t)p.pk.T * p.group / kRows + p.pk.B) * p.chunks * p.Hk;
  // a limit on the CTAs leaves SMs to other kernels, and n CTAs may be spread over n SMs
  const int budget = cta_budget(sms);
  const int grid = (int)std::min<int64_t>(most, budget < sms ? budget : sms * kCtasPerSm);
  if (p.D == DP) chunk_kernel<T, DP, true><<<grid, kThreads, 0, s>>>(p);
  else chunk_kernel<T, DP, false><<<grid, kThreads, 0, s>>>(p);
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

// Few queries per sequence: the keys are read once for every eight rows, where
// the tiles of tok_attn_fwd.cu are mostly empty.  16 sequences, this form / that
// one (us): 32 heads on 8, 8192 keys: 1 token 97 / 278, 4: 148 / 280, 8: 241 / 283,
// 16: 454 / 286; 1000 keys: 8 tokens 52 / 52; 8 heads on 8, 2000 keys: 8 tokens
// 36 / 42, 16: 56 / 42; 32 heads on 1, 2000 keys: 4 tokens 47 / 83.  The form is one
// for the whole call: a prompt of 1700 among 256 single tokens on 1000 keys makes
// it 521 us, where the two alone take 47 and 187.
bool attn_step_applies(int B, int64_t T, int group, int dtype) {
  return dtype != UPLIFT_LA_F32 && T <= 8ll * B && T <= 65536 && T * group < (1ll << 31) - 64;
}

int64_t attn_step_workspace(int64_t T, int Hq, int Hk, int D) {
  const int chunks = step::chunks_for(T, Hq / Hk, Hk);
  return chunks == 1 ? 0 : T * chunks * Hq * (D + 2) * 4;  // a token's only chunk is written at once
}

int attn_step_forward(const AttnArgs& a, void* workspace, cudaStream_t s) {
  using namespace step;
  int dev = 0, sms = 0;
  const int rc = sm_count(&dev, &sms);
  if (rc != UPLIFT_LA_OK) return rc;
  Params p = {};
  p.q = a.q; p.k = a.k; p.v = a.v; p.out = a.out; p.out_lo = a.out_lo;
  p.lse = a.lse;
  p.pk = a.pk;
  p.Hq = a.Hq; p.Hk = a.Hk; p.group = a.Hq / a.Hk; p.D = a.D;
  const int64_t tiles = std::max<int64_t>(std::min<int64_t>(a.pk.B, a.pk.T), ((int64_t)a.pk.T * p.group + kRows - 1) / kRows);
  p.units = (float)tiles;
  p.chunks = chunks_for(a.pk.T, p.group, a.Hk);
  p.part_o = static_cast<float*>(workspace);
  p.part_ml = reinterpret_cast<float2*>(p.part_o + (int64_t)a.pk.T * p.chunks * a.Hq * a.D);
  p.scale = a.scale;
  const int64_t slots = (int64_t)sms * kCtasPerSm;
  p.share = 2 * tiles * a.Hk >= slots ? 0.f : (float)a.Hk / (float)slots;
  if (a.dtype == UPLIFT_LA_BF16)
    return a.D <= 64 ? run<__nv_bfloat16, 64>(p, sms, s) : run<__nv_bfloat16, 128>(p, sms, s);
  return a.D <= 64 ? run<__half, 64>(p, sms, s) : run<__half, 128>(p, sms, s);
}

}  // namespace tok
}  // namespace ula
