// Gradients of the packed-sequence attention on the tensor cores of B200
// (sm_100a), bf16 / fp16, D <= 128.  With P = exp(scale S - lse), S = Q K^T,
//
//   dV = P^T dO,  dP = dO V^T,  dS = P (dP - delta),  delta = rowsum(dO O),
//   dQ = scale dS K,  dK = scale dS^T Q.
//
// Two passes of one kernel, each of which owns the rows it writes, so that
// no sum needs atomics and results do not depend on the order of CTAs:
//
//   KEYS:  128 keys of one key head stay, 64 queries at a time go by, over
//          all heads of the group (their sum is dK / dV):
//            S^T[128 x 64] = K Q^T,  dP^T[128 x 64] = V dO^T,
//            dV[128 x D] += P^T dO,  dK[128 x D] += dS^T Q;
//   else:  128 queries of one head stay, 64 keys at a time go by:
//            S[128 x 64] = Q K^T,    dP[128 x 64] = dO V^T,
//            dQ[128 x D] += dS K.
//
// That is 7 products where 5 would do if dQ were summed over CTAs.  In both
// passes the rows that stay (X0, X1) are the A operands of the first two
// products from shared memory, and P / dS, written over S / dP in TMEM in the
// storage type, are the A operands of the others; the tiles that go by
// (Y0, Y1) are read K-major by the first and MN-major by the second, so
// nothing is transposed or stored.  Two TMEM buffers of S and dP alternate:
// while one group of warps forms P and dS of a step the tensor cores work on
// the next.
//
// Roles (640 threads, one persistent CTA per SM): warps 0-7 and 8-15 form P
// and dS of the steps in turn (two threads per row that stays, 32 columns
// each) and store the results; warp 16 looks items up and issues TMA loads;
// warp 17 issues MMAs, and warp 19 does its waiting, so that the tensor cores
// are not idle for the length of two barrier waits per step; warp 18 (KEYS)
// fetches lse and delta of the queries that go by.
//
// The passes do not need each other.  dQ runs first; when all of its CTAs are
// running (and delta is there, which they have waited for) the other may start,
// so that its CTAs take the SMs as the first pass leaves them; it ends only
// after the first has.  Where the number of CTAs is limited, so that other
// kernels get SMs, it starts after the first has ended: both at once would be
// twice that many.
//
// P and dS are rounded to the storage type between the products.  fp16 has few
// exponents for that: dS of a large dO would overflow where dQ and dK do not,
// and that of a small one vanish.  So dS is formed of f dO and f delta, with a
// power of two f that brings the largest |dO| (the kernel that forms delta
// finds it) into 2^-5 .. 2^9, and is 1 if it is there already, so that ordinary
// gradients of one row do not depend on those of another.  P for dV is held 2^8
// times.  The factors are taken out of the fp32 sums.
//
// Rows that go by behind the end of their sequence belong to the next one:
// their P and dS are set to zero and the rows in shared memory too, since an
// infinity or NaN in them would turn the products into NaN.  The same holds in
// the steps on the causal edge, whose columns some of the rows that stay do not
// see: the groups look the tiles through before the second products, replace
// infinities and NaN by zero and put them back into the results of the rows
// that do see them.
//
// Bound by the chain of a step: scores and dP (tensor cores), P and dS (the
// warps), products with them (tensor cores), with two steps in flight, which
// for which TMEM has room (a step takes 128 columns, the sums 64 to 256; a third
// step, which would fit in all but one variant, is not built).  Six documents of
// 300 to 2500 tokens, 32 heads on 8 of 128, bf16, causal: dQ 165 us (690 TFLOP/s),
// dK and dV 196 us (770), 0.42 and 0.47 of a large library product.  16 images of
// 1025, 6 heads of 64, fp16: 73 and 97 us (a step of training 245 us).

#include <math.h>
#include <string.h>

#include <algorithm>
#include <atomic>

#include "tok_attn_tc.h"

namespace ula {

__device__ unsigned int g_tok_bwd_status;

namespace tok {
namespace bwd {

constexpr int kM = 128;   // rows that stay
constexpr int kN = 64;    // rows that go by in a step
constexpr int kThreads = 640;
constexpr int kTmemCols = 512;
constexpr int kItems = 2;
constexpr int kAux = 4;   // ring of lse / delta
constexpr uint64_t kTimeoutNs = 2000000000ull;
constexpr float kLog2e = 1.4426950408889634f;
constexpr int kHeld = 8;  // fp16: P for dV is held 2^8 times

template <int DP>
struct Cfg {
  static constexpr int kChunks = DP / 64;
  static constexpr int kXChunk = kM * 128, kYChunk = kN * 128;  // 64 channels of a tile
  static constexpr int kXBytes = kChunks * kXChunk;
  static constexpr int kYBytes = kChunks * kYChunk;
  static constexpr int kStages = DP == 128 ? 3 : 6;             // Y0 and Y1 together
  static constexpr int kOffX = 0;
  static constexpr int kOffY = 2 * kXBytes;
  static constexpr int kOffStage = kOffY + kStages * 2 * kYBytes;
  static constexpr int kStageBytes = 32 * 128;                  // a warp's 32 rows x 64 channels
  static constexpr int kOffAux = kOffStage + 16 * kStageBytes;
  static constexpr int kOffBar = kOffAux + kAux * 2 * kN * 4;
  static constexpr int kNumBars = 2 + 2 * kStages + 2 * kAux + 4 + 2 + 2 * kItems + 1;
  static constexpr int kOffMisc = kOffBar + kNumBars * 8;
  static constexpr int kOffItems = kOffMisc + 32;
  static constexpr int kSmem = kOffItems + kItems * 32;
  static_assert(kSmem <= 232448, "shared memory");
  // TMEM columns: two buffers of S and dP, then the sums
  static constexpr int kColAcc = 4 * kN;
  static_assert(kColAcc + 2 * DP <= kTmemCols, "TMEM");
};

struct Item {
  int n;       // rows that stay, 1..128; 0: no more items
  int live;    // of these, rows with a gradient (keys in use); the others get zeros
  int row;     // their first row in the tensor
  int h;       // head of the rows that stay
  int y0;      // first row that goes by (in the tensor)
  int ny;      // number of them (per head)
  int steps;   // steps of 64 of them (per head)
  int off;     // row r that stays and column c that goes by see each other, if causal, when KEYS: c >= r + off
               // at the first step (64 less at each further one); else: c < r + off (64 less ..)
};

struct Params {
  CUtensorMap x0, x1;  // rows that stay: K, V or Q, dO; box {64, 1, 128}
  CUtensorMap y0, y1;  // rows that go by: Q, dO or K, V; box {64, 1, 64}
  CUtensorMap o0, o1;  // results: dV, dK or dQ; box {64, 1, 32}
  Rows y[2];           // as y0, y1
  Rows out0, out1;
  const float* lse;
  const float* delta;
  Packing pk;
  int heads, group, D;  // heads of the rows that stay
  float scale;
  uint64_t timeout_ns;
  unsigned int* host_status;
  int test_fault;       // 1: the producer issues no loads after a few (tests the waits that run out)
  int* counter;         // items given out, beyond the first of each CTA
  const unsigned* most; // fp16: the largest |dO|, as bits of a float
};

// log2 of the factor that dO is taken times.
template <typename T>
__device__ __forceinline__ int dout_exponent(const Params& p) {
  if constexpr (St<T>::kFmt != 0) return 0;
  const int e = (int)(*p.most >> 23) - 127;
  return e == -127 ? 0 : min(max(e, -5), 8) - e;  // dO may be zero throughout
}
__device__ __forceinline__ float power_of_two(int e) { return __int_as_float((127 + e) << 23); }

__device__ __forceinline__ bool mbar_wait(uint64_t* b, uint32_t parity, volatile int* abort_flag, unsigned where,
                                          const WaitLimit& limit) {
  return mbar_wait_inline(b, parity, abort_flag, where, limit, &g_tok_bwd_status);
}

// Makes the tiles of a step (Y0, Y1) fit for the second products: rows from
// `rows` on become zero (both tiles, all channels); with `edge`, so do the
// infinities and NaN of the tiles that are multiplied (Y0, and with KEYS Y1).
// 256 threads, each its own 16-byte pieces.
template <typename T, int CHUNKS, bool KEYS>
__device__ __noinline__ void clean_step(uint8_t* y, int rows, bool edge, int tid, volatile int* cleaned) {
#pragma unroll 1
  for (int i = tid; i < 2 * CHUNKS * kN * 8; i += 256) {
    uint4* piece = reinterpret_cast<uint4*>(y) + i;
    if ((i & (kN * 8 - 1)) >= rows * 8) {
      *piece = make_uint4(0, 0, 0, 0);
    } else if (edge && (KEYS || i < CHUNKS * kN * 8)) {
      const uint4 v = *piece;
      uint32_t acc = nonfinite_probe<T>(nonfinite_probe<T>(nonfinite_probe<T>(nonfinite_probe<T>(0, v.x), v.y), v.z), v.w);
      const float2 f = St<T>::unpack(acc);
      if (f.x == 0.f && f.y == 0.f) continue;
      *cleaned = 1;
      T* e = reinterpret_cast<T*>(piece);
      for (int k = 0; k < 8; ++k)
        if (!isfinite(St<T>::f(e[k]))) e[k] = St<T>::t(0.f);
    }
  }
  fence_proxy_async();
}

// Puts what was taken out of the rows y0 .. y1 - 1 of y (the channels
// from `y` on) back into a staged row of results: weights are positive, so dV gets
// the infinity or NaN itself (`itself`); where a query or key is not finite
// neither is the score, so its weight's gradient is zero or NaN and its
// product with the value NaN.
template <typename T>
__device__ __noinline__ void put_back(uint8_t* row, int lane, const T* y, int64_t stride, int y0, int y1, int channels,
                                      bool itself) {
#pragma unroll 1
  for (int j = y0; j < y1; ++j) {
#pragma unroll 1
    for (int i = 0; i < channels; ++i) {
      const float x = St<T>::f(y[j * stride + i]);
      if (isfinite(x)) continue;
      T* e = reinterpret_cast<T*>(row + (((i >> 3) ^ (lane & 7)) << 4) + (i & 7) * 2);
      *e = St<T>::t(itself ? St<T>::f(*e) + x : __int_as_float(0x7fc00000));
    }
  }
}

template <typename T, int DP, bool KEYS>
__global__ void __launch_bounds__(kThreads, 1) gradient_kernel(const __grid_constant__ Params p) {
  using C = Cfg<DP>;
  constexpr bool kScaled = St<T>::kFmt == 0;  // fp16
  extern __shared__ __align__(1024) uint8_t smem[];
  if ((su32(smem) & 1023u) != 0) {  // the swizzled tiles need it, and the declaration asks for it
    if (threadIdx.x == 0) atomicCAS(&g_tok_bwd_status, 0u, 1u);
    return;
  }
  uint8_t* sX = smem + C::kOffX;
  uint8_t* sY = smem + C::kOffY;
  float* sAux = reinterpret_cast<float*>(smem + C::kOffAux);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + C::kOffBar);
  uint64_t* x_full = bars;
  uint64_t* x_empty = x_full + 1;
  uint64_t* y_full = x_empty + 1;             // [kStages]
  uint64_t* y_empty = y_full + C::kStages;    // [kStages]
  uint64_t* a_full = y_empty + C::kStages;    // [kAux]
  uint64_t* a_empty = a_full + kAux;          // [kAux]
  uint64_t* s_full = a_empty + kAux;          // [2] S and dP of a step
  uint64_t* p_full = s_full + 2;              // [2] P and dS of a step
  uint64_t* acc_full = p_full + 2;            // an item's sums
  uint64_t* acc_empty = acc_full + 1;
  uint64_t* item_full = acc_empty + 1;        // [kItems]
  uint64_t* item_empty = item_full + kItems;  // [kItems]
  uint64_t* drain = item_empty + kItems;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + C::kOffMisc);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + C::kOffMisc + 4);
  volatile int* cleaned = reinterpret_cast<volatile int*>(smem + C::kOffMisc + 16);  // some tile of this CTA was
  uint32_t* go = reinterpret_cast<uint32_t*>(smem + C::kOffMisc + 20);  // steps whose second products may begin
  volatile Item* items = reinterpret_cast<volatile Item*>(smem + C::kOffItems);

  const int tid = threadIdx.x;
  const int warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
  if (tid == 0) {
    mbar_init(x_full, 1);
    mbar_init(x_empty, 1);
    for (int i = 0; i < C::kStages; ++i) {
      mbar_init(&y_full[i], 1);
      mbar_init(&y_empty[i], 1);
    }
    for (int i = 0; i < kAux; ++i) {
      mbar_init(&a_full[i], 1);
      mbar_init(&a_empty[i], 8);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&s_full[i], 1);
      mbar_init(&p_full[i], 8);
    }
    mbar_init(acc_full, 1);
    mbar_init(acc_empty, 16);
    for (int i = 0; i < kItems; ++i) {
      mbar_init(&item_full[i], 1);
      mbar_init(&item_empty[i], KEYS ? 19 : 18);  // 16 warps of the groups, MMA, its forerunner, lse / delta
    }
    mbar_init(drain, 1);
    abort_flag[0] = 0;
    abort_flag[1] = 0;  // stays 0: the flag of waits that must not be aborted
    *cleaned = 0;
    *go = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 17) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(su32(tmem_slot)), "r"(kTmemCols));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  if (!KEYS) {
    asm volatile("griddepcontrol.wait;" ::: "memory");  // delta and the counters
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = __shfl_sync(0xffffffffu, *tmem_slot, 0);
  auto col_s = [&](uint32_t b) { return tmem + b * 2 * kN; };
  auto col_dp = [&](uint32_t b) { return tmem + b * 2 * kN + kN; };
  const uint32_t col_acc = tmem + C::kColAcc;
  const WaitLimit tmo{p.timeout_ns, p.host_status};
  auto wait = [&](uint64_t* bar, uint32_t parity) {
    return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag, 2, tmo));
  };
  // heads that go by per item
  const int passes = KEYS ? p.group : 1;

  if (warp == 16) {
    // ------------------------------------------------------------ producer
    if (lane == 0) {
      prefetch_map(&p.x0);
      prefetch_map(&p.x1);
      if (p.pk.T > 0 && p.pk.S > 0) {
        prefetch_map(&p.y0);
        prefetch_map(&p.y1);
      }
    }
    TileWalk walk;
    bool ok = true;
    uint32_t g = 0, nx = 0;
    for (int n = 0;; ++n) {
      // The costliest items come first, and each CTA takes the next one when
      // the loads of its last are on their way.  (Dealt out beforehand, the
      // few large items of the KEYS pass left the longest CTA with 1.5 times
      // the average over six documents.)
      int64_t i = blockIdx.x;
      if (n > 0) {
        int next = 0;
        if (lane == 0) next = atomicAdd(p.counter, 1);
        i = (int64_t)gridDim.x + __shfl_sync(0xffffffffu, next, 0);
      }
      int b = 0, local = 0, tiles = 0;
      const int64_t tile = i / p.heads;
      const bool more = tile < (1ll << 31) && walk.find(p.pk, KEYS, kM, (int)tile, &b, &local, &tiles);
      Item it{};
      if (more) {
        const Seq s = sequence(p.pk, b);
        it.h = (int)(i - tile * p.heads);
        const int shift = s.nk - s.nq;  // causal: query i sees keys <= i + shift
        if (KEYS) {
          const int seg = segment(p.pk.cu_k, b, p.pk.S).y;
          const int j0 = local * kM;
          it.row = s.k0 + j0;
          it.n = min(kM, seg - j0);
          it.live = max(0, min(it.n, s.nk - j0));
          const int i0 = p.pk.causal ? max(0, j0 - shift) : 0;
          it.y0 = s.q0 + i0;
          it.ny = it.live > 0 ? max(0, s.nq - i0) : 0;
          it.off = j0 - shift - i0;
        } else {
          const int i0 = local * kM;
          it.row = s.q0 + i0;
          it.n = min(kM, s.nq - i0);
          it.live = it.n;
          it.y0 = s.k0;
          it.ny = p.pk.causal ? max(0, min(s.nk, i0 + it.n + shift)) : s.nk;
          it.off = i0 + 1 + shift;
        }
        it.steps = (it.ny + kN - 1) / kN;
      }
      if (lane == 0) {
        const int slot = n % kItems;
        ok = mbar_wait(&item_empty[slot], ((n / kItems) & 1) ^ 1, abort_flag, 1, tmo);
        if (ok) {
          items[slot].n = it.n; items[slot].live = it.live; items[slot].row = it.row; items[slot].h = it.h;
          items[slot].y0 = it.y0; items[slot].ny = it.ny; items[slot].steps = it.steps; items[slot].off = it.off;
          mbar_arrive(&item_full[slot]);
        }
        if (ok && it.steps > 0) {
          ok = mbar_wait(x_empty, (nx & 1) ^ 1, abort_flag, 1, tmo);
          ++nx;
          if (ok) {
            mbar_expect_tx(x_full, 2 * C::kXBytes);
#pragma unroll
            for (int c = 0; c < C::kChunks; ++c) {
              load_rows(sX + c * C::kXChunk, &p.x0, x_full, 64 * c, it.h, it.row);
              load_rows(sX + C::kXBytes + c * C::kXChunk, &p.x1, x_full, 64 * c, it.h, it.row);
            }
          }
          for (int e = 0; e < passes && ok; ++e) {
            const int hy = KEYS ? it.h * p.group + e : it.h / p.group;
            for (int j = 0; j < it.steps; ++j, ++g) {
              const int s = g % C::kStages;
              ok = mbar_wait(&y_empty[s], ((g / C::kStages) & 1) ^ 1, abort_flag, 1, tmo);
              if (!ok) break;
              if (p.test_fault == 1 && g >= 3) continue;
              uint8_t* y = sY + s * 2 * C::kYBytes;
              mbar_expect_tx(&y_full[s], 2 * C::kYBytes);
#pragma unroll
              for (int c = 0; c < C::kChunks; ++c) {
                load_rows(y + c * C::kYChunk, &p.y0, &y_full[s], 64 * c, hy, it.y0 + j * kN);
                load_rows(y + C::kYBytes + c * C::kYChunk, &p.y1, &y_full[s], 64 * c, hy, it.y0 + j * kN);
              }
            }
          }
        }
      }
      ok = __shfl_sync(0xffffffffu, ok ? 1 : 0, 0) != 0;
      if (!ok || !more) break;
    }
    if (!ok) {  // let issued loads land before the CTA can exit
      const uint64_t t0 = gtimer();
      while (gtimer() - t0 < 200000ull) {}
    }
  } else if (warp == 17) {
    // ---------------------------------------------------------- MMA issuer
    constexpr uint32_t kIdS = idesc_f16(St<T>::kFmt, 0, kM, kN);
    constexpr uint32_t kIdA = idesc_f16(St<T>::kFmt, 1, kM, DP);
    const int ksteps = (p.D + 15) / 16;  // channels behind D are zero
    // descriptors: the start address counts 16 bytes in their lowest bits
    const uint64_t dx = mdesc(su32(sX), 16, 1024, kLayoutSw128), dy = mdesc(su32(sY), 16, 1024, kLayoutSw128);
    const uint64_t dyt = mdesc(su32(sY), C::kYChunk, 1024, kLayoutSw128);
    bool ok = true;
    uint32_t g = 0, nx = 0;  // steps and items with steps so far
    auto ready = [&](uint32_t gs) { return wait(&y_full[gs % C::kStages], (gs / C::kStages) & 1); };
    auto first = [&](uint32_t gs) {  // (one lane) S and dP of step gs
      const uint64_t y = dy + (gs % C::kStages) * (2 * C::kYBytes >> 4);
#pragma unroll
      for (int w = 0; w < 2; ++w) {
#pragma unroll
        for (int ks = 0; ks < DP / 16; ++ks) {
          const uint32_t c = ks >> 2, k = 32 * (ks & 3);
          if (ks < ksteps)
            tc_mma(w == 0 ? col_s(gs & 1) : col_dp(gs & 1), dx + ((w * C::kXBytes + c * C::kXChunk + k) >> 4),
                   y + ((w * C::kYBytes + c * C::kYChunk + k) >> 4), kIdS, ks > 0);
        }
      }
      tc_commit(&s_full[gs & 1]);
    };
    for (int n = 0; ok; ++n) {
      const int islot = n % kItems;
      ok = wait(&item_full[islot], (n / kItems) & 1);
      if (!ok) break;
      const int rows = items[islot].n;
      const int total = items[islot].steps * passes;
      __syncwarp();
      if (lane == 0) mbar_arrive(&item_empty[islot]);
      if (rows == 0) break;
      if (total == 0) continue;
      ok = wait(x_full, nx & 1);
      // up to two steps of first products ahead of the second ones
      for (int j = 0; j < min(2, total) && ok; ++j) {
        ok = ready(g + j);
        if (!ok) break;
        tc_fence_after();
        if (elect_one()) {
          first(g + j);
          if (j + 1 == total) tc_commit(x_empty);
        }
        __syncwarp();
      }
      ok = ok && wait(acc_empty, (nx & 1) ^ 1);
      ++nx;
      for (int j = 0; j < total && ok; ++j) {
        const uint32_t gs = g + j, b = gs & 1;
        ok = wait_raised(go, gs + 1, abort_flag, 2, tmo, &g_tok_bwd_status);
        if (!ok) break;
        tc_fence_after();
        if (elect_one()) {
          const uint64_t y = dyt + (gs % C::kStages) * (2 * C::kYBytes >> 4);
          if (KEYS) {
#pragma unroll
            for (int ks = 0; ks < kN / 16; ++ks)
              mma_tmem_a(col_acc, col_s(b) + 8 * (ks & 1) + 32 * (ks >> 1), y + ((C::kYBytes + 2048 * ks) >> 4), kIdA, (j > 0 || ks > 0) ? 1u : 0u);
          }
#pragma unroll
          for (int ks = 0; ks < kN / 16; ++ks)
            mma_tmem_a(col_acc + (KEYS ? DP : 0), col_dp(b) + 8 * (ks & 1) + 32 * (ks >> 1), y + ((2048 * ks) >> 4), kIdA, (j > 0 || ks > 0) ? 1u : 0u);
          tc_commit(&y_empty[gs % C::kStages]);
          if (j + 2 < total) first(gs + 2);
          if (j + 3 == total) tc_commit(x_empty);
          if (j + 1 == total) tc_commit(acc_full);
        }
        __syncwarp();
      }
      g += total;
    }
    // all issued MMAs complete before TMEM can be released (this wait
    // ignores the abort flag: it must not be cut short by another role)
    if (elect_one()) tc_commit(drain);
    __syncwarp();
    mbar_wait(drain, 0, abort_flag + 1, 2, tmo);
  } else if (warp == 18) {
    // ------------------------------------- lse and delta of the columns
    if (KEYS) {
      constexpr float held = kScaled ? (float)kHeld : 0.f;
      const float fd = kScaled ? power_of_two(dout_exponent<T>(p) - kHeld) : 1.f;
      bool ok = true;
      uint32_t g = 0;
      for (int n = 0; ok; ++n) {
        const int islot = n % kItems;
        ok = __all_sync(0xffffffffu, mbar_wait(&item_full[islot], (n / kItems) & 1, abort_flag, 1, tmo));
        if (!ok) break;
        const int rows = items[islot].n, h = items[islot].h, y0 = items[islot].y0, ny = items[islot].ny,
                  steps = items[islot].steps;
        __syncwarp();
        if (lane == 0) mbar_arrive(&item_empty[islot]);
        if (rows == 0) break;
        for (int e = 0; e < passes && ok; ++e) {
          const float* lse = p.lse + (int64_t)(h * p.group + e) * p.pk.T + y0;
          const float* delta = p.delta + (int64_t)(h * p.group + e) * p.pk.T + y0;
          for (int j = 0; j < steps; ++j, ++g) {
            const int s = g % kAux;
            ok = __all_sync(0xffffffffu, mbar_wait(&a_empty[s], ((g / kAux) & 1) ^ 1, abort_flag, 1, tmo));
            if (!ok) break;
#pragma unroll
            for (int c = 0; c < kN; c += 32) {
              const int i = j * kN + c + lane;
              float l = -INFINITY, d = 0.f;
              if (i < ny) {
                l = lse[i];
                d = delta[i];
              }
              // negated, in powers of two; rows without keys: P = 0
              sAux[s * 2 * kN + c + lane] = l == -INFINITY ? -INFINITY : held - l * kLog2e;
              sAux[s * 2 * kN + kN + c + lane] = -d * fd;
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(&a_full[s]);
          }
        }
      }
    }
  } else if (warp == 19) {
    // --------------------------------- forerunner of the MMA issuer: waits
    // for what a step needs (P and dS, the tiles of the step after next) and
    // raises a counter
    bool ok = true;
    uint32_t g = 0;
    for (int n = 0; ok; ++n) {
      const int islot = n % kItems;
      ok = wait(&item_full[islot], (n / kItems) & 1);
      if (!ok) break;
      const int rows = items[islot].n;
      const int total = items[islot].steps * passes;
      __syncwarp();
      if (lane == 0) mbar_arrive(&item_empty[islot]);
      if (rows == 0) break;
      for (int j = 0; j < total && ok; ++j, ++g) {
        ok = (j + 2 >= total || wait(&y_full[(g + 2) % C::kStages], ((g + 2) / C::kStages) & 1)) &&
             wait(&p_full[g & 1], (g >> 1) & 1);
        if (ok && lane == 0) raise_to(go, g + 1);
      }
    }
  } else {
    // ------------------------------------------------------------ P and dS
    const int w = warp >> 3, half = (warp >> 2) & 1, q = warp & 3;
    const int r = 32 * q + lane;  // row that stays = TMEM lane
    const uint32_t lane_off = (uint32_t)(32 * q) << 16;
    const float c2 = p.scale * kLog2e;
    const int fexp = dout_exponent<T>(p);
    const float fdp = kScaled && KEYS ? power_of_two(fexp - kHeld) : 1.f;  // of dP; without KEYS the weights take it
    uint8_t* stage = smem + C::kOffStage + warp * C::kStageBytes;
    uint32_t g = 0, na = 0;
    bool ok = true;
    for (int n = 0; ok; ++n) {
      const int islot = n % kItems;
      ok = __all_sync(0xffffffffu, mbar_wait(&item_full[islot], (n / kItems) & 1, abort_flag, 3, tmo));
      if (!ok) break;
      Item it;
      it.n = items[islot].n; it.live = items[islot].live; it.row = items[islot].row; it.h = items[islot].h;
      it.ny = items[islot].ny; it.steps = items[islot].steps; it.off = items[islot].off; it.y0 = items[islot].y0;
      __syncwarp();
      if (lane == 0) mbar_arrive(&item_empty[islot]);
      if (it.n == 0) break;
      const int total = it.steps * passes;
      // steps edge0 .. edge1 - 1 (of a head) hold columns that some row does not see
      int edge0 = 0, edge1 = 0;
      if (p.pk.causal) {
        if (KEYS) edge1 = (max(0, it.live - 1 + it.off) + kN - 1) / kN;
        else if (it.off < it.ny) edge0 = max(0, it.off) / kN, edge1 = it.steps;
      }
      float nlse = 0.f, ndelta = 0.f;
      if (!KEYS) {
        nlse = -INFINITY;
        if (r < it.n) {
          const int64_t at = (int64_t)it.h * p.pk.T + it.row + r;
          const float l = p.lse[at];
          nlse = l == -INFINITY ? -INFINITY : (kScaled ? (float)fexp - l * kLog2e : -l * kLog2e);
          ndelta = -p.delta[at];
        }
      }
      int j = 0;  // step within the head
      for (int k = 0; k < total && ok; ++k, j = j + 1 == it.steps ? 0 : j + 1) {
        const uint32_t gs = g + k;
        if ((gs & 1) != (uint32_t)w) continue;
        ok = __all_sync(0xffffffffu, mbar_wait(&s_full[w], (gs >> 1) & 1, abort_flag, 3, tmo));
        if (KEYS) ok = ok && __all_sync(0xffffffffu, mbar_wait(&a_full[gs % kAux], (gs / kAux) & 1, abort_flag, 3, tmo));
        if (!ok) break;
        tc_fence_after();
        const float* aux = sAux + (gs % kAux) * 2 * kN;
        // columns lo .. hi - 1 are seen
        int lo = 0, hi = it.ny - j * kN;
        if (p.pk.causal) {
          if (KEYS) lo = r + it.off - j * kN;
          else hi = min(hi, r + it.off - j * kN);
        }
        const bool masked = __any_sync(0xffffffffu, lo > 0 || hi < kN);
        constexpr int kCols = kN / 2;  // of this thread: columns kCols * half ..
        const uint32_t ts = col_s(w) + kCols * half + lane_off, td = col_dp(w) + kCols * half + lane_off;
#pragma unroll
        for (int c = 0; c < kCols; c += 16) {
          uint32_t s[16], d[16];
          tc_ld16(ts + c, s);
          tc_ld16(td + c, d);
          tc_wait_ld_regs16(s);
          tc_wait_ld_regs16(d);
          float* fs = reinterpret_cast<float*>(s);
          float* fd = reinterpret_cast<float*>(d);
          const float2 c22 = make_float2(c2, c2);
#pragma unroll
          for (int e = 0; e < 16; e += 4) {
            float4 nl = make_float4(nlse, nlse, nlse, nlse), nd = make_float4(ndelta, ndelta, ndelta, ndelta);
            if (KEYS) {
              nl = *reinterpret_cast<const float4*>(aux + kCols * half + c + e);
              nd = *reinterpret_cast<const float4*>(aux + kN + kCols * half + c + e);
            }
            const float2 x0 = __ffma2_rn(make_float2(fs[e], fs[e + 1]), c22, make_float2(nl.x, nl.y));
            const float2 x1 = __ffma2_rn(make_float2(fs[e + 2], fs[e + 3]), c22, make_float2(nl.z, nl.w));
            const float2 p0 = make_float2(ex2(x0.x), ex2(x0.y)), p1 = make_float2(ex2(x1.x), ex2(x1.y));
            auto less = [&](float2 dp, float2 d) { return kScaled && KEYS ? __ffma2_rn(dp, make_float2(fdp, fdp), d) : __fadd2_rn(dp, d); };
            const float2 d0 = __fmul2_rn(p0, less(make_float2(fd[e], fd[e + 1]), make_float2(nd.x, nd.y)));
            const float2 d1 = __fmul2_rn(p1, less(make_float2(fd[e + 2], fd[e + 3]), make_float2(nd.z, nd.w)));
            fs[e] = p0.x; fs[e + 1] = p0.y; fs[e + 2] = p1.x; fs[e + 3] = p1.y;
            fd[e] = d0.x; fd[e + 1] = d0.y; fd[e + 2] = d1.x; fd[e + 3] = d1.y;
          }
          if (masked) {
#pragma unroll
            for (int e = 0; e < 16; ++e) {
              const int col = kCols * half + c + e;
              const bool seen = col >= lo && col < hi;
              fs[e] = seen ? fs[e] : 0.f;
              fd[e] = seen ? fd[e] : 0.f;
            }
          }
          uint32_t ps[8], ds[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            ps[e] = St<T>::pack(fs[2 * e], fs[2 * e + 1]);
            ds[e] = St<T>::pack(fd[2 * e], fd[2 * e + 1]);
          }
          // over columns that have been read
          if (KEYS) tmem_st8(ts + c / 2, ps);
          tmem_st8(td + c / 2, ds);
        }
        const int rows = it.ny - j * kN;  // of the tile that goes by
        const bool edge = j >= edge0 && j < edge1;
        if (edge || rows < kN)  // rows of the next sequence; infinities and NaN that some row does not see
          clean_step<T, C::kChunks, KEYS>(sY + (gs % C::kStages) * 2 * C::kYBytes, rows, edge, tid & 255, cleaned);
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          if (KEYS) mbar_arrive(&a_empty[gs % kAux]);
          mbar_arrive(&p_full[w]);
        }
      }
      if (!ok) break;
      g += total;
      // ---------------------------------------------------------- results
      if (total > 0) {
        ok = __all_sync(0xffffffffu, mbar_wait(acc_full, na & 1, abort_flag, 4, tmo));
        if (!ok) break;
        ++na;
        tc_fence_after();
      }
      // KEYS: warps 0-7 store dV, 8-15 dK, a chunk of 64 channels for each half;
      // else the first halves store a chunk of dQ each
      const CUtensorMap* map = KEYS && w == 1 ? &p.o1 : &p.o0;
      const Rows& out = KEYS && w == 1 ? p.out1 : p.out0;
      const float f = KEYS && w == 0 ? (kScaled ? power_of_two(-kHeld) : 1.f) : (kScaled ? p.scale * power_of_two(-fexp) : p.scale);
      const int c = KEYS ? half : (half == 0 ? w : C::kChunks);
      const int wrows = min(32, it.n - 32 * q);
      if (c < C::kChunks && 64 * c < p.D) {
        const uint32_t src = col_acc + lane_off + (KEYS && w == 1 ? DP : 0) + 64 * c;
        const bool zero = total == 0 || r >= it.live;
        if (lane == 0) bulk_wait_read0();  // the staging buffer is free
        __syncwarp();
        uint8_t* row = stage + lane * 128;
#pragma unroll 1
        for (int h = 0; h < 2; ++h) {
          uint32_t o[32];
          if (total > 0) {
            tc_ld32(src + 32 * h, o);
            tc_wait_ld_regs(o);
          }
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            float x[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = zero ? 0.f : __uint_as_float(o[8 * e + i]) * f;
            *reinterpret_cast<uint4*>(row + (((4 * h + e) ^ (lane & 7)) << 4)) =
                make_uint4(St<T>::pack(x[0], x[1]), St<T>::pack(x[2], x[3]), St<T>::pack(x[4], x[5]), St<T>::pack(x[6], x[7]));
          }
        }
        if (*cleaned != 0 && !zero) {
          const Rows& y = p.y[KEYS && w == 0 ? 1 : 0];  // dV takes dO, dK and dQ take queries and keys
          const int from = KEYS ? max(0, r + it.off) : edge0 * kN;
          const int to = min(min(it.ny, edge1 * kN), KEYS ? it.ny : r + it.off);
          for (int e = 0; e < passes; ++e) {
            const int hy = KEYS ? it.h * p.group + e : it.h / p.group;
            put_back<T>(row, lane, static_cast<const T*>(y.p) + (int64_t)it.y0 * y.t + (int64_t)hy * y.h + 64 * c, y.t,
                        from, to, min(64, p.D - 64 * c), KEYS && w == 0);
          }
        }
        fence_proxy_async();
        __syncwarp();
        const int row0 = it.row + 32 * q;
        if (wrows == 32) {
          if (lane == 0) {
            tma_store(map, stage, 64 * c, it.h, row0, 0);
            bulk_commit();
          }
        } else {  // the rows behind the sequence are not ours
          for (int e = lane; e < wrows * 8; e += 32) {
            const int rr = e >> 3, piece = e & 7;
            if (64 * c + 8 * piece < p.D)
              *reinterpret_cast<uint4*>(static_cast<T*>(const_cast<void*>(out.p)) + (int64_t)(row0 + rr) * out.t +
                                        (int64_t)it.h * out.h + 64 * c + 8 * piece) =
                  *reinterpret_cast<const uint4*>(stage + rr * 128 + ((piece ^ (rr & 7)) << 4));
          }
          __syncwarp();
        }
      }
      if (total > 0) {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(acc_empty);
      }
    }
    // rows of no sequence: zeros
    const int rows = KEYS ? p.pk.S : p.pk.T;
    const int32_t* cu = KEYS ? p.pk.cu_k : p.pk.cu_q;
    int lo = 0, hi = 0;
    if (p.pk.B > 0) {
      lo = segment(cu, 0, rows).x;
      const int2 e = segment(cu, p.pk.B - 1, rows);
      hi = max(lo, e.x + e.y);
    }
    const int64_t gap = (int64_t)lo + (rows - hi);
    for (int64_t i = (int64_t)blockIdx.x * 16 + warp; i < gap * p.heads; i += (int64_t)gridDim.x * 16) {
      const int64_t k = i / p.heads;
      const int h = (int)(i - k * p.heads);
      const int64_t row = k < lo ? k : hi + (k - lo);
      for (int e = lane * 8; e < p.D; e += 256) {
        *reinterpret_cast<uint4*>(static_cast<T*>(const_cast<void*>(p.out0.p)) + row * p.out0.t + (int64_t)h * p.out0.h + e) =
            make_uint4(0, 0, 0, 0);
        if (KEYS)
          *reinterpret_cast<uint4*>(static_cast<T*>(const_cast<void*>(p.out1.p)) + row * p.out1.t + (int64_t)h * p.out1.h + e) =
              make_uint4(0, 0, 0, 0);
      }
    }
    if (lane == 0) bulk_wait_all();
  }

  if (KEYS) asm volatile("griddepcontrol.wait;" ::: "memory");  // what follows this pass follows the other one too
  tc_fence_before();
  __syncthreads();
  if (warp == 17) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemCols));
  }
}

// delta = rowsum(dO O): eight lanes per row, 16 bytes each at a time.  O is
// taken as out + out_lo: the rounding of out alone would be the largest error
// of dS in rows that see few keys.  Bound by HBM: 29 us for the three tensors
// of 5986 tokens of 32 heads of 128 in bf16 (147 MB, 5.1 TB/s); in fp16 the search
// for the largest |dO| takes 3 of 12 us for 16400 tokens of 6 heads of 64.
// Also sets the item counters of the passes that follow to zero, and with
// fp16 finds the largest |dO| in the rows of the sequences (most, zero before
// the launch; 16-byte pieces with an infinity or NaN do not count).
template <typename T>
__global__ void __launch_bounds__(256) delta_kernel(Rows dout, Rows out, Rows lo, float* delta, int* counters, unsigned* most, Packing pk,
                                                    int Hq, int D) {
  const int T_ = pk.T;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  if (blockIdx.x == 0 && threadIdx.x < 2) counters[threadIdx.x] = 0;
  const int64_t item = (int64_t)blockIdx.x * 32 + threadIdx.x / 8;
  const int l = threadIdx.x & 7;
  __shared__ unsigned top;
  int first = 0, end = 0;  // rows of the sequences
  unsigned big = 0;        // bits of two |dO|
  if (St<T>::kFmt == 0) {
    if (threadIdx.x == 0) top = 0;
    if (pk.B > 0) {
      const int2 last = segment(pk.cu_q, pk.B - 1, T_);
      first = segment(pk.cu_q, 0, T_).x;
      end = last.x + last.y;
    }
    __syncthreads();
  }
  float sum = 0.f;
  const bool live = item < (int64_t)T_ * Hq;
  const int64_t t = live ? item / Hq : 0;
  const int h = live ? (int)(item - t * Hq) : 0;
  if (live) {
    const T* g = static_cast<const T*>(dout.p) + t * dout.t + (int64_t)h * dout.h;
    const T* o = static_cast<const T*>(out.p) + t * out.t + (int64_t)h * out.h;
    for (int c = l * 8; c < D; c += 64) {
      const uint4 a = *reinterpret_cast<const uint4*>(g + c), b = *reinterpret_cast<const uint4*>(o + c);
      const uint32_t ua[4] = {a.x, a.y, a.z, a.w}, ub[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 x = St<T>::unpack(ua[i]), y = St<T>::unpack(ub[i]);
        sum = fmaf(x.x, y.x, fmaf(x.y, y.y, sum));
      }
      if (St<T>::kFmt == 0) {
        unsigned m = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) m = __vmaxu2(m, ua[i] & 0x7fff7fffu);
        if (max(m & 0xffffu, m >> 16) < 0x7c00u) big = __vmaxu2(big, m);
      }
      if (lo.p != nullptr) {
        const uint4 d = *reinterpret_cast<const uint4*>(static_cast<const T*>(lo.p) + t * lo.t + (int64_t)h * lo.h + c);
        const uint32_t ud[4] = {d.x, d.y, d.z, d.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float2 x = St<T>::unpack(ua[i]), y = St<T>::unpack(ud[i]);
          sum = fmaf(x.x, y.x, fmaf(x.y, y.y, sum));
        }
      }
    }
  }
#pragma unroll
  for (int o = 4; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if (live && l == 0) delta[(int64_t)h * T_ + t] = sum;
  if (St<T>::kFmt == 0) {
    const unsigned bits = t >= first && t < end ? max(big & 0xffffu, big >> 16) : 0;
    const unsigned of_warp = __reduce_max_sync(0xffffffffu, bits);
    if ((threadIdx.x & 31) == 0) atomicMax(&top, of_warp);
    __syncthreads();
    // (in any order)
    if (threadIdx.x == 0) atomicMax(most, __float_as_uint(__half2float(__ushort_as_half((unsigned short)top))));
  }
}

// early: it may start before the kernel in front of it in the stream has ended.
template <typename T, int DP, bool KEYS>
int launch(const Params& p, int dev, int grid, bool early, cudaStream_t s) {
  static std::atomic<bool> configured[64] = {};
  const int rc = opt_in_smem(gradient_kernel<T, DP, KEYS>, Cfg<DP>::kSmem, configured, dev);
  if (rc != UPLIFT_LA_OK) return rc;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)grid);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = Cfg<DP>::kSmem;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = early ? 1 : 0;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, gradient_kernel<T, DP, KEYS>, p);
  if (e != cudaSuccess) return fail(UPLIFT_LA_ERR_CUDA, "attention backward launch: %s", cudaGetErrorString(e));
  return launched("attention backward");
}

template <typename T, bool KEYS>
int launch_d(const Params& p, int dev, int grid, bool early, cudaStream_t s) {
  return p.D <= 64 ? launch<T, 64, KEYS>(p, dev, grid, early, s) : launch<T, 128, KEYS>(p, dev, grid, early, s);
}

}  // namespace bwd

int attn_tc_backward(const AttnArgs& a, cudaStream_t s) {
  using namespace bwd;
  int dev = 0, sms = 0;
  int rc = sm_count(&dev, &sms);
  if (rc != UPLIFT_LA_OK) return rc;
  const int T = a.pk.T, S = a.pk.S;
  const bool bf16 = a.dtype == UPLIFT_LA_BF16;
  Params p;
  memset(&p, 0, sizeof(p));
  p.lse = a.lse;
  p.delta = a.delta;
  p.pk = a.pk;
  p.group = a.Hq / a.Hk;
  p.D = a.D;
  p.scale = a.scale;
  p.timeout_ns = tc_test_timeout_ns() != 0 ? tc_test_timeout_ns() : kTimeoutNs;
  p.host_status = host_status_word();
  p.test_fault = tc_test_fault();
  int* counters = reinterpret_cast<int*>(a.delta + (int64_t)T * a.Hq);
  const int64_t blocks = std::max<int64_t>(1, ((int64_t)T * a.Hq + 31) / 32);
  if (blocks >= (1ll << 31)) return fail(UPLIFT_LA_ERR_SHAPE, "attention backward: too many rows");
  unsigned* most = reinterpret_cast<unsigned*>(counters + 2);
  p.most = most;
  if (!bf16 && cudaMemsetAsync(most, 0, sizeof(*most), s) != cudaSuccess) return launched("attention backward");
  if (bf16) delta_kernel<__nv_bfloat16><<<(int)blocks, 256, 0, s>>>(a.dout, a.out, a.out_lo, a.delta, counters, most, a.pk, a.Hq, a.D);
  else delta_kernel<__half><<<(int)blocks, 256, 0, s>>>(a.dout, a.out, a.out_lo, a.delta, counters, most, a.pk, a.Hq, a.D);
  if ((rc = launched("attention backward")) != UPLIFT_LA_OK) return rc;
  if (T > 0) {
    // queries stay; without keys no box is loaded and the maps stay empty
    if ((rc = make_row_map(&p.x0, a.dtype, a.q, T, a.Hq, a.D, kM)) != UPLIFT_LA_OK) return rc;
    if ((rc = make_row_map(&p.x1, a.dtype, a.dout, T, a.Hq, a.D, kM)) != UPLIFT_LA_OK) return rc;
    if (S > 0) {
      if ((rc = make_row_map(&p.y0, a.dtype, a.k, S, a.Hk, a.D, kN)) != UPLIFT_LA_OK) return rc;
      if ((rc = make_row_map(&p.y1, a.dtype, a.v, S, a.Hk, a.D, kN)) != UPLIFT_LA_OK) return rc;
    }
    if ((rc = make_row_map(&p.o0, a.dtype, a.dq, T, a.Hq, a.D, 32)) != UPLIFT_LA_OK) return rc;
    p.y[0] = a.k;
    p.y[1] = a.v;
    p.out0 = a.dq;
    p.heads = a.Hq;
    p.counter = counters;
    const int64_t most = ((int64_t)T / kM + a.pk.B) * a.Hq;
    const int grid = (int)std::min<int64_t>(std::max<int64_t>(most, 1), cta_budget(sms));
    rc = bf16 ? launch_d<__nv_bfloat16, false>(p, dev, grid, true, s) : launch_d<__half, false>(p, dev, grid, true, s);
    if (rc != UPLIFT_LA_OK) return rc;
  }
  if (S > 0) {
    if ((rc = make_row_map(&p.x0, a.dtype, a.k, S, a.Hk, a.D, kM)) != UPLIFT_LA_OK) return rc;
    if ((rc = make_row_map(&p.x1, a.dtype, a.v, S, a.Hk, a.D, kM)) != UPLIFT_LA_OK) return rc;
    if (T > 0) {
      if ((rc = make_row_map(&p.y0, a.dtype, a.q, T, a.Hq, a.D, kN)) != UPLIFT_LA_OK) return rc;
      if ((rc = make_row_map(&p.y1, a.dtype, a.dout, T, a.Hq, a.D, kN)) != UPLIFT_LA_OK) return rc;
    }
    if ((rc = make_row_map(&p.o0, a.dtype, a.dv, S, a.Hk, a.D, 32)) != UPLIFT_LA_OK) return rc;
    if ((rc = make_row_map(&p.o1, a.dtype, a.dk, S, a.Hk, a.D, 32)) != UPLIFT_LA_OK) return rc;
    p.y[0] = a.q;
    p.y[1] = a.dout;
    p.out0 = a.dv;
    p.out1 = a.dk;
    p.heads = a.Hk;
    p.counter = counters + 1;
    const int64_t most = ((int64_t)S / kM + a.pk.B) * a.Hk;
    const int grid = (int)std::min<int64_t>(std::max<int64_t>(most, 1), cta_budget(sms));
    const bool early = T > 0 && cta_budget(sms) == sms;
    rc = bf16 ? launch_d<__nv_bfloat16, true>(p, dev, grid, early, s) : launch_d<__half, true>(p, dev, grid, early, s);
  }
  return rc;
}

int attn_bwd_device_status(bool clear) { return read_status(g_tok_bwd_status, clear); }

}  // namespace tok
}  // namespace ula
