// Attention over packed sequences on the tensor cores of B200 (sm_100a),
// bf16 / fp16, D <= 128.
//
// An item is two tiles of 128 query rows (M = 128) of one sequence that read
// the same key head: the same rows of two query heads where the group has an
// even number of them, else 256 rows of one head.  It walks the key tiles (64
// keys) that its rows see:
//
//   S_t[128 x 64] = Q_t . K_j^T                     (tcgen05, fp32 in TMEM)
//   m = max(m, rowmax S), P = exp2((S - m) scale log2 e), l += rowsum P
//   O_t[128 x D] += P . V_j                         (P from TMEM, V MN-major)
//
// with the running maximum m and sum l in the registers of the thread that
// owns the row (TMEM lane = query row), so that one pass over K and V
// suffices and S never leaves the SM.  O stays in TMEM for the whole item; a
// row is rescaled by exp2((m_old - m_new) scale log2 e) only when its maximum
// has grown by more than 2^8 (weights up to 2^8 lose nothing in fp32 and bf16
// or fp16, and the final division by l takes any common factor out), which
// after the first tiles hardly ever happens.
//
// Roles (640 threads, one persistent CTA per SM): warps 0-7 and 8-15 the
// softmax of a tile each, as two groups of four warps that take the key tiles
// in turn (a thread per row); warp 16 looks the items up and issues the TMA
// loads; warps 17 and 18 issue the MMAs of a tile each, so that the waits of
// one overlap the products of the other.  Each tile has two score buffers in
// TMEM, one per group, so the scores of the next key tile are there when a
// group is done.  A warp alone gets one exponential every 15 cycles out of the
// unit that could give one every 8, and none while it loads, compares and
// stores: with one group per tile (two warps per SM quarter) the unit was
// busy half of the time.  P is rounded to the storage type in place of S --
// the tensor cores multiply 16-bit operands; the sum l uses the unrounded
// weights.
//
// The maximum of a row is kept in shared memory.  A group decides on it for
// key tile j (and rescales O, after the product of tile j - 1) only when the
// other group has decided for tile j - 1, so weights and sums always agree
// on it; the decision needs the scores' maximum alone and comes long before
// the other group asks for it.
//
// Scores that a row does not see -- behind its sequence's end, where a tile
// holds rows of the next sequence, or behind the causal edge -- are set to
// -inf before the maximum.  P = 0 there, which an infinity or NaN in the same
// V row would turn into NaN: in the tiles that some row sees only in part the
// groups look V through, replace such values by zero and add them at the end
// to the rows that see them.  The two query tiles share V, so the tiles to look
// through are the item's (from the first key that its first row does not see),
// and the groups of both do so before their own products.
//
// D = 128 is bound by the tensor cores: a score product with 64 keys takes 48
// cycles per 16 channels where 32 would do (128 keys: 64), but tiles of 128
// keys leave TMEM no second score buffer (1212 us against 1104 for the prompt
// below).  One prompt of 16384 tokens, 16 heads on 4, bf16, causal: 1.1 ms,
// 1.0 PFLOP/s, 0.6 of a large library product; the tensor pipe is busy 56 % of
// the time.  D = 64 is bound by the exponentials, one for 256 operations: 8
// images of 5330 tokens, 6 heads, bf16: 520 us, 670 TFLOP/s, the unit busy
// 68 % of the time (a third score buffer: 546 us against 529; polynomial
// exponentials on the FMA units beside it: slower, for the instructions).
//
// Every mbarrier wait is bounded; on expiry the CTA records the role in this
// kernel's status word (and the registered host word), drains and exits.

#include <math.h>
#include <string.h>

#include <algorithm>
#include <atomic>

#include "tok_attn_tc.h"

namespace ula {

__device__ unsigned int g_tok_fwd_status;

namespace tok {
namespace fwd {

constexpr int kM = 128;            // query rows of a tile
constexpr int kN = 64;             // keys of a tile
constexpr int kQChunk = kM * 128, kKvChunk = kN * 128;  // 64 channels of a tile
constexpr int kThreads = 640;
constexpr int kTmemCols = 512;
constexpr int kItems = 2;          // ring of looked-up items
constexpr uint64_t kTimeoutNs = 2000000000ull;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kRescale = 8.f;    // log2 of the growth of the maximum that O is rescaled for

template <int DP>
struct Cfg {
  static constexpr int kChunks = DP / 64;
  static constexpr int kQBytes = kChunks * kQChunk;  // one query tile
  static constexpr int kSlotBytes = kChunks * kKvChunk;
  static constexpr int kSlots = 8;                   // K and V tiles
  static constexpr int kOffQ = 0;
  static constexpr int kOffKV = 2 * kQBytes;
  static constexpr int kOffStage = kOffKV + kSlots * kSlotBytes;
  static constexpr int kStageBytes = 32 * 128;           // a warp's 32 rows x 64 channels
  static constexpr int kOffRows = kOffStage + 8 * kStageBytes;  // [query tile][row]: maximum and the key tile it is of
  static constexpr int kOffBar = kOffRows + 2 * kM * 8;
  static constexpr int kNumBars = 2 + 2 * kSlots + 4 + 4 + 4 + 2 + 2 * kItems + 2;
  static constexpr int kOffMisc = kOffBar + kNumBars * 8;
  static constexpr int kOffItems = kOffMisc + 32;
  static constexpr int kSmem = kOffItems + kItems * 32;
  static_assert(kSmem <= 232448, "shared memory");
};

struct Item {
  int row;        // first query row in the tensor
  int n;          // its rows, 1..128 (256 if one head); 0: no more items
  int h;          // (first) query head
  int k0;         // first key row in the tensor
  int nk;         // keys of the sequence
  int see;        // keys that the first row sees (may be negative; each next row sees one more when causal)
  int nt[2];      // key tiles of each query tile
};

struct Params {
  CUtensorMap qmap, kmap, vmap;  // boxes {64, 1, 128, 1}
  CUtensorMap omap, lmap;        // out, out_lo; box {64, 1, 32, 1}
  Rows v, out, out_lo;           // out_lo.p: null if not wanted
  float* lse;
  Packing pk;
  int Hq, group, D;
  int heads;     // query heads of an item: 1 or 2
  int row_step;  // from the rows of the first query tile to those of the second: 128, or 0 with two heads
  float scale;
  uint64_t timeout_ns;
  unsigned int* host_status;
  int test_fault;  // 1: the producer issues no loads after a few (tests the waits that run out)
};

__device__ __forceinline__ bool mbar_wait(uint64_t* b, uint32_t parity, volatile int* abort_flag, unsigned where,
                                          const WaitLimit& limit) {
  if (mbar_try(b, parity)) return true;  // completed phase: no call into the bounded slow path
  return mbar_wait_status(b, parity, abort_flag, where, limit, &g_tok_fwd_status);
}

// Position of K_j and V_j of an item with `tiles` key tiles in the order in
// which they are loaded: K_0, K_1, V_0, K_2, V_1, K_3, ..
__device__ __forceinline__ uint32_t k_pos(int j) { return j < 2 ? j : 2 * j - 1; }
__device__ __forceinline__ uint32_t v_pos(int j, int tiles) { return min(2 * j + 2, 2 * tiles - 1); }

// The part of V row tid % 64 of a tile that thread tid of a group looks
// through: every second 16-byte piece of each chunk of 64 channels.
template <typename T, int CHUNKS>
__device__ __forceinline__ bool row_is_finite(const uint8_t* tile, int tid) {
  const int r = tid & 63;
  uint32_t acc = 0;
#pragma unroll
  for (int c = 0; c < CHUNKS; ++c) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint4 v = *reinterpret_cast<const uint4*>(tile + c * kKvChunk + r * 128 + (((2 * i + (tid >> 6)) ^ (r & 7)) << 4));
      acc = nonfinite_probe<T>(acc, v.x);
      acc = nonfinite_probe<T>(acc, v.y);
      acc = nonfinite_probe<T>(acc, v.z);
      acc = nonfinite_probe<T>(acc, v.w);
    }
  }
  const float2 f = St<T>::unpack(acc);
  return f.x == 0.f && f.y == 0.f;
}
// Replaces infinities and NaN in it by zero.
template <typename T, int CHUNKS>
__device__ __noinline__ void clean_row(uint8_t* tile, int tid) {
  const int r = tid & 63;
  for (int i = 0; i < CHUNKS * 32; ++i) {
    const int piece = 2 * ((i >> 3) & 3) + (tid >> 6);
    T* e = reinterpret_cast<T*>(tile + (i >> 5) * kKvChunk + r * 128 + ((piece ^ (r & 7)) << 4) + (i & 7) * 2);
    if (!isfinite(St<T>::f(*e))) *e = St<T>::t(0.f);
  }
}

// Adds the infinities and NaN of the rows j0 .. j1 - 1 of v (channels i0 ..
// i1 - 1) to a staged output row.
template <typename T>
__device__ __noinline__ void add_nonfinite(uint8_t* row, int lane, const T* v, int64_t stride, int j0, int j1, int i0, int i1) {
#pragma unroll 1
  for (int j = j0; j < j1; ++j) {
#pragma unroll 1
    for (int i = i0; i < i1; ++i) {
      const float x = St<T>::f(v[j * stride + i]);
      if (isfinite(x)) continue;
      T* e = reinterpret_cast<T*>(row + (((i >> 3) ^ (lane & 7)) << 4) + (i & 7) * 2);
      *e = St<T>::t(St<T>::f(*e) + x);
    }
  }
}

template <int N>
__device__ __forceinline__ float row_max(const float* f) {
  float mx[4] = {f[0], f[1], f[2], f[3]};
#pragma unroll
  for (int c = 4; c < N; c += 4) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if (c % 8 == 4 && c + 4 < N) mx[e] = max3(mx[e], f[c + e], f[c + 4 + e]);
      else if (c % 8 == 4) mx[e] = fmaxf(mx[e], f[c + e]);
    }
  }
  return fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
}

// LO: out_lo is written as well: 134 us against 116 for six documents of 5986
// tokens, 32 heads of 128 (its 49 MB are 8 of them), so only in training; a
// kernel of its own for the registers that it takes.
template <typename T, int DP, bool LO>
__global__ void __launch_bounds__(kThreads, 1) attention_kernel(const __grid_constant__ Params p) {
  using C = Cfg<DP>;
  extern __shared__ __align__(1024) uint8_t smem[];
  if ((su32(smem) & 1023u) != 0) {  // the swizzled tiles need it, and the declaration asks for it
    if (threadIdx.x == 0) atomicCAS(&g_tok_fwd_status, 0u, 1u);
    return;
  }
  uint8_t* sQ = smem + C::kOffQ;
  uint8_t* sKV = smem + C::kOffKV;
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + C::kOffBar);
  uint64_t* q_full = bars;
  uint64_t* q_empty = q_full + 1;             // the item's score MMAs are done
  uint64_t* kv_full = q_empty + 1;            // [kSlots]
  uint64_t* kv_empty = kv_full + C::kSlots;   // [kSlots]
  uint64_t* s_full = kv_empty + C::kSlots;    // [2][2] scores: query tile, buffer
  uint64_t* p_full = s_full + 4;              // [2][2] weights
  uint64_t* o_done = p_full + 4;              // [2][2] a product with V is complete: query tile, parity of the key tile
  uint64_t* o_full = o_done + 4;              // [2] an item's last product is complete
  uint64_t* item_full = o_full + 2;           // [kItems]
  uint64_t* item_empty = item_full + kItems;  // [kItems]
  uint64_t* drain = item_empty + kItems;      // [2]
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + C::kOffMisc);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + C::kOffMisc + 4);
  volatile int* v_cleaned = reinterpret_cast<volatile int*>(smem + C::kOffMisc + 16);
  int* issuing = reinterpret_cast<int*>(smem + C::kOffMisc + 20);
  volatile Item* items = reinterpret_cast<volatile Item*>(smem + C::kOffItems);

  const int tid = threadIdx.x;
  const int warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
  if (tid == 0) {
    mbar_init(q_full, 1);
    mbar_init(q_empty, 2);  // both MMA warps
    for (int i = 0; i < C::kSlots; ++i) {
      mbar_init(&kv_full[i], 1);
      mbar_init(&kv_empty[i], 2);
    }
    for (int i = 0; i < 4; ++i) {
      mbar_init(&s_full[i], 1);
      mbar_init(&p_full[i], 4);  // 4 warps
      mbar_init(&o_done[i], 1);
    }
    for (int i = 0; i < 2; ++i) mbar_init(&o_full[i], 1);
    for (int i = 0; i < kItems; ++i) {
      mbar_init(&item_full[i], 1);
      mbar_init(&item_empty[i], 18);  // 16 softmax warps, 2 MMA warps
    }
    mbar_init(&drain[0], 1);
    mbar_init(&drain[1], 1);
    abort_flag[0] = 0;
    abort_flag[1] = 0;  // stays 0: the flag of waits that must not be aborted
    *v_cleaned = 0;
    *issuing = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 17) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(su32(tmem_slot)), "r"(kTmemCols));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = __shfl_sync(0xffffffffu, *tmem_slot, 0);
  auto t_s = [&](int t, uint32_t b) { return tmem + (2 * t + b) * kN; };  // scores, then weights of tile t
  auto t_o = [&](int t) { return tmem + 4 * kN + t * DP; };               // output of tile t
  const WaitLimit tmo{p.timeout_ns, p.host_status};

  if (warp >= 16) {
    if (warp == 16) {
      // ---------------------------------------------------------- producer
      if (lane == 0) {
        prefetch_map(&p.qmap);
        prefetch_map(&p.omap);
        if (p.pk.S > 0) {
          prefetch_map(&p.kmap);
          prefetch_map(&p.vmap);
        }
      }
      TileWalk walk;
      bool ok = true;
      uint32_t g = 0;  // K / V slot uses
      uint32_t nq = 0;  // items with loads
      for (int n = 0;; ++n) {
        const int64_t i = dealt(n);
        int b = 0, local = 0, tiles = 0;
        const int per_tile = p.Hq / p.heads, item_rows = kM + p.row_step;
        const int64_t tile = i / per_tile;
        const bool more = tile < (1ll << 31) && walk.find(p.pk, false, item_rows, (int)tile, &b, &local, &tiles);
        Item it{};
        if (more) {
          const Seq s = sequence(p.pk, b);
          const int i0 = local * item_rows;
          it.row = s.q0 + i0;
          it.n = min(item_rows, s.nq - i0);
          it.h = (int)(i - tile * per_tile) * p.heads;
          it.k0 = s.k0;
          it.nk = s.nk;
          it.see = p.pk.causal ? i0 + 1 - s.nq + s.nk : s.nk;
#pragma unroll
          for (int t = 0; t < 2; ++t) {
            const int last = min(it.n, t * p.row_step + kM) - 1;  // last row of the tile
            const int see = p.pk.causal ? max(0, min(s.nk, it.see + last)) : s.nk;
            it.nt[t] = last >= t * p.row_step ? (see + kN - 1) / kN : 0;
          }
        }
        if (lane == 0) {
          const int slot = n % kItems;
          ok = mbar_wait(&item_empty[slot], ((n / kItems) & 1) ^ 1, abort_flag, 1, tmo);
          if (ok) {
            items[slot].row = it.row; items[slot].n = it.n; items[slot].h = it.h; items[slot].k0 = it.k0;
            items[slot].nk = it.nk; items[slot].see = it.see; items[slot].nt[0] = it.nt[0]; items[slot].nt[1] = it.nt[1];
            mbar_arrive(&item_full[slot]);
          }
          const int tiles_k = max(it.nt[0], it.nt[1]);
          if (ok && tiles_k > 0) {
            ok = mbar_wait(q_empty, (nq & 1) ^ 1, abort_flag, 1, tmo);
            if (ok) {
              const int qt = p.heads > 1 || it.n > kM ? 2 : 1;  // query tiles with rows
              mbar_expect_tx(q_full, qt * C::kQBytes);
              for (int t = 0; t < qt; ++t) {
#pragma unroll
                for (int c = 0; c < C::kChunks; ++c)
                  load_rows(sQ + t * C::kQBytes + c * kQChunk, &p.qmap, q_full, 64 * c, it.h + t * (p.heads - 1), it.row + t * p.row_step);
              }
            }
            ++nq;
            const int hk = it.h / p.group;
            auto load = [&](const CUtensorMap* map, int j) {
              const int s = g % C::kSlots;
              ok = ok && mbar_wait(&kv_empty[s], ((g / C::kSlots) & 1) ^ 1, abort_flag, 1, tmo);
              ++g;
              if (!ok || (p.test_fault == 1 && g > 4)) return;  // (K_0, K_1, V_0, K_2: the first decisions and products)
              mbar_expect_tx(&kv_full[s], C::kSlotBytes);
#pragma unroll
              for (int c = 0; c < C::kChunks; ++c)
                load_rows(sKV + s * C::kSlotBytes + c * kKvChunk, map, &kv_full[s], 64 * c, hk, it.k0 + j * kN);
            };
            load(&p.kmap, 0);
            if (tiles_k > 1) load(&p.kmap, 1);
            for (int j = 0; j < tiles_k && ok; ++j) {
              load(&p.vmap, j);
              if (j + 2 < tiles_k) load(&p.kmap, j + 2);
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
    } else if (warp < 19) {
      // ------------------------------------------- MMA issuer of a query tile
      const int t = warp - 17;
      constexpr uint32_t kIdS = idesc_f16(St<T>::kFmt, 0, kM, kN);
      constexpr uint32_t kIdO = idesc_f16(St<T>::kFmt, 1, kM, DP);
      const int ksteps = (p.D + 15) / 16;  // channels behind D are zero
      // descriptors: the start address counts 16 bytes in their lowest bits
      const uint64_t dq = mdesc(su32(sQ) + t * C::kQBytes, 16, 1024, kLayoutSw128);
      const uint64_t dk = mdesc(su32(sKV), 16, 1024, kLayoutSw128), dv = mdesc(su32(sKV), kKvChunk, 1024, kLayoutSw128);
      const uint32_t o = t_o(t);
      bool ok = true;
      uint32_t g = 0, nq = 0, ns = 0;  // ns: key tiles of this query tile so far
      auto wait = [&](uint64_t* bar, uint32_t parity) {
        return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag, 2, tmo));
      };
      auto ready = [&](uint32_t pos) { return wait(&kv_full[pos % C::kSlots], (pos / C::kSlots) & 1); };
      // (one lane) scores of key tile n, counted over items, with the K tile
      // at `pos`; a tile that this query tile does not see is only given back
      auto scores = [&](uint32_t n, uint32_t pos, bool seen, bool last) {
        if (seen) {
          const uint64_t k = dk + (pos % C::kSlots) * (C::kSlotBytes >> 4);
#pragma unroll
          for (int ks = 0; ks < DP / 16; ++ks)
            if (ks < ksteps)
              tc_mma(t_s(t, n & 1), dq + (((ks >> 2) * kQChunk + 32 * (ks & 3)) >> 4),
                     k + (((ks >> 2) * kKvChunk + 32 * (ks & 3)) >> 4), kIdS, ks > 0);
          tc_commit(&s_full[2 * t + (n & 1)]);
          if (last) tc_commit(q_empty);
        }
        tc_commit(&kv_empty[pos % C::kSlots]);
      };
      for (int n = 0; ok; ++n) {
        const int islot = n % kItems;
        ok = wait(&item_full[islot], (n / kItems) & 1);
        if (!ok) break;
        const int rows = items[islot].n, mine = items[islot].nt[t], tiles = max(items[islot].nt[0], items[islot].nt[1]);
        __syncwarp();
        if (lane == 0) mbar_arrive(&item_empty[islot]);
        if (rows == 0) break;
        if (tiles == 0) continue;
        ok = wait(q_full, nq & 1);
        ++nq;
        if (ok && mine == 0 && lane == 0) mbar_arrive(q_empty);
        for (int j = 0; j < min(2, tiles) && ok; ++j) {
          ok = ready(g + j);
          if (!ok) break;
          tc_fence_after();
          if (elect_one()) scores(ns + j, g + j, j < mine, j + 1 == mine);
          __syncwarp();
        }
        for (int j = 0; j < tiles && ok; ++j) {
          // V_j and K_j+2 are there long before the weights, which are waited
          // for last: the products follow them at once
          const uint32_t gv = g + v_pos(j, tiles), gk = g + k_pos(j + 2);
          ok = ready(gv) && (j + 2 >= tiles || ready(gk)) &&
               (j >= mine || wait(&p_full[2 * t + ((ns + j) & 1)], ((ns + j) >> 1) & 1));
          if (!ok) break;
          tc_fence_after();
          if (elect_one()) {
            // One tile's products at a time: interleaved, both tiles' would
            // end together, and the tensor cores wait while both groups work.
            // (Only a matter of speed: after a while it goes on regardless.)
            for (int spin = 0; atomicExch(issuing, 1) != 0 && spin < 4096; ++spin) {}
            if (j < mine) {
              const uint64_t v = dv + (gv % C::kSlots) * (C::kSlotBytes >> 4);
              const uint32_t w = t_s(t, (ns + j) & 1);
#pragma unroll
              for (int ks = 0; ks < kN / 16; ++ks)
                mma_tmem_a(o, w + 8 * (ks & 1) + 32 * (ks >> 1), v + ((2048 * ks) >> 4), kIdO, (j > 0 || ks > 0) ? 1u : 0u);
              // announced before the scores of tile j + 2 are: who sees those
              // and waits for V_j+1's product must find this phase complete
              tc_commit(&o_done[2 * t + ((ns + j) & 1)]);
              if (j + 1 == mine) tc_commit(&o_full[t]);
            }
            if (j + 2 < tiles) scores(ns + j + 2, gk, j + 2 < mine, j + 3 == mine);
            tc_commit(&kv_empty[gv % C::kSlots]);
            atomicExch(issuing, 0);
          }
          __syncwarp();
        }
        g += 2 * tiles;
        ns += mine;
      }
      // all issued MMAs complete before TMEM can be released (this wait
      // ignores the abort flag: it must not be cut short by another role)
      if (elect_one()) tc_commit(&drain[t]);
      __syncwarp();
      mbar_wait(&drain[t], 0, abort_flag + 1, 2, tmo);
    }
  } else {
    // ------------------------------------------------------------ softmax
    const int t = warp >> 3, group = (warp >> 2) & 1, q = warp & 3;
    const int r = 32 * q + lane;     // row of the tile = TMEM lane
    const int pair = 1 + 4 * t + q;  // named barrier of the two warps with the same rows
    volatile uint64_t* decided = reinterpret_cast<volatile uint64_t*>(smem + C::kOffRows) + t * kM + r;
    const uint32_t lane_off = (uint32_t)(32 * q) << 16;
    const uint32_t ts = t_s(t, group) + lane_off, to = t_o(t) + lane_off;
    const float c2 = p.scale * kLog2e;
    uint8_t* stage = smem + C::kOffStage + (4 * t + q) * C::kStageBytes;
    uint32_t ns = 0, no = 0, g = 0;  // key tiles and items of this query tile, K / V tiles before this item
    // A wait that ran out sets ok = false and ends the steps; the warps of a
    // pair tell each other at the item's pair barriers.
    bool ok = true;
    auto wait = [&](uint64_t* bar, uint32_t parity, unsigned where) {
      return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag, where, tmo));
    };
    // The row's maximum and the number of the key tile that it was decided
    // for, in one word: the thread of the other group sees both at once.
    auto decide = [&](float m, uint32_t step) { *decided = ((uint64_t)(step + 1) << 32) | __float_as_uint(m); };
    auto decision = [&](uint32_t step, float* m) {
      uint64_t t0 = 0;
      bool got = false;
      for (uint32_t it = 1;; ++it) {
        const uint64_t v = *decided;
        got = (uint32_t)(v >> 32) == step + 1;
        *m = __uint_as_float((uint32_t)v);
        if (__all_sync(0xffffffffu, got)) return true;
        if ((it & 63u) == 0) {
          if (t0 == 0) t0 = gtimer();
          const bool late = gtimer() - t0 > tmo.ns;
          if (__any_sync(0xffffffffu, late || *abort_flag)) {
            if (late) give_up(abort_flag, 3, tmo, &g_tok_fwd_status);
            return false;
          }
        }
      }
    };
    *decided = 0;
    for (int n = 0;; ++n) {
      const int islot = n % kItems;
      ok = ok && wait(&item_full[islot], (n / kItems) & 1, 3);
      if (bar_any(pair, 64, !ok)) break;
      Item it;
      it.row = items[islot].row; it.n = items[islot].n; it.h = items[islot].h; it.k0 = items[islot].k0;
      it.nk = items[islot].nk; it.see = items[islot].see;
      const int tiles = items[islot].nt[t], all_tiles = max(items[islot].nt[0], items[islot].nt[1]);
      __syncwarp();
      if (lane == 0) mbar_arrive(&item_empty[islot]);
      if (it.n == 0) break;
      it.h += t * (p.heads - 1);
      const int first = t * p.row_step;            // first row of this tile
      const int rows = min(kM, it.n - first);      // its rows; may be <= 0
      const int see = p.pk.causal ? max(0, min(it.nk, it.see + first + r)) : it.nk;  // keys this row sees
      // tiles from edge on hold keys that the item's first row does not see
      const int edge = (p.pk.causal ? max(0, min(it.nk, it.see)) : it.nk) / kN;
      float m = -INFINITY, l = 0.f;  // l: of this group's key tiles, for the maximum m
      // l for a new maximum
      auto adopt = [&](float mn) {
        if (mn != m) l *= ex2((m - mn) * c2);
        m = mn;
      };
      for (int j = (ns & 1) == (uint32_t)group ? 0 : 1; j < tiles; j += 2) {
        const uint32_t nn = ns + j;
        ok = wait(&s_full[2 * t + group], (nn >> 1) & 1, 3);
        if (!ok) break;
        tc_fence_after();
        const int lim = j >= edge ? see - j * kN : kN;  // columns from lim on are not seen
        uint32_t s[32];
        float* f = reinterpret_cast<float*>(s);
        auto cut = [&](int first) {
          if (j >= edge) {
#pragma unroll
            for (int c = 0; c < 32; ++c) f[c] = first + c < lim ? f[c] : -INFINITY;
          }
        };
        tc_ld32(ts, s);
        tc_wait_ld_regs(s);
        cut(0);
        float mj = row_max<32>(f);
        tc_ld32(ts + 32, s);
        tc_wait_ld_regs(s);
        cut(32);
        mj = fmaxf(mj, row_max<32>(f));
        if (j == 0) {
          m = mj;
        } else {
          float before;
          ok = decision(nn - 1, &before);
          if (!ok) break;
          adopt(before);
          const bool grow = (mj - m) * c2 > kRescale;  // also from m = -inf
          if (__any_sync(0xffffffffu, grow)) {
            // the last product that wrote O has to be complete; the one two
            // before it, the last phase of the same barrier, is: it was
            // announced long before the scores of this tile
            ok = wait(&o_done[2 * t + ((nn - 1) & 1)], ((nn - 1) >> 1) & 1, 3);
            if (!ok) break;
            tc_fence_after();
            const float a = grow ? ex2((m - mj) * c2) : 1.f;
            if (grow) adopt(mj);
#pragma unroll 1
            for (int c = 0; c < DP; c += 16) {
              uint32_t o[16];
              tc_ld16(to + c, o);
              tc_wait_ld_regs16(o);
#pragma unroll
              for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * a);
              tmem_st16(to + c, o);
            }
          }
        }
        decide(m, nn);
        const float mc = m == -INFINITY ? 0.f : m * c2;
        const float2 c22 = make_float2(c2, c2), mc2 = make_float2(-mc, -mc);
        float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
        auto weights = [&](uint32_t dst) {  // over scores that have been read
          uint32_t w[16];
#pragma unroll
          for (int c = 0; c < 32; c += 2) {
            const float2 x = __ffma2_rn(make_float2(f[c], f[c + 1]), c22, mc2);
            const float2 y = make_float2(ex2(x.x), ex2(x.y));
            sum[(c >> 1) & 1] = __fadd2_rn(sum[(c >> 1) & 1], y);
            w[c / 2] = St<T>::pack(y.x, y.y);
          }
          tmem_st16(dst, w);
        };
        weights(ts + 32);
        tc_ld32(ts, s);  // the first half once more: 64 scores and their weights at a time do not fit the registers
        tc_wait_ld_regs(s);
        cut(0);
        weights(ts);
        l += (sum[0].x + sum[1].x) + (sum[0].y + sum[1].y);
        if (j >= edge) {
          // V tile j: infinities and NaN out (see above)
          const uint32_t gv = g + v_pos(j, all_tiles);
          uint8_t* tile = sKV + (gv % C::kSlots) * C::kSlotBytes;
          ok = wait(&kv_full[gv % C::kSlots], (gv / C::kSlots) & 1, 3);
          if (!ok) break;
          if (!row_is_finite<T, C::kChunks>(tile, tid & 127)) {
            *v_cleaned = 1;
            __threadfence_block();
            clean_row<T, C::kChunks>(tile, tid & 127);
          }
          // also for what the other query tile's warps have cleaned
          fence_proxy_async();
        }
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[2 * t + group]);
      }
      ns += tiles;
      g += 2 * all_tiles;
      if (rows <= 0) continue;
      // ---------------------------------------------------------- epilogue
      if (tiles > 0) {
        float last;
        ok = ok && decision(ns - 1, &last) && wait(&o_full[t], no & 1, 4);
        ++no;
        tc_fence_after();
        if (ok) adopt(last);
      }
      if (bar_any(pair, 64, !ok)) break;
      // both have the final maximum: its word serves to exchange the sums
      reinterpret_cast<volatile float*>(decided)[group] = l;
      named_bar(pair, 64);
      l += reinterpret_cast<volatile float*>(decided)[1 - group];
      named_bar(pair, 64);
      if (group == 0) *decided = 0;
      const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);  // NaN stays NaN
      if (p.lse != nullptr && r < rows && group == 0)
        p.lse[(int64_t)it.h * p.pk.T + it.row + first + r] = l == 0.f ? -INFINITY : m * p.scale + logf(l);
      const int wrows = min(32, rows - 32 * q);  // of this warp's rows
      const bool fix = *v_cleaned != 0;
      // 64 channels at a time, half of them by each warp of the pair
#pragma unroll 1
      for (int c = 0; c < C::kChunks; ++c) {
        if (64 * c >= p.D) break;
        uint8_t* row = stage + lane * 128;
        const int row0 = it.row + first + 32 * q;
        // out, then (for the gradients) what its rounding left
#pragma unroll 1
        for (int part = 0; part < (LO ? 2 : 1); ++part) {
          uint32_t o[32];
          if (tiles > 0) tc_ld32(to + 64 * c + 32 * group, o);
          if (group == 0 && lane == 0) bulk_wait_read0();  // the staging buffer is free
          named_bar(pair, 64);
          if (tiles > 0) tc_wait_ld_regs(o);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            uint32_t y[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              float2 x = make_float2(__uint_as_float(o[8 * e + 2 * i]) * inv, __uint_as_float(o[8 * e + 2 * i + 1]) * inv);
              if (inv == 0.f) x = make_float2(0.f, 0.f);
              y[i] = St<T>::pack(x.x, x.y);
              if (LO && part == 1) {
                const float2 hi = St<T>::unpack(y[i]);
                y[i] = St<T>::pack(isfinite(hi.x) ? x.x - hi.x : 0.f, isfinite(hi.y) ? x.y - hi.y : 0.f);
              }
            }
            *reinterpret_cast<uint4*>(row + (((4 * group + e) ^ (lane & 7)) << 4)) = make_uint4(y[0], y[1], y[2], y[3]);
          }
          if (fix && tiles > 0 && part == 0) {
            // add the values taken out of the tiles on the edge of this item
            add_nonfinite<T>(row, lane, static_cast<const T*>(p.v.p) + (int64_t)it.k0 * p.v.t + (it.h / p.group) * p.v.h + 64 * c,
                             p.v.t, edge * kN, see, 32 * group, min(32 * group + 32, p.D - 64 * c));
          }
          fence_proxy_async();
          named_bar(pair, 64);
          if (wrows == 32) {
            if (group == 0 && lane == 0) {
              tma_store(!LO || part == 0 ? &p.omap : &p.lmap, stage, 64 * c, it.h, row0, 0);
              bulk_commit();
            }
          } else {  // the rows behind the sequence are not ours
            const Rows& out = !LO || part == 0 ? p.out : p.out_lo;
            for (int e = 32 * group + lane; e < wrows * 8; e += 64) {
              const int rr = e >> 3, piece = e & 7;
              if (64 * c + 8 * piece < p.D)
                *reinterpret_cast<uint4*>(static_cast<T*>(const_cast<void*>(out.p)) + (int64_t)(row0 + rr) * out.t +
                                          (int64_t)it.h * out.h + 64 * c + 8 * piece) =
                    *reinterpret_cast<const uint4*>(stage + rr * 128 + ((piece ^ (rr & 7)) << 4));
            }
          }
        }
      }
      tc_fence_before();  // O has been read: the next item's first product (after p_full) may overwrite it
    }
    // rows of no sequence: zeros, lse -inf
    const int lo = p.pk.B > 0 ? segment(p.pk.cu_q, 0, p.pk.T).x : 0;
    int hi = lo;
    if (p.pk.B > 0) {
      const int2 e = segment(p.pk.cu_q, p.pk.B - 1, p.pk.T);
      hi = max(lo, e.x + e.y);
    }
    const int64_t gap = (int64_t)lo + (p.pk.T - hi);
    for (int64_t i = (int64_t)blockIdx.x * 16 + warp; i < gap * p.Hq; i += (int64_t)gridDim.x * 16) {
      const int64_t k = i / p.Hq;
      const int h = (int)(i - k * p.Hq);
      const int64_t row = k < lo ? k : hi + (k - lo);
      T* o = static_cast<T*>(const_cast<void*>(p.out.p)) + row * p.out.t + (int64_t)h * p.out.h;
      for (int e = lane * 8; e < p.D; e += 256) *reinterpret_cast<uint4*>(o + e) = make_uint4(0, 0, 0, 0);
      if constexpr (LO) {
        T* ol = static_cast<T*>(const_cast<void*>(p.out_lo.p)) + row * p.out_lo.t + (int64_t)h * p.out_lo.h;
        for (int e = lane * 8; e < p.D; e += 256) *reinterpret_cast<uint4*>(ol + e) = make_uint4(0, 0, 0, 0);
      }
      if (p.lse != nullptr && lane == 0) p.lse[(int64_t)h * p.pk.T + row] = -INFINITY;
    }
    if (lane == 0) bulk_wait_all();
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 17) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemCols));
  }
}

template <typename T, int DP, bool LO>
int launch(const Params& p, int dev, int grid, cudaStream_t s) {
  static std::atomic<bool> configured[64] = {};
  const int rc = opt_in_smem(attention_kernel<T, DP, LO>, Cfg<DP>::kSmem, configured, dev);
  if (rc != UPLIFT_LA_OK) return rc;
  attention_kernel<T, DP, LO><<<grid, kThreads, Cfg<DP>::kSmem, s>>>(p);
  return launched("attention");
}

template <typename T>
int launch(const Params& p, int dev, int grid, cudaStream_t s) {
  if (p.out_lo.p != nullptr) return p.D <= 64 ? launch<T, 64, true>(p, dev, grid, s) : launch<T, 128, true>(p, dev, grid, s);
  return p.D <= 64 ? launch<T, 64, false>(p, dev, grid, s) : launch<T, 128, false>(p, dev, grid, s);
}

}  // namespace fwd

int make_row_map(CUtensorMap* map, int dtype, const Rows& r, int64_t rows, int heads, int D, int box_rows) {
  const CUtensorMapDataType dt = dtype == UPLIFT_LA_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  return tc_make_map(map, dt, 2, r.p, D, heads, (int)rows, 1, r.h, r.t, r.t * rows, 64, 1, box_rows);
}

int sm_count(int* dev, int* sms) {
  if (cudaGetDevice(dev) != cudaSuccess) return fail(UPLIFT_LA_ERR_NO_DEVICE, "cudaGetDevice failed");
  static std::atomic<int> counts[64] = {};
  *sms = (*dev >= 0 && *dev < 64) ? counts[*dev].load(std::memory_order_relaxed) : 0;
  if (*sms == 0) {
    if (cudaDeviceGetAttribute(sms, cudaDevAttrMultiProcessorCount, *dev) != cudaSuccess || *sms < 1)
      return fail(UPLIFT_LA_ERR_NO_DEVICE, "no multiprocessor count");
    if (*dev >= 0 && *dev < 64) counts[*dev].store(*sms, std::memory_order_relaxed);
  }
  return UPLIFT_LA_OK;
}

int attn_tc_forward(const AttnArgs& a, cudaStream_t s) {
  using namespace fwd;
  Params p;
  memset(&p, 0, sizeof(p));
  int dev = 0, sms = 0;
  int rc = sm_count(&dev, &sms);
  if (rc == UPLIFT_LA_OK) rc = make_row_map(&p.qmap, a.dtype, a.q, a.pk.T, a.Hq, a.D, kM);
  // without key rows no K / V box is ever loaded; the maps stay empty
  if (rc == UPLIFT_LA_OK && a.pk.S > 0) rc = make_row_map(&p.kmap, a.dtype, a.k, a.pk.S, a.Hk, a.D, kN);
  if (rc == UPLIFT_LA_OK && a.pk.S > 0) rc = make_row_map(&p.vmap, a.dtype, a.v, a.pk.S, a.Hk, a.D, kN);
  if (rc == UPLIFT_LA_OK) rc = make_row_map(&p.omap, a.dtype, a.out, a.pk.T, a.Hq, a.D, 32);
  if (rc == UPLIFT_LA_OK && a.out_lo.p != nullptr) rc = make_row_map(&p.lmap, a.dtype, a.out_lo, a.pk.T, a.Hq, a.D, 32);
  if (rc != UPLIFT_LA_OK) return rc;
  p.v = a.v;
  p.out = a.out;
  p.out_lo = a.out_lo;
  p.lse = a.lse;
  p.pk = a.pk;
  p.Hq = a.Hq;
  p.group = a.Hq / a.Hk;
  p.heads = p.group % 2 == 0 ? 2 : 1;
  p.row_step = p.heads == 2 ? 0 : kM;
  p.D = a.D;
  p.scale = a.scale;
  p.timeout_ns = tc_test_timeout_ns() != 0 ? tc_test_timeout_ns() : kTimeoutNs;
  p.host_status = host_status_word();
  p.test_fault = tc_test_fault();
  const int64_t most = ((int64_t)a.pk.T / (kM + p.row_step) + a.pk.B) * (a.Hq / p.heads);  // items, at most
  const int grid = (int)std::min<int64_t>(std::max<int64_t>(most, 1), cta_budget(sms));
  return a.dtype == UPLIFT_LA_BF16 ? launch<__nv_bfloat16>(p, dev, grid, s) : launch<__half>(p, dev, grid, s);
}

int attn_fwd_device_status(bool clear) { return read_status(g_tok_fwd_status, clear); }

}  // namespace tok
}  // namespace ula
