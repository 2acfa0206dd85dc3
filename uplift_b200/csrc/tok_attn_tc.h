// Parts shared by the tensor-core kernels of the packed-sequence attention
// (tok_attn_fwd.cu, tok_attn_bwd.cu): tensor maps, bounded waits, the walk
// over sequences, TMEM operands and packed fp32 arithmetic.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "la_tc_common.h"
#include "tok_attn.h"

namespace ula {
namespace tok {

using namespace ::ula::tc;

// ------------------------------------------------------------ tensor maps
// [rows, heads, D] as axes (D, head, row), box {64 channels, 1, box_rows}.
// Boxes that reach beyond a sequence hold rows of the next one (zeros behind
// the tensor's last row); the kernels see to it that these reach no result.
int make_row_map(CUtensorMap* map, int dtype, const Rows& r, int64_t rows, int heads, int D, int box_rows);

__device__ __forceinline__ void load_rows(void* dst, const CUtensorMap* map, uint64_t* bar, int c, int h, int row) {
  tma_load(dst, map, bar, c, h, row, 0);
}

// Current device and its number of SMs.
int sm_count(int* dev, int* sms);

// Reads (and clears) a kernel's status word; -1 if that failed.
inline int read_status(unsigned int& symbol, bool clear) {
  unsigned int v = 0;
  cudaError_t e = cudaMemcpyFromSymbol(&v, symbol, sizeof(v));
  if (e == cudaSuccess && clear && v != 0) {
    const unsigned int zero = 0;
    e = cudaMemcpyToSymbol(symbol, &zero, sizeof(zero));
  }
  if (e != cudaSuccess) {
    fail(UPLIFT_LA_ERR_CUDA, "status word: %s", cudaGetErrorString(e));
    return -1;
  }
  return (int)v;
}

// ------------------------------------------------------------ waits
// Ends the CTA's work: every bounded wait returns false from now on.
__device__ __forceinline__ void give_up(volatile int* abort_flag, unsigned where, const WaitLimit& limit,
                                        unsigned int* status) {
  *abort_flag = 1;
  atomicCAS(status, 0u, where);
  if (limit.host_word != nullptr) {
    *reinterpret_cast<volatile unsigned int*>(limit.host_word) = where;
    __threadfence_system();
  }
}
// mbar_wait_status of la_tc_common.h as inline code.
__device__ __forceinline__ bool mbar_wait_inline(uint64_t* b, uint32_t parity, volatile int* abort_flag, unsigned where,
                                                 const WaitLimit& limit, unsigned int* status) {
  if (mbar_try(b, parity)) return true;
  const uint64_t t0 = gtimer();
  bool ok = true;
#pragma unroll 1
  for (uint32_t it = 1; !mbar_try(b, parity); ++it) {
    if ((it & 63u) != 0) continue;
    if (*abort_flag) {
      ok = false;
      break;
    }
    if (gtimer() - t0 > limit.ns) {
      give_up(abort_flag, where, limit, status);
      ok = false;
      break;
    }
  }
  return ok;
}

// A counter in shared memory that one thread raises and others wait for:
// cheaper to look at than an mbarrier.
__device__ __forceinline__ void raise_to(uint32_t* c, uint32_t v) {
  asm volatile("st.release.cta.shared::cta.u32 [%0], %1;" ::"r"(su32(c)), "r"(v) : "memory");
}
// Whole warp; false if the wait was given up.
__device__ __forceinline__ bool wait_raised(uint32_t* c, uint32_t v, volatile int* abort_flag, unsigned where,
                                            const WaitLimit& limit, unsigned int* status) {
  uint64_t t0 = 0;
  for (uint32_t it = 1;; ++it) {
    uint32_t now;
    asm volatile("ld.acquire.cta.shared::cta.u32 %0, [%1];" : "=r"(now) : "r"(su32(c)) : "memory");
    if (__all_sync(0xffffffffu, (int32_t)(now - v) >= 0)) return true;
    if ((it & 63u) == 0) {
      if (t0 == 0) t0 = gtimer();
      const bool late = gtimer() - t0 > limit.ns;
      if (__any_sync(0xffffffffu, late || *abort_flag)) {
        if (late) give_up(abort_flag, where, limit, status);
        return false;
      }
    }
  }
}

// Named barrier of n threads that tells all of them whether any had `pred`.
__device__ __forceinline__ bool bar_any(int id, int n, bool pred) {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.u32 p, %3, 0;\n\t"
      "barrier.cta.red.or.pred q, %1, %2, p;\n\t"
      "selp.u32 %0, 1, 0, q;\n\t}\n"
      : "=r"(r)
      : "r"(id), "r"(n), "r"((uint32_t)pred)
      : "memory");
  return r != 0;
}

// ------------------------------------------------------------ sequences
// Tile number -> (sequence, tile of the sequence), for numbers that only
// grow: a warp looks at 32 sequences at a time (a lane each) and goes on from
// where the last search ended.  `by_keys`: tiles of the key segments, else of
// the queries.
//
// A causal query tile costs in proportion to its index, a causal key tile to
// its distance from the end.  Among 32 sequences the costliest tiles come
// first: level by level, from the longest sequence's last tile (first, by
// keys) down, the tiles of equal cost of all sequences that have them.  Dealt
// to the CTAs forth and back, that evens out their work without a counter.
struct TileWalk {
  int b0 = 0;       // first sequence of the window
  int before = 0;   // tiles before the window (not causal) or the level
  int n = -1;       // tiles of the lane's sequence; -1: not read yet
  int level = 0;    // cost, in tiles, of the tiles at hand
  // all lanes; false: there is no such tile
  __device__ __forceinline__ bool find(const Packing& p, bool by_keys, int tile_rows, int tile, int* b, int* local,
                                       int* tiles) {
    const int lane = threadIdx.x & 31;
    for (;;) {
      if (n < 0) {
        if (b0 >= p.B) return false;
        n = 0;
        if (b0 + lane < p.B)
          n = ((by_keys ? segment(p.cu_k, b0 + lane, p.S).y : segment(p.cu_q, b0 + lane, p.T).y) + tile_rows - 1) /
              tile_rows;
        level = __reduce_max_sync(0xffffffffu, n);
      }
      if (p.causal) {
        while (level > 0) {
          const unsigned have = __ballot_sync(0xffffffffu, n >= level);
          const int cnt = __popc(have);
          if (tile < before + cnt) {
            const int l = __fns(have, 0, tile - before + 1);
            *tiles = __shfl_sync(0xffffffffu, n, l);
            *local = by_keys ? *tiles - level : level - 1;
            *b = b0 + l;
            return true;
          }
          before += cnt;
          --level;
        }
      } else {
        int sum = n;  // inclusive scan
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int v = __shfl_up_sync(0xffffffffu, sum, o);
          if (lane >= o) sum += v;
        }
        const int total = __shfl_sync(0xffffffffu, sum, 31);
        if (tile < before + total) {
          const int l = __ffs(__ballot_sync(0xffffffffu, tile < before + sum)) - 1;
          *tiles = __shfl_sync(0xffffffffu, n, l);
          *local = tile - before - (__shfl_sync(0xffffffffu, sum, l) - *tiles);
          *b = b0 + l;
          return true;
        }
        before += total;
      }
      b0 += 32;
      n = -1;
    }
  }
};

// Item number of a CTA's n-th turn: items are dealt forth and back.
__device__ __forceinline__ int64_t dealt(int n) {
  return (int64_t)n * gridDim.x + ((n & 1) ? gridDim.x - 1 - blockIdx.x : blockIdx.x);
}

// ------------------------------------------------------------ MMA issue
// One lane of a converged warp.  The MMA warp runs its loop with all lanes,
// so that descriptors and TMEM addresses are uniform over the warp and stay
// in uniform registers; only the instructions are issued by the elected lane.
__device__ __forceinline__ bool elect_one() {
  uint32_t pred;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "elect.sync _|p, 0xffffffff;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}\n"
      : "=r"(pred));
  return pred != 0;
}

// ------------------------------------------------------------ TMEM
// kind::f16 MMA with the A operand in TMEM (lane = row; a 32-bit column
// holds two consecutive K elements).
__device__ __forceinline__ void mma_tmem_a(uint32_t d_tmem, uint32_t a_tmem, uint64_t bdesc, uint32_t idesc,
                                           uint32_t accum) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}\n"
      ::"r"(d_tmem), "r"(a_tmem), "l"(bdesc), "r"(idesc), "r"(accum)
      : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};"
      ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
        "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void tmem_st8(uint32_t taddr, const uint32_t* r) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(taddr), "r"(r[0]),
               "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
               : "memory");
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// ------------------------------------------------------------ arithmetic
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
template <typename T>
__device__ __forceinline__ uint32_t nonfinite_probe(uint32_t acc, uint32_t x);  // acc stays 0 in both halves iff x is finite
template <>
__device__ __forceinline__ uint32_t nonfinite_probe<__nv_bfloat16>(uint32_t acc, uint32_t x) {
  __nv_bfloat162 r = __hfma2(*reinterpret_cast<__nv_bfloat162*>(&x), __nv_bfloat162(__nv_bfloat16(0.f), __nv_bfloat16(0.f)),
                             *reinterpret_cast<__nv_bfloat162*>(&acc));
  return *reinterpret_cast<uint32_t*>(&r);
}
template <>
__device__ __forceinline__ uint32_t nonfinite_probe<__half>(uint32_t acc, uint32_t x) {
  __half2 r = __hfma2(*reinterpret_cast<__half2*>(&x), __half2(__half(0.f), __half(0.f)), *reinterpret_cast<__half2*>(&acc));
  return *reinterpret_cast<uint32_t*>(&r);
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float y;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b), "f"(c));
  return y;
}

}  // namespace tok
}  // namespace ula
