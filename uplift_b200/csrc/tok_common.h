// Shared by the token-sequence kernels (C ABI in include/uplift_tokens.h):
// storage types, 16-byte vectors and the lookup of packed sequences.
#pragma once

#include <cuda_runtime.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <atomic>
#include <stdint.h>

#include "uplift_tokens.h"
#include "la_internal.h"

namespace ula {
namespace tok {

template <typename T> struct St;
template <> struct St<float> {
  __device__ __forceinline__ static float f(float x) { return x; }
  __device__ __forceinline__ static float t(float x) { return x; }
};
template <> struct St<__nv_bfloat16> {
  static constexpr uint32_t kFmt = 1;  // tcgen05 kind::f16 operand type
  __device__ __forceinline__ static float f(__nv_bfloat16 x) { return __bfloat162float(x); }
  __device__ __forceinline__ static __nv_bfloat16 t(float x) { return __float2bfloat16_rn(x); }
  __device__ __forceinline__ static uint32_t pack(float lo, float hi) {
    __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<uint32_t*>(&h);
  }
  __device__ __forceinline__ static float2 unpack(uint32_t v) {
    return __bfloat1622float2(*reinterpret_cast<__nv_bfloat162*>(&v));
  }
};
template <> struct St<__half> {
  static constexpr uint32_t kFmt = 0;
  __device__ __forceinline__ static float f(__half x) { return __half2float(x); }
  __device__ __forceinline__ static __half t(float x) { return __float2half_rn(x); }
  __device__ __forceinline__ static uint32_t pack(float lo, float hi) {
    __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<uint32_t*>(&h);
  }
  __device__ __forceinline__ static float2 unpack(uint32_t v) {
    return __half22float2(*reinterpret_cast<__half2*>(&v));
  }
};

// One sequence: first row and count of its queries and keys, clamped to the
// tensors.
struct Seq {
  int q0, nq, k0, nk;
};

struct Packing {
  const int32_t* cu_q;
  const int32_t* cu_k;
  const int32_t* used_k;  // or null
  int B, T, S;            // sequences, query rows, key rows
  int causal;
};

__device__ __forceinline__ int2 segment(const int32_t* cu, int b, int rows) {
  const int r0 = min(max(__ldg(cu + b), 0), rows);
  const int r1 = min(max(__ldg(cu + b + 1), r0), rows);
  return make_int2(r0, r1 - r0);
}

__device__ __forceinline__ Seq sequence(const Packing& p, int b) {
  const int2 q = segment(p.cu_q, b, p.T), k = segment(p.cu_k, b, p.S);
  Seq s{q.x, q.y, k.x, k.y};
  if (p.used_k != nullptr) s.nk = min(s.nk, max(__ldg(p.used_k + b), 0));
  return s;
}

// Number of keys that query i of the sequence sees.
__device__ __forceinline__ int keys_seen(const Seq& s, int i, int causal) {
  return causal ? max(0, min(s.nk, i + 1 - s.nq + s.nk)) : s.nk;
}

// Dynamic shared memory above 48 KB is an opt-in per function and device;
// `configured` remembers it (racing threads set the same value).
template <typename F>
inline int opt_in_smem(F fn, int bytes, std::atomic<bool>* configured, int dev) {
  if (dev < 0 || dev >= 64 || !configured[dev].load(std::memory_order_acquire)) {
    const cudaError_t e = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e != cudaSuccess) return fail(UPLIFT_LA_ERR_CUDA, "cudaFuncSetAttribute: %s", cudaGetErrorString(e));
    if (dev >= 0 && dev < 64) configured[dev].store(true, std::memory_order_release);
  }
  return UPLIFT_LA_OK;
}

inline int launched(const char* what) {
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return fail(UPLIFT_LA_ERR_CUDA, "%s launch: %s", what, cudaGetErrorString(e));
  return UPLIFT_LA_OK;
}

}  // namespace tok
}  // namespace ula
