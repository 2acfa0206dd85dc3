// Internal interface of the packed-sequence attention kernels.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

#include "tok_common.h"

namespace ula {
namespace tok {

struct Rows {  // [rows, heads, D], channel stride 1; strides in elements
  const void* p;
  int64_t t, h;
};

struct AttnArgs {
  Rows q, k, v, out;  // forward writes out
  float* lse;         // [Hq][T] or null
  Packing pk;
  int Hq, Hk, D;
  float scale;
  int dtype;
  // backward
  Rows dout, dq, dk, dv;
  float* delta;  // [Hq][T]
};

// fp32 attention on CUDA cores (tok_attn_simt.cu).
int attn_simt_forward(const AttnArgs& a, cudaStream_t s);
int attn_simt_backward(const AttnArgs& a, cudaStream_t s);

}  // namespace tok
}  // namespace ula
