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
  Rows out_lo;        // 16-bit out only: out before its rounding, less out; p null: not wanted, not known
  float* lse;         // [Hq][T] or null
  Packing pk;
  int Hq, Hk, D;
  float scale;
  int dtype;
  // backward
  Rows dout, dq, dk, dv;
  float* delta;  // [Hq][T], then 16 words: item counters of the two passes, fp16: the largest |dout|
};

// bf16 / fp16 attention on the tensor cores (tok_attn_fwd.cu).
int attn_tc_forward(const AttnArgs& a, cudaStream_t s);
int attn_fwd_device_status(bool clear);
// Their gradients (tok_attn_bwd.cu).
int attn_tc_backward(const AttnArgs& a, cudaStream_t s);
int attn_bwd_device_status(bool clear);

// The form for a few queries per sequence (tok_attn_step.cu).
bool attn_step_applies(int B, int64_t T, int group, int dtype);
int64_t attn_step_workspace(int64_t T, int Hq, int Hk, int D);  // bytes
int attn_step_forward(const AttnArgs& a, void* workspace, cudaStream_t s);

// fp32 attention on CUDA cores (tok_attn_simt.cu).
int attn_simt_forward(const AttnArgs& a, cudaStream_t s);
int attn_simt_backward(const AttnArgs& a, cudaStream_t s);

}  // namespace tok
}  // namespace ula
