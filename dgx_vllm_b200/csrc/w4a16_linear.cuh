// The weight-only linear layer's call, as its two kernels take it.
#pragma once

#include "common.cuh"

namespace b200fp4 {

struct LinearCall {
  const void* x;              // [M, K], rows ldx apart
  int x_dtype;
  int64_t ldx;
  const uint8_t* packed;
  const float* g;
  const void* bias;           // [N] or null
  int bias_dtype;
  void* out;                  // [M, N]
  int out_dtype;
  int64_t M, N, K;
  int* status;
};

// many tokens: tcgen05, the tokens the MMA's columns (w4a16_gemm.cu)
int launch_w4a16_gemm(const LinearCall& c, cudaStream_t st);

}  // namespace b200fp4
