// The weight-only linear layer's call, as its two kernels take it.
#pragma once

#include "common.cuh"

namespace b200fp4 {

struct LinearCall {
  const void* x;              // [M, K], rows ldx apart
  int x_dtype;
  int64_t ldx;
  const uint8_t* packed;
  const uint32_t* tail;       // behind its units
  const float* g;
  const void* bias;           // [N] or null
  int bias_dtype;
  void* out;                  // [M, N]
  int out_dtype;
  int64_t M, N, K;
  int* status;
};

// Units (128 of k) that are summed in one accumulator where the result is f32.  Matrix instructions of both kinds truncate what they add to a sum,
// which therefore drifts with its length: against 64 bits a chain of tcgen05's of K = 1024 is off by 9e-7 (norm of the differences over that of the
// result), one of 4912 by 43e-7 and of 14336 by 130e-7; mma.sync's of K = 768 by 9e-7; sums that are rounded by 5 to 20e-7.  Chains are added up in
// f32, rounded.  A result of 16 bits, off by 2e-4 or more in its own rounding, needs none.
constexpr int kChain = 8, kWarpChain = 6;

// many tokens: tcgen05, the tokens the MMA's columns (w4a16_gemm.cu)
int launch_w4a16_gemm(const LinearCall& c, cudaStream_t st);

}  // namespace b200fp4
