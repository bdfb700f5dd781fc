// Weight-only NVFP4: 4-bit weights, 16-bit activations.  The packed weight, its decoding, and what the kernels over it share.
//
// value(n, k) = e2m1(code[n, k]) * e4m3(scale[n, k / 16]) * g.  A code has two significant bits and a scale four, so that their product
// is exact in f16: the operand of a 16-bit matrix instruction loses nothing, and the sums are f32.
//
// f16 and not bf16, because a B200 converts two codes to two f16 in one instruction and has none for bf16: 16 rows x 128 of k take 32 cycles of
// an SM from registers to the matrix instruction, by shifts and masks to bf16 51, and 50 is what they take to arrive from HBM.  bf16 activations
// become f16 exactly, after a power of two for each row has brought its largest value below 2^15: what is then below f16's
// smallest, 2^-39 of that largest value, is the only part that can be rounded.
//
// Packed weight: units of 32 rows x 128 of k, 2304 bytes, [matrix][128 rows][k / 128][32 rows][unit] (fewer rows in a last block): one copy brings
// 128 rows x 128 of k, and one a unit.  A unit is two tiles of the 16x8x16 matrix instruction, whose lane l holds rows l / 4 and l / 4 + 8 and four k
// of each: with the k of an instruction taken from four blocks of 16, lane l needs block l % 4 only, so it converts one scale a row for four
// instructions, and its operands of a whole block are 16 neighbouring values:
//   codes   [tile][half: 64 of k][chunk_at(l / 4, l % 4)][16 bytes: row l / 4, k 0..15 | row l / 4 + 8, k 0..15]
//   scales  [lane][tile][4 bytes: half 0 row l / 4, row l / 4 + 8 | half 1 likewise]
// The chunks are ordered so that no two lanes meet in a bank when each reads its 16 bytes, nor when a lane is one of 32 rows and reads the 8 bytes of
// a block (the decoding of w4a16_gemm.cu).  Negative scales give their sign to their codes when the weight is packed.
// Gated: the 16 rows of a tile are eight gate rows and the same eight up rows, so that a lane holds both of a value's products.
// Behind the units, for each matrix (gated: for its gate rows and its up rows) a word: the largest magnitude of code times scale, which the upper half
// of an f32 holds exactly, and in the lower half a tag of the sizes.  Packed bytes do not tell K = 112 from 128, or [64, 128] from [32, 256]: kernels
// compare the tag with the sizes that they are called with, and every row of a result of a weight that was packed for others has NaN, a linear's in the
// columns of its last strip (status kOtherSizes).
#pragma once

#include "common.cuh"

namespace b200fp4 {
namespace w4 {

constexpr int kUnitBytes = 2304, kUnitScales = 2048, kUnitK = 128, kUnitRows = 32;
constexpr int kOtherSizes = 63;

// the same for no two sizes within 64 rows and 64 blocks of 16 of each other
__host__ __device__ __forceinline__ uint32_t size_tag(int64_t N, int64_t K, int gated) {
  return (uint32_t)((uint64_t)N * 40503u + (uint64_t)(K / 16) * 30011u + (gated ? 0x5555u : 0u)) & 0xFFFFu;
}
__device__ __forceinline__ bool packed_for(uint32_t tail, uint32_t tag) { return (tail & 0xFFFFu) == tag; }
__device__ __forceinline__ float peak_of(uint32_t word) { return __uint_as_float(word & 0xFFFF0000u); }

__host__ __device__ __forceinline__ int64_t strips_of(int64_t rows) { return (rows + kUnitRows - 1) / kUnitRows; }      // of 32 rows
__host__ __device__ __forceinline__ int64_t units_of(int64_t K) { return (K + kUnitK - 1) / kUnitK; }

// Units of a matrix before those of a strip of 32 rows, and from one 128 of k to the next
template <typename Int>
__host__ __device__ __forceinline__ Int strip_at(Int strip, Int strips, Int units, Int unit, int& step) {
  const Int block = strip & ~(Int)3;
  step = (int)(strips - block < 4 ? strips - block : 4);
  return block * units + unit * step + (strip - block);
}

// where the chunk of row r8 (and r8 + 8) and block t of a half begins
__device__ __forceinline__ uint32_t chunk_at(int r8, int t) { return (uint32_t)(t * 8 + ((r8 + 2 * t) & 7)) * 16; }

__device__ __forceinline__ __half2 as_half2(uint32_t v) { return *reinterpret_cast<const __half2*>(&v); }
__device__ __forceinline__ uint32_t as_u32(__half2 v) { return *reinterpret_cast<const uint32_t*>(&v); }

// Eight codes -> four pairs of f16
__device__ __forceinline__ void codes_to_pairs(uint32_t w, uint32_t (&p)[4]) {
  asm("{\n"
      ".reg .b8 q0, q1, q2, q3;\n"
      "mov.b32 {q0, q1, q2, q3}, %4;\n"
      "cvt.rn.f16x2.e2m1x2 %0, q0;\n"
      "cvt.rn.f16x2.e2m1x2 %1, q1;\n"
      "cvt.rn.f16x2.e2m1x2 %2, q2;\n"
      "cvt.rn.f16x2.e2m1x2 %3, q3;\n"
      "}\n"
      : "=r"(p[0]), "=r"(p[1]), "=r"(p[2]), "=r"(p[3])
      : "r"(w));
}

// The scales of rows l / 4 (x) and l / 4 + 8 (y) for one half of a unit: a byte's fields, moved to those of f16, are the scale times 2^-8
__device__ __forceinline__ __half2 scales_of(uint32_t bytes, int half) {
  return __hmul2(as_half2(prmt(bytes, 0u, half ? 0x3424u : 0x1404u) >> 1), as_half2(0x5C005C00u));
}

// two E4M3 bytes -> two f16
__device__ __forceinline__ __half2 e4m3_pair(uint32_t bytes) {
  uint32_t r;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"((unsigned short)bytes));
  return as_half2(r);
}

// two bf16 times a power of two (twice in `factor`) -> two f16
__device__ __forceinline__ uint32_t bf16_to_f16_pair(uint32_t x, uint32_t factor) {
  const __nv_bfloat162 v = __hmul2(*reinterpret_cast<const __nv_bfloat162*>(&x), *reinterpret_cast<const __nv_bfloat162*>(&factor));
  const uint32_t b = *reinterpret_cast<const uint32_t*>(&v);
  return as_u32(__floats2half2_rn(__uint_as_float(b << 16), __uint_as_float(b & 0xFFFF0000u)));
}

__device__ __forceinline__ void mma_16x8x16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint2 lds64(uint32_t addr) {
  uint2 v;
  asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(addr) : "memory");
  return v;
}

// outputs and biases of any of the three types
__device__ __forceinline__ void store_value(void* out, int dtype, size_t at, float v) {
  if (dtype == B200FP4_DTYPE_BF16) static_cast<__nv_bfloat16*>(out)[at] = __float2bfloat16_rn(v);
  else if (dtype == B200FP4_DTYPE_F16) static_cast<__half*>(out)[at] = __float2half_rn(v);
  else static_cast<float*>(out)[at] = v;
}
__device__ __forceinline__ float load_value(const void* p, int dtype, size_t at) {
  if (dtype == B200FP4_DTYPE_BF16) return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[at]);
  if (dtype == B200FP4_DTYPE_F16) return __half2float(static_cast<const __half*>(p)[at]);
  return static_cast<const float*>(p)[at];
}

}  // namespace w4
}  // namespace b200fp4
