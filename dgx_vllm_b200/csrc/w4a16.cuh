// Weight-only NVFP4: 4-bit weights, 16-bit activations.  The packed weight, its decoding, and what the kernels over it share.
//
// value(n, k) = e2m1(code[n, k]) * e4m3(scale[n, k / 16]) * g.  A code has two significant bits and a scale four, so that their product
// is exact in bf16 and in f16: the operand of a 16-bit matrix instruction loses nothing, and the sums are f32.
//
// Packed weight: units of 16 rows x 128 of k, 1152 bytes, [matrix][row tile][k / 128][unit].  A unit is laid out for the 16x8x16 matrix
// instruction, whose lane l holds rows l / 4 and l / 4 + 8 and four k of each: with the k of an instruction taken from four blocks of 16,
// lane l needs block l % 4 only, so it converts one scale a row for four instructions, and its operands of a whole block are 16
// neighbouring bytes:
//   codes   [half: 64 of k][lane][16 bytes: row l / 4, k 0..7 | k 8..15 | row l / 4 + 8, k 0..7 | k 8..15]
//   scales  [lane][4 bytes: half 0 row l / 4, row l / 4 + 8 | half 1 likewise]
// Both are read with one coalesced load a lane.  A word's eight codes are spread over its halves (even k low, odd k high) so that a
// pair becomes two 16-bit values by a shift and a mask: the magnitude's three bits land on the lowest exponent bits and the highest
// mantissa bit, subnormal 0.5 included, which makes it the code's value times 2^-126 (bf16) or 2^-14 (f16).  Bits of a half:
//   pair 0: sign 15, magnitude 8..6    1: 12, 5..3    2: 13, 2..0    3: 14, 11..9
// The scale, raised by 2^119 (bf16) or 2^7 (f16), brings the product to value * 2^-7 / g; 2^7 goes with g.
// Negative scales give their sign to their codes when the weight is packed.
#pragma once

#include "common.cuh"

namespace b200fp4 {
namespace w4 {

constexpr int kUnitBytes = 1152, kUnitScales = 1024, kUnitK = 128, kTileRows = 16;
constexpr float kOutScale = 128.f;

__host__ __device__ __forceinline__ int64_t tiles_of(int64_t rows) { return (rows + kTileRows - 1) / kTileRows; }
__host__ __device__ __forceinline__ int64_t units_of(int64_t K) { return (K + kUnitK - 1) / kUnitK; }

template <typename T>
__device__ __forceinline__ uint32_t mul2(uint32_t a, uint32_t b);
template <>
__device__ __forceinline__ uint32_t mul2<__nv_bfloat16>(uint32_t a, uint32_t b) {
  const __nv_bfloat162 r = __hmul2(*reinterpret_cast<const __nv_bfloat162*>(&a), *reinterpret_cast<const __nv_bfloat162*>(&b));
  return *reinterpret_cast<const uint32_t*>(&r);
}
template <>
__device__ __forceinline__ uint32_t mul2<__half>(uint32_t a, uint32_t b) {
  const __half2 r = __hmul2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b));
  return *reinterpret_cast<const uint32_t*>(&r);
}

// Eight codes -> four pairs of 16-bit values, times 2^-126 (bf16) or 2^-14 (f16)
template <typename T>
__device__ __forceinline__ void codes_to_pairs(uint32_t w, uint32_t (&p)[4]);
template <>
__device__ __forceinline__ void codes_to_pairs<__nv_bfloat16>(uint32_t w, uint32_t (&p)[4]) {
  p[0] = w & 0x81C081C0u;
  p[1] = (w << 3) & 0x81C081C0u;
  p[2] = ((w << 6) & 0x01C001C0u) | ((w << 2) & 0x80008000u);
  p[3] = ((w >> 3) & 0x01C001C0u) | ((w << 1) & 0x80008000u);
}
template <>
__device__ __forceinline__ void codes_to_pairs<__half>(uint32_t w, uint32_t (&p)[4]) {
  p[0] = ((w << 3) & 0x0E000E00u) | (w & 0x80008000u);
  p[1] = ((w << 6) & 0x0E000E00u) | ((w << 3) & 0x80008000u);
  p[2] = ((w << 9) & 0x0E000E00u) | ((w << 2) & 0x80008000u);
  p[3] = (w & 0x0E000E00u) | ((w << 1) & 0x80008000u);
}

// The scales of rows l / 4 (lo) and l / 4 + 8 (hi) for one half of a unit, each twice in a register, raised as above
template <typename T>
__device__ __forceinline__ void scales_of(uint32_t bytes, int half, uint32_t& lo, uint32_t& hi);
template <>
__device__ __forceinline__ void scales_of<__nv_bfloat16>(uint32_t bytes, int half, uint32_t& lo, uint32_t& hi) {
  const uint32_t raw = prmt(bytes, 0u, half ? 0x4342u : 0x4140u) << 4;                      // scale * 2^-120
  const uint32_t s = mul2<__nv_bfloat16>(mul2<__nv_bfloat16>(raw, 0x7F007F00u), 0x77807780u);      // * 2^127 * 2^112
  lo = prmt(s, s, 0x1010u);
  hi = prmt(s, s, 0x3232u);
}
template <>
__device__ __forceinline__ void scales_of<__half>(uint32_t bytes, int half, uint32_t& lo, uint32_t& hi) {
  const uint32_t raw = prmt(bytes, 0u, half ? 0x3424u : 0x1404u) >> 1;                      // scale * 2^-8
  const uint32_t s = mul2<__half>(raw, 0x78007800u);                                        // * 2^15
  lo = prmt(s, s, 0x1010u);
  hi = prmt(s, s, 0x3232u);
}

template <typename T>
__device__ __forceinline__ void mma_16x8x16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void mma_16x8x16<__nv_bfloat16>(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                                           uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void mma_16x8x16<__half>(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                                    uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

}  // namespace w4
}  // namespace b200fp4
