// Microscaled 4-bit floating point (MXFP4): device helpers shared by the
// quantisers (quant_fp4.cu) and the GEMM (gemm_fp4.cu).
//
// 32 neighbours along K share one power-of-two scale 2^e (a UE8M0 byte e + 127);
// each value is e2m1: 0, 0.5, 1, 1.5, 2, 3, 4, 6 and a sign. The scale is the
// smallest with max|x| <= 7 * 2^e: a value above 6 becomes 6, which is off by at
// most 1, the same half step as between 4 and 6, and normal data lose 3% less
// (2-norm) than with the smallest scale that keeps every value at or below 6, or
// with the exponent of max|x| alone. e is at most 125, so that a finite block (its 6 * 2^e)
// stays finite in bf16: what is above 7 * 2^125 saturates. A block that holds an infinity or a NaN gets
// the scale byte 255 (NaN) and zero codes, so its products are NaN, as they would
// be unquantised.
//
// Two codes a byte, the lower K in the low nibble. Scale bytes lie in 512-byte
// atoms, [row tile of 128][K tile of 128][512]: row r's bytes of the tile's four
// blocks are at 16 (r % 32) + 4 (r / 32). The number of K tiles is even (K padded to
// 256, one GEMM stage), and the bytes past K are 0.
#pragma once

#include "common.cuh"

#include <cuda_fp4.h>

namespace gsb {
namespace f4 {

constexpr int kBlock = 32;

__host__ __device__ constexpr int64_t k_tiles(int64_t K) { return (K + 255) / 256 * 2; }

// Scale byte of a block whose largest magnitude has the fp32 bits `amax` (sign clear, or a NaN's).
__device__ __forceinline__ uint32_t scale_byte(uint32_t amax) {
  // 7 = 1.75 * 2^2: the exponent less two, one more when the mantissa is above 1.75 (the sum
  // then carries into the exponent)
  const int f = (int)((amax + 0x1fffffu) >> 23);
  const uint32_t byte = (uint32_t)(max(2, min(254, f)) - 2);
  return amax >= 0x7f800000u ? 255u : byte;
}

// 2^-e of a scale byte, exact for 0..252. For 255 it means nothing: the caller stores codes of 0.
__device__ __forceinline__ float inv_scale(uint32_t byte) { return __uint_as_float((254u - byte) << 23); }

// 2^e of a scale byte: 2^-127 is a subnormal, 255 is NaN.
__device__ __forceinline__ float scale_value(uint32_t byte) {
  return __uint_as_float(byte == 0u ? 0x400000u : (byte == 255u ? 0x7fc00000u : byte << 23));
}

// Eight values -> eight codes, v[0] in the lowest nibble (round to nearest even, above 6 -> 6).
__device__ __forceinline__ uint32_t pack8(const float (&v)[8]) {
  uint32_t r;
  // a pair's first operand goes to the high nibble
  asm("{\n\t.reg .b8 a, b, c, d;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 c, %6, %5;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 d, %8, %7;\n\t"
      "mov.b32 %0, {a, b, c, d};\n\t}"
      : "=r"(r)
      : "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]));
  return r;
}

// Eight values times `inv` -> eight codes.
__device__ __forceinline__ uint32_t pack8(const float (&v)[8], float inv) {
  float f[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) f[j] = v[j] * inv;
  return pack8(f);
}

// The same of packed pairs.
__device__ __forceinline__ uint32_t pack8(const uint64_t (&v)[4], float inv) {
  float f[8];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const uint64_t p = f32x2_mul(v[j], f32x2_pack(inv, inv));
    f[2 * j] = f32x2_lo(p);
    f[2 * j + 1] = f32x2_hi(p);
  }
  return pack8(f);
}

__device__ __forceinline__ uint32_t max_abs_bits(const float (&v)[8]) {
  uint32_t m = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j) m = max(m, __float_as_uint(v[j]) & 0x7fffffffu);  // NaN bits are above infinity's
  return m;
}

// Largest of four neighbouring lanes (one block of 32 values, eight per lane).
__device__ __forceinline__ uint32_t quad_max(uint32_t v) {
  v = max(v, __shfl_xor_sync(0xffffffffu, v, 1));
  return max(v, __shfl_xor_sync(0xffffffffu, v, 2));
}

__device__ __forceinline__ void unpack8(const uint4& q, float (&v)[8]) {
  const uint32_t p[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float2 f = unpack_bf16x2(p[j]);
    v[2 * j] = f.x;
    v[2 * j + 1] = f.y;
  }
}

// Eight bf16 values as fp32 pairs.
__device__ __forceinline__ void unpack_pairs(const uint4& q, uint64_t (&v)[4]) {
  const uint32_t p[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
  for (int j = 0; j < 4; ++j) v[j] = f32x2_pack_bits(p[j] << 16, p[j] & 0xffff0000u);
}

// fp32 bits of the largest magnitude of eight packed bf16 values (as 16-bit integers, so a
// NaN is above infinity).
__device__ __forceinline__ uint32_t max_abs_bits_bf16(const uint4& q) {
  const uint32_t m = __vmaxu2(__vmaxu2(q.x & 0x7fff7fffu, q.y & 0x7fff7fffu),
                              __vmaxu2(q.z & 0x7fff7fffu, q.w & 0x7fff7fffu));
  return max(m << 16, m & 0xffff0000u);
}

// Eight bf16 values a lane, four lanes a block -> the block's scale byte and the lane's codes.
__device__ __forceinline__ uint32_t quantise8(const uint4& q, uint32_t& codes) {
  const uint32_t byte = scale_byte(quad_max(max_abs_bits_bf16(q)));
  float v[8];
  unpack8(q, v);
  codes = pack8(v, inv_scale(byte));
  if (byte == 255u) codes = 0u;
  return byte;
}

// Offset of the 4-byte word with the scales of row `row`, K tile `kt` (128 values).
__device__ __forceinline__ int64_t sf_word(int64_t row, int64_t kt, int64_t ktiles) {
  const int r = (int)(row & 127);
  return ((row >> 7) * ktiles + kt) * 512 + 16 * (r & 31) + 4 * (r >> 5);
}

// Scale bytes of a whole warp's 256 neighbours (`byte` of each lane's block of four lanes)
// -> the words of both K tiles; `sf` is the first tile's word.
__device__ __forceinline__ void store_scales256(uint32_t byte, int lane, uint8_t* sf) {
  uint32_t word = byte << (8 * ((lane >> 2) & 3));
  word |= __shfl_xor_sync(0xffffffffu, word, 4);
  word |= __shfl_xor_sync(0xffffffffu, word, 8);
  if ((lane & 15) == 0) *reinterpret_cast<uint32_t*>(sf + (lane >> 4) * 512) = word;
}

}  // namespace f4
}  // namespace gsb
