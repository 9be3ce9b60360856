// Weights in 4 bits: for 32 consecutive values v of a row a power of two s and,
// for each value, a sign (bit 3) and the magnitude |v| / s rounded to one of
// 0, 1/2, 1, 3/2, 2, 3, 4, 6 (bits 0 to 2), halves to the even code: the E2M1
// and E8M0 of the MX formats, which v_cvt_scalef32_pk_bf16_fp4 turns into a
// pair of bf16 values in one instruction.  Every product is exact in bf16 (and
// fp32) but for the largest, which are infinite there.
//
// pack4 takes as s the smallest power of two that is at least 2^-125 and has
// max|v| <= 7 s.  What lies between 6 s and 7 s becomes 6 s, off by no more than
// the half step of s that values from 4 s to 6 s are off by; of normal values
// the root mean square error is 0.112 of theirs (0.115 with 6 s as the limit, or
// with 8 s, which cuts more off).  The scale byte is s's biased exponent, 2 to
// 253; 255 marks a block with a value that is not finite, which is restored as
// NaN whole.
//
// Codes and scales lie in tiles of 16 rows by 128 columns, zeros where the matrix
// ends inside a tile, a tile's codes being 1 KB in the order in which a wave's
// lanes (row l % 16, block l / 16) take the weight operand of the MFMA: a wave
// reads its weights as whole lines, 16 bytes a lane, without LDS.
//   q      [N/16][K/128][block 4][row 16][16 bytes]
//   scale  [N/16][K/128][row 16][block 4]
#pragma once
#include "wave_topk.h"

namespace moe {

constexpr int kPack4Block = 32;
constexpr int kPack4Rows = 16;    // of a tile
constexpr int kPack4Cols = 128;
constexpr int kPack4Q = 1024;     // bytes of a tile's codes
constexpr int kPack4S = 64;       // and of its scales

static inline int64_t pack4_tiles(int64_t n, int64_t k) {
  return (n + kPack4Rows - 1) / kPack4Rows * ((k + kPack4Cols - 1) / kPack4Cols);
}

// The scale byte from the bits of the block's largest |v| as fp32 (NaN above
// all).  7 2^k >= 1.m 2^e: k = e - 2, or e - 1 where 1.m > 7/4 (m > 0x600000, which
// the addition carries into the exponent).
__device__ __forceinline__ uint32_t pack4_scale(uint32_t absmax_bits) {
  const int e = (int)((absmax_bits + 0x1fffffu) >> 23) - 2;
  return absmax_bits >= 0x7f800000u ? 255u : (uint32_t)(e < 2 ? 2 : e);
}
// 1 / s, or 0 for a block that is not finite.
__device__ __forceinline__ float pack4_inverse(uint32_t scale) {
  return scale == 255u ? 0.f : __uint_as_float((254u - scale) << 23);
}
// Eight values in units of s, |v| <= 7 -> eight codes, the first one lowest.
__device__ __forceinline__ uint32_t pack4_eight(const float (&v)[8]) {
  uint32_t q = 0;
  q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, v[0], v[1], 1.f, 0);
  q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, v[2], v[3], 1.f, 1);
  q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, v[4], v[5], 1.f, 2);
  q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, v[6], v[7], 1.f, 3);
  return q;
}

// A scale byte as the operand of the conversions, which read its exponent only (255: NaN).
__device__ __forceinline__ float unpack4_scale(uint32_t byte) { return __uint_as_float(byte << 23); }
// Eight codes -> eight bf16 values, exact.
__device__ __forceinline__ u32x4 unpack4_eight(uint32_t q, float s) {
  return u32x4{
      __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(q, s, 0)),
      __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(q, s, 1)),
      __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(q, s, 2)),
      __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(q, s, 3))};
}

}  // namespace moe
