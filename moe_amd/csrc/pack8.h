// Activations in 8 bits: for 64 consecutive values v of a row a power of two s
// and the integers q = rint(v / s), halves to even.  s is the smallest power of
// two that is at least 2^-126 and has max|v| <= 127 s, so q * s is exact in bf16
// (7 bits) and in fp32, whoever restores it (past 127/128 2^128 it is 2^128,
// infinity in both).  (An s of max|v| / 127 would halve
// the step at best, sqrt(2) on average, and make the restored value a rounding
// of its own.)  The scale byte is s's biased exponent, 1 .. 249; 255 marks a
// block with a value that is not finite, whose q are 0: it is restored as
// 0 * inf, NaN in every place, rather than hidden.
#pragma once
#include "wave_topk.h"

namespace moe {

constexpr int kPack8Block = 64;

typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));

// The scale byte from the bits of the block's largest |v| as fp32 (NaN above
// all).  2^k >= a / 127 for a = 1.m 2^e: k = e - 6, or e - 5 where 1.m > 127/64
// (m > 0x7e0000, which the addition carries into the exponent).
__device__ __forceinline__ uint32_t pack8_scale(uint32_t absmax_bits) {
  const int e = (int)((absmax_bits + 0x1ffffu) >> 23) - 6;
  return absmax_bits >= 0x7f800000u ? 255u : (uint32_t)(e < 1 ? 1 : e);
}
// 1 / s, or 0 for a block that is not finite.
__device__ __forceinline__ float pack8_inverse(uint32_t scale) {
  return scale == 255u ? 0.f : __uint_as_float((254u - scale) << 23);
}
// q in the low byte: v / s is exact, and adding 1.5 2^23 rounds it to an
// integer, halves to even, whose two's complement ends the sum's bits.  In a
// block that is not finite: 0 for finite v and for 0 * inf, whose NaN ends in a
// zero byte, and for a NaN of bf16, the low half of whose bits is 0; a NaN of
// fp32 keeps its payload, so packing from fp32 sets that block's q to 0 itself.
__device__ __forceinline__ uint32_t pack8_one(float v, float inv) {
  return __float_as_uint(__builtin_fmaf(v, inv, 12582912.f));
}
__device__ __forceinline__ uint32_t pack8_four(float a, float b, float c, float d, float inv) {
  const uint32_t lo = __builtin_amdgcn_perm(pack8_one(b, inv), pack8_one(a, inv), 0x0c0c0400u);
  const uint32_t hi = __builtin_amdgcn_perm(pack8_one(d, inv), pack8_one(c, inv), 0x0c0c0400u);
  return hi << 16 | lo;
}
// Eight bf16 values (four pairs) -> eight bytes.
__device__ __forceinline__ u32x2 pack8_bf16x8(const u32x4& v, float inv) {
  return u32x2{pack8_four(bf_lo(v[0]), bf_hi(v[0]), bf_lo(v[1]), bf_hi(v[1]), inv),
               pack8_four(bf_lo(v[2]), bf_hi(v[2]), bf_lo(v[3]), bf_hi(v[3]), inv)};
}

__device__ __forceinline__ uint32_t max_u16x2(uint32_t a, uint32_t b) {
  return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2, a),
                                                                __builtin_bit_cast(u16x2, b)));
}
// Two blocks of 64 bf16 values, eight of each (a, b) in each of eight consecutive
// lanes -> their bytes {a, b} and their scale bytes (a's low).  Magnitudes
// compare as 16-bit integers, the two blocks' in one register.
__device__ __forceinline__ u32x4 pack8_two_blocks(const u32x4& a, const u32x4& b,
                                                  uint32_t& scales) {
  uint32_t ma = a[0] & 0x7fff7fffu, mb = b[0] & 0x7fff7fffu;
#pragma unroll
  for (int w = 1; w < 4; ++w) {
    ma = max_u16x2(ma, a[w] & 0x7fff7fffu);
    mb = max_u16x2(mb, b[w] & 0x7fff7fffu);
  }
  uint32_t m = max_u16x2(__builtin_amdgcn_perm(mb, ma, 0x05040100u),
                         __builtin_amdgcn_perm(mb, ma, 0x07060302u));
  group_steps<8>([&](auto c) { m = max_u16x2(m, dpp_u32<decltype(c)::value>(m)); });
  const uint32_t ea = pack8_scale(m << 16), eb = pack8_scale(m & 0xffff0000u);
  scales = ea | eb << 8;
  const u32x2 qa = pack8_bf16x8(a, pack8_inverse(ea)), qb = pack8_bf16x8(b, pack8_inverse(eb));
  return u32x4{qa[0], qa[1], qb[0], qb[1]};
}

__device__ __forceinline__ float unpack8_scale(uint32_t scale) { return __uint_as_float(scale << 23); }
// Value `byte` (0 .. 3) of four packed ones.
__device__ __forceinline__ float unpack8(uint32_t q, int byte, float scale) {
  return (float)(int8_t)(q >> (8 * byte)) * scale;
}

}  // namespace moe
