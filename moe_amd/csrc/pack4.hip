// A matrix's rows in 4 bits and back (pack4.h): batch matrices [n, k], row-major,
// to their tiles, each matrix beginning a tile of its own.
//
// Bound by memory: 2 or 4 bytes of each value one way, 17/32 the other.  A wave
// takes a tile; its lane (row l / 4, piece l % 4) moves the piece's eight columns
// of each of the four blocks in turn, so that four lanes read or write 64 (bf16)
// or 128 consecutive bytes and a wave's 64 codes words are 256 bytes.
// Values to pack come by non-temporal loads: sixteen matrices [1536, 2048] of fp32 take
// 41 us (5.5 TB/s; 56 us otherwise).  Unpacked ones are stored as usual: 35 us (6.6
// TB/s; 80 us by non-temporal stores).  128 matrices, beyond the memory-side cache: fp32
// 359 and 485 us (5.1 and 3.8 TB/s), bf16 268 and 277 us (3.8 and 3.7 TB/s).
#include "common.h"
#include "pack4.h"

namespace moe {
namespace {

constexpr int kThreads = 256;

// Eight values from x on, of which the first `have` exist (the others read as
// zeros); whole pieces at the alignment of the type.
template <typename T>
__device__ __forceinline__ void load8(const T* x, int have, float (&v)[8]) {
  if (have >= 8) {
    typedef uint32_t Raw __attribute__((ext_vector_type(2 * sizeof(T)), aligned(sizeof(T))));
    const Raw r = __builtin_nontemporal_load((const Raw*)x);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if constexpr (sizeof(T) == 2) v[i] = i & 1 ? bf_hi(r[i >> 1]) : bf_lo(r[i >> 1]);
      else v[i] = __uint_as_float(r[i]);
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = i < have ? (float)x[i] : 0.f;
}

template <typename T>
__global__ __launch_bounds__(kThreads) void pack4_kernel(const T* __restrict__ x, int64_t tiles,
                                                         int n, int k, int nt, int kt,
                                                         uint32_t* __restrict__ q,
                                                         uint32_t* __restrict__ scale) {
  const int lane = threadIdx.x & 63, r = lane >> 2, p = lane & 3;
  const int64_t step = (int64_t)gridDim.x * (kThreads / 64);
  for (int64_t t = (int64_t)blockIdx.x * (kThreads / 64) + (threadIdx.x >> 6); t < tiles; t += step) {
    const int64_t rt = t / kt;  // tile rows so far, of all matrices
    const int col0 = (int)(t - rt * kt) * kPack4Cols + p * 8;
    const int64_t m = rt / nt;
    const int row = (int)(rt - m * nt) * kPack4Rows + r;
    const T* at = x + (m * n + row) * k + col0;
    float v[4][8];
#pragma unroll
    for (int b = 0; b < 4; ++b)
      load8(at + b * kPack4Block, row < n ? k - col0 - b * kPack4Block : 0, v[b]);
    uint32_t scales = 0;
#pragma unroll
    for (int b = 0; b < 4; ++b) {
      uint32_t a = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) a = max(a, __float_as_uint(v[b][i]) & 0x7fffffffu);
      const uint32_t e = pack4_scale(group_max_key<4>(a));
      const float inv = pack4_inverse(e);
#pragma unroll
      for (int i = 0; i < 8; ++i) v[b][i] *= inv;
      const uint32_t w = pack4_eight(v[b]);
      q[t * (kPack4Q / 4) + b * 64 + lane] = e == 255u ? 0u : w;
      scales |= e << (8 * b);
    }
    if (p == 0) scale[t * (kPack4S / 4) + r] = scales;
  }
}

template <typename T>
__global__ __launch_bounds__(kThreads) void unpack4_kernel(const uint32_t* __restrict__ q,
                                                           const uint32_t* __restrict__ scale,
                                                           int64_t tiles, int n, int k, int nt,
                                                           int kt, T* __restrict__ x) {
  const int lane = threadIdx.x & 63, r = lane >> 2, p = lane & 3;
  const int64_t step = (int64_t)gridDim.x * (kThreads / 64);
  for (int64_t t = (int64_t)blockIdx.x * (kThreads / 64) + (threadIdx.x >> 6); t < tiles; t += step) {
    const int64_t rt = t / kt;
    const int col0 = (int)(t - rt * kt) * kPack4Cols + p * 8;
    const int64_t m = rt / nt;
    const int row = (int)(rt - m * nt) * kPack4Rows + r;
    if (row >= n) continue;
    T* at = x + (m * n + row) * k + col0;
    const uint32_t scales = scale[t * (kPack4S / 4) + r];
    uint32_t w[4];
#pragma unroll
    for (int b = 0; b < 4; ++b) w[b] = q[t * (kPack4Q / 4) + b * 64 + lane];
#pragma unroll
    for (int b = 0; b < 4; ++b) {
      const int have = k - col0 - b * kPack4Block;
      const float s = unpack4_scale(scales >> (8 * b) & 0xffu);
      typedef uint32_t Raw __attribute__((ext_vector_type(2 * sizeof(T)), aligned(sizeof(T))));
      Raw o;
      if constexpr (sizeof(T) == 2) {
        o = unpack4_eight(w[b], s);
      } else {
        const f32x2 v0 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[b], s, 0);
        const f32x2 v1 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[b], s, 1);
        const f32x2 v2 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[b], s, 2);
        const f32x2 v3 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[b], s, 3);
        const float f[8] = {v0[0], v0[1], v1[0], v1[1], v2[0], v2[1], v3[0], v3[1]};
#pragma unroll
        for (int i = 0; i < 8; ++i) o[i] = __float_as_uint(f[i]);
      }
      if (have >= 8) {
        *(Raw*)(at + b * kPack4Block) = o;
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (i < have) {
            if constexpr (sizeof(T) == 2)
              at[b * kPack4Block + i] =
                  __builtin_bit_cast(bf16, (uint16_t)(i & 1 ? o[i >> 1] >> 16 : o[i >> 1] & 0xffffu));
            else at[b * kPack4Block + i] = __uint_as_float(o[i]);
          }
      }
    }
  }
}

int check(const void* x, int dtype, int64_t batch, int64_t n, int64_t k, const void* q,
          const void* scale, const char* who) {
  MOE_REQUIRE(dtype == MOE_DTYPE_BF16 || dtype == MOE_DTYPE_F32, MOE_ERR_DTYPE,
              "%s: dtype %d is neither bf16 nor fp32", who, dtype);
  MOE_REQUIRE(batch >= 0 && n >= 0 && k >= 0, MOE_ERR_ARG, "%s: batch=%lld n=%lld k=%lld", who,
              (long long)batch, (long long)n, (long long)k);
  constexpr int64_t most = ((int64_t)1 << 31) - kPack4Cols;
  MOE_REQUIRE(n < most && k < most && batch < most, MOE_ERR_UNSUPPORTED,
              "%s: batch=%lld n=%lld k=%lld too large", who, (long long)batch, (long long)n,
              (long long)k);
  if (batch == 0 || n == 0 || k == 0) return MOE_OK;
  // (a matrix has at most 2^27 by 2^24 tiles here)
  MOE_REQUIRE(pack4_tiles(n, k) <= ((int64_t)1 << 40) / batch, MOE_ERR_UNSUPPORTED,
              "%s: batch=%lld n=%lld k=%lld too large", who, (long long)batch, (long long)n,
              (long long)k);
  MOE_REQUIRE(x && q && scale, MOE_ERR_ARG, "%s: null pointer", who);
  MOE_REQUIRE(((uintptr_t)x & (dtype == MOE_DTYPE_BF16 ? 1 : 3)) == 0 && ((uintptr_t)q & 3) == 0 &&
                  ((uintptr_t)scale & 3) == 0,
              MOE_ERR_ALIGN, "%s: x not aligned to its values, or q or scale not to 4 bytes", who);
  return MOE_OK;
}

// A wave a tile, at most 32 workgroups for each of 256 CUs.
int grid_for(int64_t tiles) {
  const int64_t g = (tiles + kThreads / 64 - 1) / (kThreads / 64);
  return (int)(g < 256 * 32 ? g : 256 * 32);
}

}  // namespace
}  // namespace moe

using namespace moe;

extern "C" int moe_amd_pack4(const void* x, int dtype, int64_t batch, int64_t n, int64_t k, void* q,
                             void* scale, void* stream) {
  const int rc = check(x, dtype, batch, n, k, q, scale, "pack4");
  if (rc) return rc;
  if (batch == 0 || n == 0 || k == 0) return MOE_OK;
  const int nt = (int)((n + kPack4Rows - 1) / kPack4Rows), kt = (int)((k + kPack4Cols - 1) / kPack4Cols);
  const int64_t tiles = batch * nt * kt;
  const hipStream_t st = (hipStream_t)stream;
  if (dtype == MOE_DTYPE_BF16)
    pack4_kernel<bf16><<<grid_for(tiles), kThreads, 0, st>>>((const bf16*)x, tiles, (int)n, (int)k, nt,
                                                            kt, (uint32_t*)q, (uint32_t*)scale);
  else
    pack4_kernel<float><<<grid_for(tiles), kThreads, 0, st>>>((const float*)x, tiles, (int)n, (int)k,
                                                             nt, kt, (uint32_t*)q, (uint32_t*)scale);
  return check_launch("pack4");
}

extern "C" int moe_amd_unpack4(const void* q, const void* scale, int64_t batch, int64_t n, int64_t k,
                               void* x, int dtype, void* stream) {
  const int rc = check(x, dtype, batch, n, k, q, scale, "unpack4");
  if (rc) return rc;
  if (batch == 0 || n == 0 || k == 0) return MOE_OK;
  const int nt = (int)((n + kPack4Rows - 1) / kPack4Rows), kt = (int)((k + kPack4Cols - 1) / kPack4Cols);
  const int64_t tiles = batch * nt * kt;
  const hipStream_t st = (hipStream_t)stream;
  if (dtype == MOE_DTYPE_BF16)
    unpack4_kernel<bf16><<<grid_for(tiles), kThreads, 0, st>>>(
        (const uint32_t*)q, (const uint32_t*)scale, tiles, (int)n, (int)k, nt, kt, (bf16*)x);
  else
    unpack4_kernel<float><<<grid_for(tiles), kThreads, 0, st>>>(
        (const uint32_t*)q, (const uint32_t*)scale, tiles, (int)n, (int)k, nt, kt, (float*)x);
  return check_launch("unpack4");
}
