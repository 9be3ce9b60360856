// A tensor's rows in 8 bits and back (pack8.h): q int8 [rows, cols] and one scale
// byte per 64 values of a row, [rows, ceil(cols / 64)], the last block of a row
// being shorter where 64 does not divide cols.
//
// Bound by memory: 2 or 4 bytes of each value one way, 1 + 1/64 the other.  Eight
// lanes hold a block, eight values each: a wave moves 16 bytes (bf16) or 32 (fp32)
// a lane on the wide side, 8 on the packed one, whole lines both ways.
#include "common.h"
#include "pack8.h"

namespace moe {
namespace {

constexpr int kThreads = 256;
constexpr int kLanes = 8;  // of a block

template <typename T> __device__ __forceinline__ void load8(const T* p, float (&v)[8]) {
  if constexpr (sizeof(T) == 2) {
    const u32x4 w = __builtin_nontemporal_load((const u32x4*)p);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = (i & 1) ? bf_hi(w[i >> 1]) : bf_lo(w[i >> 1]);
  } else {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const f32x4 w = __builtin_nontemporal_load((const f32x4*)p + h);
#pragma unroll
      for (int i = 0; i < 4; ++i) v[4 * h + i] = w[i];
    }
  }
}
template <typename T> __device__ __forceinline__ void store8(T* p, const float (&v)[8]) {
  if constexpr (sizeof(T) == 2) {
    u32x4 w;
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = pack_bf2(v[2 * i], v[2 * i + 1]);
    __builtin_nontemporal_store(w, (u32x4*)p);
  } else {
#pragma unroll
    for (int h = 0; h < 2; ++h)
      __builtin_nontemporal_store(f32x4{v[4 * h], v[4 * h + 1], v[4 * h + 2], v[4 * h + 3]},
                                  (f32x4*)p + h);
  }
}

// WHOLE: 64 divides cols and the pointers allow vectors, so block b is 64 values
// from 64 b on.
template <typename T, bool WHOLE>
__global__ __launch_bounds__(kThreads) void pack8_kernel(const T* __restrict__ x, int64_t blocks,
                                                         int cols, int row_blocks,
                                                         uint8_t* __restrict__ q,
                                                         uint8_t* __restrict__ scale) {
  const int g = threadIdx.x % kLanes;
  const int64_t step = (int64_t)gridDim.x * (kThreads / kLanes);
  for (int64_t b = (int64_t)blockIdx.x * (kThreads / kLanes) + threadIdx.x / kLanes; b < blocks;
       b += step) {
    float v[8];
    int64_t at;
    int n = 8;
    if constexpr (WHOLE) {
      at = b * kPack8Block + g * 8;
      load8(x + at, v);
    } else {
      const int64_t row = b / row_blocks;
      const int col = (int)(b - row * row_blocks) * kPack8Block + g * 8;
      at = row * cols + col;
      n = min(8, cols - col);  // none or fewer past the row's end
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = i < n ? (float)x[at + i] : 0.f;
    }
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) m = max(m, __float_as_uint(v[i]) & 0x7fffffffu);
    const uint32_t e = pack8_scale(group_max_key<kLanes>(m));
    const float inv = pack8_inverse(e);
    const u32x2 w = {pack8_four(v[0], v[1], v[2], v[3], inv),
                     pack8_four(v[4], v[5], v[6], v[7], inv)};
    if constexpr (WHOLE) {
      __builtin_nontemporal_store(w, (u32x2*)(q + at));
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (i < n) q[at + i] = (uint8_t)(w[i >> 2] >> (8 * (i & 3)));
    }
    if (g == 0) scale[b] = (uint8_t)e;
  }
}

template <typename T, bool WHOLE>
__global__ __launch_bounds__(kThreads) void unpack8_kernel(const uint8_t* __restrict__ q,
                                                           const uint8_t* __restrict__ scale,
                                                           int64_t blocks, int cols,
                                                           int row_blocks, T* __restrict__ x) {
  const int g = threadIdx.x % kLanes;
  const int64_t step = (int64_t)gridDim.x * (kThreads / kLanes);
  for (int64_t b = (int64_t)blockIdx.x * (kThreads / kLanes) + threadIdx.x / kLanes; b < blocks;
       b += step) {
    const float s = unpack8_scale(scale[b]);
    float v[8];
    if constexpr (WHOLE) {
      const int64_t at = b * kPack8Block + g * 8;
      const u32x2 w = __builtin_nontemporal_load((const u32x2*)(q + at));
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = unpack8(w[i >> 2], i & 3, s);
      store8(x + at, v);
    } else {
      const int64_t row = b / row_blocks;
      const int col = (int)(b - row * row_blocks) * kPack8Block + g * 8;
      const int64_t at = row * cols + col;
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (i < cols - col) x[at + i] = (T)unpack8(q[at + i], 0, s);
    }
  }
}

int check(const void* x, int dtype, int64_t rows, int64_t cols, const void* q, const void* scale,
          const char* who) {
  MOE_REQUIRE(dtype == MOE_DTYPE_BF16 || dtype == MOE_DTYPE_F32, MOE_ERR_DTYPE,
              "%s: dtype %d is neither bf16 nor fp32", who, dtype);
  MOE_REQUIRE(rows >= 0 && cols >= 0, MOE_ERR_ARG, "%s: rows=%lld cols=%lld", who,
              (long long)rows, (long long)cols);
  MOE_REQUIRE(cols < ((int64_t)1 << 31) - 64 && rows < ((int64_t)1 << 40), MOE_ERR_UNSUPPORTED,
              "%s: rows=%lld cols=%lld too large", who, (long long)rows, (long long)cols);
  MOE_REQUIRE(rows == 0 || cols == 0 || (x && q && scale), MOE_ERR_ARG, "%s: null pointer", who);
  MOE_REQUIRE(((uintptr_t)x & (dtype == MOE_DTYPE_BF16 ? 1 : 3)) == 0, MOE_ERR_ALIGN,
              "%s: pointer not aligned to its values", who);
  return MOE_OK;
}

// Up to 32 workgroups of four waves a CU in four rounds; a grid-stride loop past
// that.
int grid_for(int64_t blocks) {
  const int64_t n = (blocks * kLanes + kThreads - 1) / kThreads;
  return (int)(n < 256 * 32 ? n : 256 * 32);
}

template <typename T>
void pack_launch(const void* x, int64_t rows, int cols, void* q, void* scale, hipStream_t st) {
  const int rb = (cols + kPack8Block - 1) / kPack8Block;
  const int64_t blocks = rows * rb;
  const bool whole = cols % kPack8Block == 0 && al16(x) && ((uintptr_t)q & 7) == 0;
  if (whole)
    pack8_kernel<T, true><<<grid_for(blocks), kThreads, 0, st>>>((const T*)x, blocks, cols, rb,
                                                                (uint8_t*)q, (uint8_t*)scale);
  else
    pack8_kernel<T, false><<<grid_for(blocks), kThreads, 0, st>>>((const T*)x, blocks, cols, rb,
                                                                 (uint8_t*)q, (uint8_t*)scale);
}
template <typename T>
void unpack_launch(const void* q, const void* scale, int64_t rows, int cols, void* x,
                   hipStream_t st) {
  const int rb = (cols + kPack8Block - 1) / kPack8Block;
  const int64_t blocks = rows * rb;
  const bool whole = cols % kPack8Block == 0 && al16(x) && ((uintptr_t)q & 7) == 0;
  if (whole)
    unpack8_kernel<T, true><<<grid_for(blocks), kThreads, 0, st>>>(
        (const uint8_t*)q, (const uint8_t*)scale, blocks, cols, rb, (T*)x);
  else
    unpack8_kernel<T, false><<<grid_for(blocks), kThreads, 0, st>>>(
        (const uint8_t*)q, (const uint8_t*)scale, blocks, cols, rb, (T*)x);
}

}  // namespace
}  // namespace moe

using namespace moe;

extern "C" int moe_amd_pack8(const void* x, int dtype, int64_t rows, int64_t cols, void* q,
                             void* scale, void* stream) {
  const int rc = check(x, dtype, rows, cols, q, scale, "pack8");
  if (rc) return rc;
  if (rows == 0 || cols == 0) return MOE_OK;
  if (dtype == MOE_DTYPE_BF16) pack_launch<bf16>(x, rows, (int)cols, q, scale, (hipStream_t)stream);
  else pack_launch<float>(x, rows, (int)cols, q, scale, (hipStream_t)stream);
  return check_launch("pack8");
}

extern "C" int moe_amd_unpack8(const void* q, const void* scale, int64_t rows, int64_t cols,
                               void* x, int dtype, void* stream) {
  const int rc = check(x, dtype, rows, cols, q, scale, "unpack8");
  if (rc) return rc;
  if (rows == 0 || cols == 0) return MOE_OK;
  if (dtype == MOE_DTYPE_BF16)
    unpack_launch<bf16>(q, scale, rows, (int)cols, x, (hipStream_t)stream);
  else
    unpack_launch<float>(q, scale, rows, (int)cols, x, (hipStream_t)stream);
  return check_launch("unpack8");
}
