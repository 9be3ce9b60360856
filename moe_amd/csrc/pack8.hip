// A tensor's rows in 8 bits and back (pack8.h): q int8 [rows, cols] and one scale
// byte per 64 values of a row, [rows, ceil(cols / 64)], the last block of a row
// being shorter where 64 does not divide cols.
//
// Bound by memory: 2 or 4 bytes of each value one way, 1 + 1/64 the other.
#include "common.h"
#include "pack8.h"

namespace moe {
namespace {

constexpr int kThreads = 256;

// 64 divides cols and the pointers allow vectors: block b is 64 values from 64 b
// on, 16 bytes of them a lane on the wide side.  A thread has kAhead such pieces
// in flight.
constexpr int kAhead = 4;
template <typename T> constexpr int kPer = 16 / sizeof(T);       // values a lane
template <typename T> constexpr int kOf = kPack8Block / kPer<T>;  // lanes a block
template <typename T>
__global__ __launch_bounds__(kThreads) void pack8_kernel(const T* __restrict__ x, int64_t blocks,
                                                         uint8_t* __restrict__ q,
                                                         uint8_t* __restrict__ scale) {
  constexpr int V = kPer<T>, L = kOf<T>;
  const int64_t pieces = blocks * L, step = (int64_t)gridDim.x * kThreads;
  for (int64_t i0 = (int64_t)blockIdx.x * kThreads + threadIdx.x; i0 < pieces;
       i0 += kAhead * step) {
    u32x4 w[kAhead];
#pragma unroll
    for (int k = 0; k < kAhead; ++k)
      if (i0 + k * step < pieces) w[k] = __builtin_nontemporal_load((const u32x4*)(x + (i0 + k * step) * V));
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      const int64_t i = i0 + k * step;
      if (i >= pieces) break;  // all lanes of a block alike
      uint32_t m;
      if constexpr (V == 8) {
        m = w[k][0] & 0x7fff7fffu;
#pragma unroll
        for (int j = 1; j < 4; ++j) m = max_u16x2(m, w[k][j] & 0x7fff7fffu);
        m = max(m << 16, m & 0xffff0000u);
      } else {
        m = max(max(w[k][0] & 0x7fffffffu, w[k][1] & 0x7fffffffu),
                max(w[k][2] & 0x7fffffffu, w[k][3] & 0x7fffffffu));
      }
      const uint32_t e = pack8_scale(group_max_key<L>(m));
      const float inv = pack8_inverse(e);
      if constexpr (V == 8) {
        __builtin_nontemporal_store(pack8_bf16x8(w[k], inv), (u32x2*)q + i);
      } else {
        const uint32_t v = pack8_four(__uint_as_float(w[k][0]), __uint_as_float(w[k][1]),
                                      __uint_as_float(w[k][2]), __uint_as_float(w[k][3]), inv);
        __builtin_nontemporal_store(e == 255u ? 0u : v, (uint32_t*)q + i);  // no NaN's payload
      }
      if (i % L == 0) scale[i / L] = (uint8_t)e;
    }
  }
}

template <typename T>
__global__ __launch_bounds__(kThreads) void unpack8_kernel(const uint8_t* __restrict__ q,
                                                           const uint8_t* __restrict__ scale,
                                                           int64_t blocks, T* __restrict__ x) {
  constexpr int V = kPer<T>, L = kOf<T>;
  const int64_t pieces = blocks * L, step = (int64_t)gridDim.x * kThreads;
  for (int64_t i0 = (int64_t)blockIdx.x * kThreads + threadIdx.x; i0 < pieces;
       i0 += kAhead * step) {
    uint32_t w[kAhead][V / 4], e[kAhead];
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      const int64_t i = i0 + k * step;
      if (i >= pieces) break;
      if constexpr (V == 8) {
        const u32x2 v = __builtin_nontemporal_load((const u32x2*)q + i);
        w[k][0] = v[0];
        w[k][1] = v[1];
      } else {
        w[k][0] = __builtin_nontemporal_load((const uint32_t*)q + i);
      }
      e[k] = scale[i / L];
    }
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      const int64_t i = i0 + k * step;
      if (i >= pieces) break;
      const float s = unpack8_scale(e[k]);
      float v[V];
#pragma unroll
      for (int j = 0; j < V; ++j) v[j] = unpack8(w[k][j >> 2], j & 3, s);
      u32x4 o;
#pragma unroll
      for (int j = 0; j < 4; ++j)
        o[j] = V == 8 ? pack_bf2(v[(2 * j) % V], v[(2 * j + 1) % V]) : __float_as_uint(v[j]);
      __builtin_nontemporal_store(o, (u32x4*)(x + i * V));
    }
  }
}

// Rows of any length and pointers of any alignment: eight lanes a block, eight
// values a lane, one at a time.
template <typename T>
__global__ __launch_bounds__(kThreads) void pack8_any_kernel(const T* __restrict__ x,
                                                             int64_t blocks, int cols,
                                                             int row_blocks,
                                                             uint8_t* __restrict__ q,
                                                             uint8_t* __restrict__ scale) {
  const int g = threadIdx.x % 8;
  const int64_t step = (int64_t)gridDim.x * (kThreads / 8);
  for (int64_t b = (int64_t)blockIdx.x * (kThreads / 8) + threadIdx.x / 8; b < blocks; b += step) {
    const int64_t row = b / row_blocks;
    const int col = (int)(b - row * row_blocks) * kPack8Block + g;
    const int64_t at = row * cols + col;
    float v[8];
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      v[i] = col + 8 * i < cols ? (float)x[at + 8 * i] : 0.f;
      m = max(m, __float_as_uint(v[i]) & 0x7fffffffu);
    }
    const uint32_t e = pack8_scale(group_max_key<8>(m));
    const float inv = pack8_inverse(e);
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (col + 8 * i < cols) q[at + 8 * i] = e == 255u ? 0 : (uint8_t)pack8_one(v[i], inv);
    if (g == 0) scale[b] = (uint8_t)e;
  }
}

template <typename T>
__global__ __launch_bounds__(kThreads) void unpack8_any_kernel(const uint8_t* __restrict__ q,
                                                               const uint8_t* __restrict__ scale,
                                                               int64_t blocks, int cols,
                                                               int row_blocks,
                                                               T* __restrict__ x) {
  const int g = threadIdx.x % 8;
  const int64_t step = (int64_t)gridDim.x * (kThreads / 8);
  for (int64_t b = (int64_t)blockIdx.x * (kThreads / 8) + threadIdx.x / 8; b < blocks; b += step) {
    const int64_t row = b / row_blocks;
    const int col = (int)(b - row * row_blocks) * kPack8Block + g;
    const int64_t at = row * cols + col;
    const float s = unpack8_scale(scale[b]);
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (col + 8 * i < cols) x[at + 8 * i] = (T)unpack8(q[at + 8 * i], 0, s);
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

// Workgroups for n threads' work, at most 32 for each of 256 CUs.
int grid_for(int64_t n) {
  n = (n + kThreads - 1) / kThreads;
  return (int)(n < 256 * 32 ? n : 256 * 32);
}

bool whole_blocks(int cols, const void* x, const void* q) {
  return cols % kPack8Block == 0 && al16(x) && ((uintptr_t)q & 7) == 0;
}

template <typename T>
void pack_launch(const void* x, int64_t rows, int cols, void* q, void* scale, hipStream_t st) {
  const int rb = (cols + kPack8Block - 1) / kPack8Block;
  const int64_t blocks = rows * rb;
  if (whole_blocks(cols, x, q))
    pack8_kernel<T><<<grid_for((blocks * kOf<T> + kAhead - 1) / kAhead), kThreads, 0, st>>>(
        (const T*)x, blocks, (uint8_t*)q, (uint8_t*)scale);
  else
    pack8_any_kernel<T><<<grid_for(blocks * 8), kThreads, 0, st>>>((const T*)x, blocks, cols, rb,
                                                                  (uint8_t*)q, (uint8_t*)scale);
}
template <typename T>
void unpack_launch(const void* q, const void* scale, int64_t rows, int cols, void* x,
                   hipStream_t st) {
  const int rb = (cols + kPack8Block - 1) / kPack8Block;
  const int64_t blocks = rows * rb;
  if (whole_blocks(cols, x, q))
    unpack8_kernel<T><<<grid_for((blocks * kOf<T> + kAhead - 1) / kAhead), kThreads, 0, st>>>(
        (const uint8_t*)q, (const uint8_t*)scale, blocks, (T*)x);
  else
    unpack8_any_kernel<T><<<grid_for(blocks * 8), kThreads, 0, st>>>(
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
