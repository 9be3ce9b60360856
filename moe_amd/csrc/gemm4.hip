// Grouped products of the expert layer on a bank in 4 bits (gfx950), forward
// only, bf16 rows: the routed rows of each expert, as the permutation sorted
// them, times its packed weights (pack4.h).
//
//   gemm4_kernel<BR, true>   act [S,I] = silu(x Wg^T) * (x Wu^T), x gathered by token
//   gemm4_kernel<BR, false>  y [S,H] = act W2^T, in 16-bit blocks
//   combine16_kernel         out [T,H] = sum_k w[t,k] y[row of (t,k)]
//
// A workgroup owns BR rows by 256 weight rows (gate and up: 128 features of
// each), a wave all its rows by 64 weight rows of its own.  So no weight is
// wanted by two waves: each goes from memory to its lane's registers, 16 bytes of
// codes a load and whole lines a wave, and becomes an MFMA operand there by four
// conversions for eight values; converted or not, weights never pass
// through LDS, which holds rows only.  MFMA v_mfma_f32_32x32x16_bf16: weights as
// A (a lane's accumulators hold four consecutive columns of one row), rows as B.
// The contraction runs in the order of the tiles' blocks: lane half h of step j
// takes columns 32 h + 8 j of a stage's 64, of both operands alike.
//
// Rows come by LDS DMA, 64 columns a stage (128-byte lines, 16-byte chunks
// XOR-swizzled by row: no bank conflicts), into a ring of four slots, three stages
// in flight; weights D stage pairs ahead, in registers.  Loads past the end of the
// contraction are issued all the same, from empty descriptors (zeros, no memory
// access), so that the wait counts hold in every stage.
//
// act is rounded to bf16 once.  y is held in 16 bits a value with a power of two for
// 64 columns of a row: as small as bf16, but within 2^-15 of the block's largest
// value instead of 2^-9 of each (three roundings of bf16 size in a row would
// show: 1.7 times the error of one); a block with a value that is not finite is
// NaN whole.  Each output is rounded once.
//
// Reference: transformers/integrations/moe.py:377-478.
#include "common.h"
#include "pack4.h"

namespace moe {
namespace {

constexpr int BK = 64;     // columns of the contraction a stage
constexpr int BC = 256;    // weight rows of a workgroup's tile
constexpr int NSLOT = 4;   // stages of rows in LDS
constexpr int kBlock16 = 64;  // columns of a block of y

template <int BR> constexpr int kSlot = BR * BK * 2;  // bytes

struct Gemm4Args {
  const bf16* x;         // hidden states [T,H] (gate/up) or act [S,I]
  const char *q, *s;     // codes and scales of the bank
  const int* row_src;    // [S] flat entry of a sorted row
  const int* tile_count; // row tiles
  const int4* tile_info; // {expert, first row, end row, 0} of each
  bf16* act;             // [S,I]
  int16_t* y;            // [S,H] and its scale bytes [S,H/64]
  uint8_t* ys;
  int64_t T;
  int K;                 // contraction
  int N;                 // output columns
  int kt;                // tiles along the contraction
  int nt;                // tile rows of an expert
  int n_ct;
  uint32_t tok_mul;      // n / top_k == (n * tok_mul) >> tok_shift
  int tok_shift;
};

constexpr uint32_t kOOB = 0x80000000u;  // offset that always reads as zero
typedef __attribute__((address_space(3))) void lds_void_t;
typedef __attribute__((address_space(3))) char lds_char_t;

__device__ __forceinline__ void dma16(__amdgpu_buffer_rsrc_t r, uint32_t voff, void* lds) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (lds_void_t*)lds, 16, voff, 0, 0, 0);
}
// s_waitcnt with vmcnt(n), lgkmcnt(0).
constexpr int wait_imm(int n) { return (n & 15) | (7 << 4) | (((n >> 4) & 3) << 14); }

// 1 / (1 + e^-x) from the hardware's exponential and reciprocal (1 ulp each).
__device__ __forceinline__ float fast_sigmoid(float x) {
  return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(x * -1.44269504088896341f));
}

// The biased exponent of a block's power of two from the bits of its largest |v|:
// |v| < 2^15 of it.  255: a value is not finite.
__device__ __forceinline__ uint32_t block16_scale(uint32_t absmax_bits) {
  const int e = (int)(absmax_bits >> 23) - 14;
  return absmax_bits >= 0x7f800000u ? 255u : (uint32_t)(e < 1 ? 1 : e);
}

template <int BR, bool GATE, int D>
__global__ __launch_bounds__(256, BR == 256 ? 1 : 2) void gemm4_kernel(Gemm4Args p) {
  constexpr int TJ = BR / 32;   // row sub-tiles, all of them every wave's
  constexpr int RPW = BR / 32;  // 1 KB DMA blocks of a stage's rows per wave
  constexpr int W = 6;          // loads of a pair of stages' weights
  constexpr int NB = D + 1;     // weight buffers
  static_assert(2 * RPW + D * W <= 63, "vmcnt");
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wid = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int l32 = lane & 31, hl = lane >> 5;

  // The tiles are cut into eight ranges, one an XCD, so that the tiles that run at
  // a time share rows and weights in its L2.
  const int n_tiles = *p.tile_count * p.n_ct;
  const int xcd = blockIdx.x & 7, stride = gridDim.x >> 3, chunk = (n_tiles + 7) >> 3;
  const int t_end = min(n_tiles, (xcd + 1) * chunk);
  const int nk = (p.K + BK - 1) / BK, np = p.kt;
  const uint32_t ebytes = (uint32_t)p.nt * p.kt * kPack4Q, sbytes = (uint32_t)p.nt * p.kt * kPack4S;

  const uint32_t lds0 = (uint32_t)(uintptr_t)(const lds_char_t*)smem;
  auto lds_at = [](uint32_t a) { return (const lds_char_t*)(uintptr_t)a; };
  uint32_t b_off[4];  // of sub-step j: row l32, chunk 4 hl + j
#pragma unroll
  for (int j = 0; j < 4; ++j)
    b_off[j] = lds0 + l32 * 128 + (((4 * hl + j) ^ ((l32 >> 1) & 7)) << 4);

  struct Pair {  // a pair of stages' weights: [column sub-tile][stage]
    u32x4 q[2][2];
    uint32_t s[2];
  };

  for (int t = xcd * chunk + (int)(blockIdx.x >> 3); t < t_end; t += stride) {
    const int ct = __builtin_amdgcn_readfirstlane(t % p.n_ct);
    const int4 ti = p.tile_info[t / p.n_ct];
    const int e = __builtin_amdgcn_readfirstlane(ti.x);
    const int row0 = __builtin_amdgcn_readfirstlane(ti.y);
    const int row_end = __builtin_amdgcn_readfirstlane(ti.z);

    // ------------------------------------------------------------ operands
    const char* rptr = (const char*)(GATE ? p.x : p.x + (int64_t)row0 * p.K);
    const uint32_t rbytes =
        GATE ? (uint32_t)(p.T * p.K * 2) : (uint32_t)((int64_t)min(row_end - row0, BR) * p.K * 2);
    uint32_t roff[RPW];
#pragma unroll
    for (int i = 0; i < RPW; ++i) {
      const int f = (wid + 4 * i) * 8 + (lane >> 3);
      const uint32_t c = ((lane & 7) ^ ((f >> 1) & 7)) * 16;
      const bool there = row0 + f < row_end;
      int r = f;
      if constexpr (GATE) {
        const int src = p.row_src[there ? row0 + f : row0];
        r = (int)(((uint64_t)(uint32_t)src * p.tok_mul) >> p.tok_shift);
      }
      roff[i] = there ? (uint32_t)r * (uint32_t)(p.K * 2) + c : kOOB;
    }
    // weight rows of the wave's two sub-tiles: gate and up of 32 features, or 64 columns
    const char* qptr = p.q + (int64_t)e * ebytes;
    const char* sptr = p.s + (int64_t)e * sbytes;
    uint32_t qoff[2], soff[2];
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const int f0 = GATE ? ct * 128 + wid * 32 : ct * BC + wid * 64 + c * 32;
      const uint32_t tile = (uint32_t)(((GATE && c ? p.N : 0) + f0) / 16 + (l32 >> 4)) * p.kt;
      qoff[c] = f0 < p.N ? tile * kPack4Q + hl * 256 + (l32 & 15) * 16 : kOOB;
      soff[c] = f0 < p.N ? tile * kPack4S + (l32 & 15) * 4 : kOOB;
    }
    auto issue_rows = [&](int s) {
      const uint32_t adv = (uint32_t)s * (BK * 2);
      const auto rs = make_rsrc(
          rptr + adv, __builtin_amdgcn_readfirstlane(s < nk && adv < rbytes ? rbytes - adv : 0u));
      char* slot = smem + (s & 3) * kSlot<BR>;
#pragma unroll
      for (int i = 0; i < RPW; ++i) dma16(rs, roff[i], slot + (wid + 4 * i) * 1024);
    };
    auto issue_weights = [&](int pr, Pair& w) {
      const bool in = pr < np;
      const uint32_t aq = (uint32_t)pr * kPack4Q, as = (uint32_t)pr * kPack4S;
      const auto rq = make_rsrc(qptr + aq, __builtin_amdgcn_readfirstlane(in ? ebytes - aq : 0u));
      const auto rs = make_rsrc(sptr + as, __builtin_amdgcn_readfirstlane(in ? sbytes - as : 0u));
#pragma unroll
      for (int c = 0; c < 2; ++c)
#pragma unroll
        for (int st = 0; st < 2; ++st)
          w.q[c][st] = __builtin_bit_cast(
              u32x4, __builtin_amdgcn_raw_buffer_load_b128(rq, qoff[c] + st * 512, 0, 0));
#pragma unroll
      for (int c = 0; c < 2; ++c)
        w.s[c] = __builtin_amdgcn_raw_buffer_load_b32(rs, soff[c], 0, 0);
    };

    f32x16 acc[2][TJ];
#pragma unroll
    for (int c = 0; c < 2; ++c)
#pragma unroll
      for (int r = 0; r < TJ; ++r)
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[c][r][i] = 0.f;

    Pair w[NB];
    issue_rows(0);
    __builtin_amdgcn_sched_barrier(0);
    issue_weights(0, w[0]);
    __builtin_amdgcn_sched_barrier(0);
    issue_rows(1);
    __builtin_amdgcn_sched_barrier(0);
    issue_rows(2);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int d = 1; d < D; ++d) {
      issue_weights(d, w[d]);
      __builtin_amdgcn_sched_barrier(0);
    }

    // One stage: its rows are waited for, those three stages on (and, in an even
    // stage, the weights D pairs on) asked for, then four steps of 16 columns.
    auto stage = [&](int s, int pr, const Pair& cur, Pair* next, auto st_t) {
      constexpr int st = decltype(st_t)::value;
      // issued after these rows: two stages of rows, and weights: D pairs' in the first
      // three stages, one pair's later (two in odd stages, of which one is in use)
      if (pr == 0 || (D > 1 && s < 3)) __builtin_amdgcn_s_waitcnt(wait_imm(2 * RPW + D * W));
      else __builtin_amdgcn_s_waitcnt(wait_imm(2 * RPW + W));
      __builtin_amdgcn_s_barrier();
      __builtin_amdgcn_sched_barrier(0);
      issue_rows(s + 3);
      __builtin_amdgcn_sched_barrier(0);
      if (next) issue_weights(pr + D, *next);
      __builtin_amdgcn_sched_barrier(0);
      const uint32_t base = (uint32_t)(s & 3) * kSlot<BR>;
      float sc[2];
#pragma unroll
      for (int c = 0; c < 2; ++c) sc[c] = unpack4_scale(cur.s[c] >> (16 * st + 8 * hl) & 0xffu);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        bf16x8 fa[2], fb[TJ];
#pragma unroll
        for (int r = 0; r < TJ; ++r)
          fb[r] = *(const __attribute__((address_space(3))) bf16x8*)lds_at(base + b_off[j] + r * 4096);
#pragma unroll
        for (int c = 0; c < 2; ++c)
          fa[c] = __builtin_bit_cast(bf16x8, unpack4_eight(cur.q[c][st][j], sc[c]));
#pragma unroll
        for (int r = 0; r < TJ; ++r)
#pragma unroll
          for (int c = 0; c < 2; ++c)
            acc[c][r] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(fa[c], fb[r], acc[c][r], 0, 0, 0);
      }
    };
    for (int p0 = 0; p0 < np; p0 += NB) {
#pragma unroll
      for (int u = 0; u < NB; ++u) {
        if (p0 + u >= np) break;
        stage(2 * (p0 + u), p0 + u, w[u], &w[(u + D) % NB], std::integral_constant<int, 0>{});
        stage(2 * (p0 + u) + 1, p0 + u, w[u], nullptr, std::integral_constant<int, 1>{});
      }
    }
    // what is still in flight are loads from empty descriptors, into the ring
    __builtin_amdgcn_s_waitcnt(wait_imm(0));
    __syncthreads();

    // ------------------------------------------------------------ epilogue
    // The tile to LDS in row order (16-byte chunks swizzled by row), then out in
    // whole lines.
    const int rows = min(row_end - row0, BR);
    if constexpr (GATE) {
#pragma unroll
      for (int r = 0; r < TJ; ++r)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          float v[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float g = acc[0][r][4 * q + i];
            v[i] = g * fast_sigmoid(g) * acc[1][r][4 * q + i];
          }
          const int row = r * 32 + l32, ch = wid * 4 + q;
          *(u32x2*)(smem + row * 256 + ((ch ^ (row & 15)) << 4) + hl * 8) =
              u32x2{pack_bf2(v[0], v[1]), pack_bf2(v[2], v[3])};
        }
      __syncthreads();
      for (int i = tid; i < rows * 16; i += 256) {
        const int row = i >> 4, ch = i & 15, col = ct * 128 + ch * 8;
        if (col < p.N)
          __builtin_nontemporal_store(*(const u32x4*)(smem + row * 256 + ((ch ^ (row & 15)) << 4)),
                                      (u32x4*)(p.act + (int64_t)(row0 + row) * p.N + col));
      }
    } else {
#pragma unroll
      for (int r = 0; r < TJ; ++r) {
        uint32_t m = 0;
#pragma unroll
        for (int c = 0; c < 2; ++c)
#pragma unroll
          for (int i = 0; i < 16; ++i) m = max(m, __float_as_uint(acc[c][r][i]) & 0x7fffffffu);
        m = max(m, (uint32_t)__shfl_xor((int)m, 32, 64));
        const uint32_t sb = block16_scale(m);
        const float inv = sb == 255u ? 0.f : __uint_as_float((254u - sb) << 23);
        const int row = r * 32 + l32;
#pragma unroll
        for (int c = 0; c < 2; ++c)
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            int v[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = (int)__builtin_rintf(acc[c][r][4 * q + i] * inv);
            const int ch = wid * 8 + c * 4 + q;
            *(u32x2*)(smem + row * 512 + ((ch ^ (row & 31)) << 4) + hl * 8) =
                u32x2{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pk_i16(v[0], v[1])),
                      __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pk_i16(v[2], v[3]))};
          }
        const int blk = ct * 4 + wid;
        if (hl == 0 && row < rows && blk * kBlock16 < p.N)
          p.ys[(int64_t)(row0 + row) * (p.N / kBlock16) + blk] = (uint8_t)sb;
      }
      __syncthreads();
      for (int i = tid; i < rows * 32; i += 256) {
        const int row = i >> 5, ch = i & 31, col = ct * BC + ch * 8;
        if (col < p.N)
          __builtin_nontemporal_store(*(const u32x4*)(smem + row * 512 + ((ch ^ (row & 31)) << 4)),
                                      (u32x4*)(p.y + (int64_t)(row0 + row) * p.N + col));
      }
    }
    __syncthreads();  // read out before the next tile's rows land
  }
}

// ---------------------------------------------------------------- combine
// A wave a token, eight columns a lane; up to eight rows of y in flight.
constexpr int kCombineWaves = 4;
__global__ __launch_bounds__(64 * kCombineWaves) void combine16_kernel(
    const int16_t* __restrict__ y, const uint8_t* __restrict__ ys, const int* __restrict__ slot,
    const int* __restrict__ offsets, const void* __restrict__ w, int wdt, int64_t T, int K, int E,
    int H, bf16* __restrict__ out) {
  const int lane = threadIdx.x & 63;
  const int nvalid = offsets[E];
  const int64_t nw = (int64_t)gridDim.x * kCombineWaves;
  for (int64_t t = (int64_t)blockIdx.x * kCombineWaves + (threadIdx.x >> 6); t < T; t += nw) {
    for (int h = ((int)blockIdx.y * 64 + lane) * 8; h < H; h += (int)gridDim.y * 512) {
      float o[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) o[i] = 0.f;
      for (int k0 = 0; k0 < K; k0 += 8) {
        u32x4 v[8];
        float f[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          f[k] = 0.f;
          v[k] = u32x4{0, 0, 0, 0};
          if (k0 + k >= K) continue;  // uniform
          const int64_t at = t * K + k0 + k;
          const int s = __builtin_amdgcn_readfirstlane(slot[at]);
          if (s >= nvalid) continue;  // a sentinel contributes nothing
          v[k] = __builtin_nontemporal_load((const u32x4*)(y + (int64_t)s * H + h));
          const uint32_t sb = ys[(int64_t)s * (H / kBlock16) + h / kBlock16];
          // 0 * inf, NaN, for a block that is not finite
          f[k] = __uint_as_float(sb << 23) *
                 (wdt == MOE_DTYPE_BF16 ? bf2f(((const bf16*)w)[at]) : ((const float*)w)[at]);
        }
#pragma unroll
        for (int k = 0; k < 8; ++k)
#pragma unroll
          for (int i = 0; i < 8; ++i)
            o[i] = fmaf((float)(int16_t)(v[k][i >> 1] >> (16 * (i & 1))), f[k], o[i]);
      }
      u32x4 r;
#pragma unroll
      for (int i = 0; i < 4; ++i) r[i] = pack_bf2(o[2 * i], o[2 * i + 1]);
      *(u32x4*)(out + t * H + h) = r;
    }
  }
}

// ------------------------------------------------------------------- host
std::atomic<int> g_num_cu[64];
int num_cus() {
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= 64) return 256;
  int n = g_num_cu[dev].load(std::memory_order_relaxed);
  if (!n) {
    if (hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess || n <= 0)
      n = 256;
    g_num_cu[dev].store(n, std::memory_order_relaxed);
  }
  return n;
}

int check4(int64_t S, int E, int H, int I, const char* who) {
  MOE_REQUIRE(S >= 0 && E >= 1 && H > 0 && I > 0, MOE_ERR_ARG, "%s: bad sizes", who);
  MOE_REQUIRE(H % 64 == 0 && I % 64 == 0, MOE_ERR_ARG, "%s: H=%d and I=%d must be multiples of 64",
              who, H, I);
  MOE_REQUIRE(S < ((int64_t)1 << 29), MOE_ERR_UNSUPPORTED, "%s: S=%lld routed rows, limit 2^29", who,
              (long long)S);
  // an expert's codes are read through a descriptor of 32 bits
  MOE_REQUIRE(pack4_tiles(2 * (int64_t)I, H) * kPack4Q < ((int64_t)1 << 31) &&
                  pack4_tiles(H, I) * kPack4Q < ((int64_t)1 << 31),
              MOE_ERR_UNSUPPORTED, "%s: H=%d, I=%d: an expert's weights exceed 2 GB", who, H, I);
  return MOE_OK;
}

template <int BR, bool GATE, int D>
int launch4(Gemm4Args& a, int64_t S, int E, const void* tile_plan, int b, hipStream_t st,
            const char* who) {
  const char* pb = (const char*)tile_plan;
  a.tile_count = (const int*)pb + (size_t)b * (E + 1) + E;
  a.tile_info = (const int4*)(pb + plan_info_offset(S, E, b));
  const int64_t most = plan_max_tiles(S, E, b) * a.n_ct;
  MOE_REQUIRE(most <= (int64_t)1 << 30, MOE_ERR_UNSUPPORTED, "%s: too many tiles", who);
  constexpr int lds = NSLOT * kSlot<BR>;
  static std::atomic<int> done[64];
  const hipError_t err = set_dynamic_lds_once(done, (const void*)gemm4_kernel<BR, GATE, D>, lds);
  MOE_REQUIRE(err == hipSuccess, MOE_ERR_HIP, "%s: HIP error %d (%s)", who, (int)err,
              hipGetErrorString(err));
  int64_t grid = (int64_t)num_cus() / 8 * 8 * (BR == 256 ? 1 : 2);
  if (grid > (most + 7) / 8 * 8) grid = (most + 7) / 8 * 8;
  if (grid < 8) grid = 8;
  gemm4_kernel<BR, GATE, D><<<(int)grid, 256, lds, st>>>(a);
  return check_launch(who);
}

template <bool GATE>
int launch4(Gemm4Args& a, int64_t S, int E, const void* tile_plan, hipStream_t st, const char* who) {
  const int64_t mean = S / E;
  if (mean >= 256) return launch4<256, GATE, 1>(a, S, E, tile_plan, 2, st, who);
  if (mean >= 96) return launch4<128, GATE, 2>(a, S, E, tile_plan, 1, st, who);
  return launch4<64, GATE, 3>(a, S, E, tile_plan, 0, st, who);
}

}  // namespace
}  // namespace moe

using namespace moe;

#define MOE_ALIGNED(ptr, who) \
  MOE_REQUIRE(al16(ptr), MOE_ERR_ALIGN, "%s: pointer %s not 16-byte aligned", who, #ptr)

extern "C" int moe_amd_gemm_gate_up_swiglu4(const void* hidden_states, const int32_t* row_src,
                                            int top_k, const int32_t* offsets,
                                            const void* tile_plan, const void* gate_up_q,
                                            const void* gate_up_scale, int64_t T, int64_t S, int E,
                                            int H, int I, void* act_out, void* stream) {
  const char* who = "gemm_gate_up_swiglu4";
  const int rc = check4(S, E, H, I, who);
  if (rc) return rc;
  MOE_REQUIRE(top_k >= 1 && S == T * top_k, MOE_ERR_ARG, "%s: S != T*top_k", who);
  MOE_REQUIRE(T * (int64_t)H * 2 < ((int64_t)1 << 31), MOE_ERR_UNSUPPORTED, "%s: T*H too large", who);
  MOE_REQUIRE(offsets && tile_plan && gate_up_q && gate_up_scale &&
                  (S == 0 || (hidden_states && row_src && act_out)),
              MOE_ERR_ARG, "%s: null pointer", who);
  MOE_ALIGNED(hidden_states, who);
  MOE_ALIGNED(gate_up_q, who);
  MOE_ALIGNED(gate_up_scale, who);
  MOE_ALIGNED(act_out, who);
  if (S == 0) return MOE_OK;
  Gemm4Args a{};
  a.x = (const bf16*)hidden_states;
  a.q = (const char*)gate_up_q;
  a.s = (const char*)gate_up_scale;
  a.row_src = row_src;
  a.act = (bf16*)act_out;
  a.T = T;
  a.K = H;
  a.N = I;
  a.kt = (H + kPack4Cols - 1) / kPack4Cols;
  a.nt = 2 * I / kPack4Rows;
  a.n_ct = (I + 127) / 128;
  // division by top_k as in gemm.hip: exact for 31 bits
  int sh = 0;
  while ((1 << sh) < top_k) ++sh;
  a.tok_shift = 31 + sh;
  a.tok_mul = (uint32_t)((((uint64_t)1 << (31 + sh)) + (uint64_t)top_k - 1) / (uint64_t)top_k);
  return launch4<true>(a, S, E, tile_plan, (hipStream_t)stream, who);
}

extern "C" int moe_amd_gemm_down4(const void* act, const int32_t* offsets, const void* tile_plan,
                                  const void* down_q, const void* down_scale, int64_t S, int E,
                                  int H, int I, void* y_out, void* y_scale_out, void* stream) {
  const char* who = "gemm_down4";
  const int rc = check4(S, E, H, I, who);
  if (rc) return rc;
  MOE_REQUIRE(offsets && tile_plan && down_q && down_scale &&
                  (S == 0 || (act && y_out && y_scale_out)),
              MOE_ERR_ARG, "%s: null pointer", who);
  MOE_ALIGNED(act, who);
  MOE_ALIGNED(down_q, who);
  MOE_ALIGNED(down_scale, who);
  MOE_ALIGNED(y_out, who);
  if (S == 0) return MOE_OK;
  Gemm4Args a{};
  a.x = (const bf16*)act;
  a.q = (const char*)down_q;
  a.s = (const char*)down_scale;
  a.y = (int16_t*)y_out;
  a.ys = (uint8_t*)y_scale_out;
  a.K = I;
  a.N = H;
  a.kt = (I + kPack4Cols - 1) / kPack4Cols;
  a.nt = H / kPack4Rows;
  a.n_ct = (H + BC - 1) / BC;
  return launch4<false>(a, S, E, tile_plan, (hipStream_t)stream, who);
}

extern "C" int moe_amd_combine16(const void* y, const void* y_scale, const int32_t* slot,
                                 const int32_t* offsets, const void* topk_weights,
                                 int weights_dtype, int64_t T, int K, int E, int H, void* out,
                                 void* stream) {
  const char* who = "combine16";
  MOE_REQUIRE(weights_dtype == MOE_DTYPE_F32 || weights_dtype == MOE_DTYPE_BF16, MOE_ERR_DTYPE,
              "%s: weights dtype %d", who, weights_dtype);
  MOE_REQUIRE(T >= 0 && K >= 1 && E >= 1 && H > 0 && H % 64 == 0, MOE_ERR_ARG,
              "%s: T=%lld K=%d E=%d H=%d", who, (long long)T, K, E, H);
  if (T == 0) return MOE_OK;
  MOE_REQUIRE(y && y_scale && slot && offsets && topk_weights && out, MOE_ERR_ARG,
              "%s: null pointer", who);
  MOE_ALIGNED(y, who);
  MOE_ALIGNED(out, who);
  // few tokens: a row's columns to several waves
  int64_t gx = (T + kCombineWaves - 1) / kCombineWaves;
  int gy = (H + 511) / 512;
  if (gx >= 2048) gy = 1;
  if (gx > 256 * 32) gx = 256 * 32;
  combine16_kernel<<<dim3((unsigned)gx, (unsigned)gy), 64 * kCombineWaves, 0, (hipStream_t)stream>>>(
      (const int16_t*)y, (const uint8_t*)y_scale, slot, offsets, topk_weights, weights_dtype, T, K, E,
      H, (bf16*)out);
  return check_launch(who);
}
