// Grouped products of the expert layer on a bank in 4 bits (gfx950), forward
// only, bf16 rows: the routed rows of each expert, as the permutation sorted
// them, times its packed weights (pack4.h).
//
//   gemm4_kernel<.., GATE = true>   act [S,I] = silu(x Wg^T) * (x Wu^T), x gathered by token
//   gemm4_kernel<.., GATE = false>  y [S,H] = act W2^T, fp16 in blocks of 64 columns
//   combine16_kernel                out [T,H] = sum_k w[t,k] y[row of (t,k)]
//
// A workgroup of NW waves owns BR rows by 64 NW weight rows (gate and up: 32 NW
// features of each), a wave all its rows by 64 weight rows of its own.  So no weight
// is wanted by two waves: each goes from memory to its lane's registers, 16 bytes of
// codes a load and whole lines a wave, and becomes an MFMA operand there by four
// conversions for eight values; converted or not, weights never pass
// through LDS, which holds rows only.  MFMA v_mfma_f32_32x32x16_bf16: weights as
// A (a lane's accumulators hold four consecutive columns of one row), rows as B.
// The contraction runs in the order of the tiles' blocks: lane half h of step j
// takes columns 32 h + 8 j of a stage's 64, of both operands alike.
//
// Rows come by LDS DMA, 64 columns a stage (128-byte lines, 16-byte chunks
// XOR-swizzled by row: no bank conflicts), into a ring of four slots; weights into
// registers, four stages ahead too.  The stages of a workgroup's tiles are one
// stream: a tile's last stages ask for the next tile's first ones, which arrive
// under its epilogue.  Loads past the end of the contraction are issued all the same,
// from empty descriptors (zeros, no memory access), so that the wait counts hold in
// every stage.
//
// act is rounded to bf16 once.  y is held in fp16 with a power of two for 64 columns of
// a row, which puts the largest finite one at 2^14 or above: as small as bf16, but within
// 2^-11 of each value instead of 2^-8 (three roundings of bf16 size in a row would
// show: 1.7 times the error of one) down to 2^-28 of the largest, and within 2^-39 of the
// largest below that.  (As whole numbers of the power of two, within 2^-15 of the
// largest, a column 2^12 times its neighbours leaves those 5e-2 off.)  Each output is
// rounded once.
//
// Measured (gate/up, down, combine; H 2048, I 768, top 8 of 128 experts; medians, ranges
// are boxes):
//   16384 tokens  646 to 676 us (1.28 to 1.22 PF), 349 to 369 us (1.18 to 1.12 PF), 99 us
//                 (6.1 TB/s); a plain bf16 product reaches 1.4 to 1.6 PF on this card.  The
//                 matrix units are busy 70 and 60% of the cycles, at the 1.8 GHz that the
//                 power leaves: the epilogues are 8% and 19% of the time; the rest are the
//                 conversions' issue slots and each expert's last, partial tile
//    1021 tokens  58 to 72 us, 37 to 45 us, 8 us: 320 MB of weights and 64 rows an expert, so
//                 that both bounds are near (3.6 TB/s, 0.85 PF)
// and 2048 tokens on 1792 experts (9 rows each): 475 to 492 us, 292 to 302 us, 14 us, bound by
// the 4.5 GB of weights (6.2 and 5.0 TB/s).
//
// Reference: transformers/integrations/moe.py:377-478.
#include "common.h"
#include "pack4.h"

namespace moe {
namespace {

constexpr int BK = 64;     // columns of the contraction a stage
constexpr int NSLOT = 4;   // stages of rows in LDS
constexpr int kBlock16 = 64;  // columns of a block of y
constexpr int kMostColumns = 1 << 22;

template <int BR> constexpr int kSlot = BR * BK * 2;  // bytes
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

struct Gemm4Args {
  const bf16* x;         // hidden states [T,H] (gate/up) or act [S,I]
  const char *q, *s;     // codes and scales of the bank
  const int* row_src;    // [S] flat entry of a sorted row
  const int* tile_count; // row tiles
  const int4* tile_info; // {expert, first row, end row, 0} of each
  bf16* act;             // [S,I]
  _Float16* y;           // [S,H] and its scale bytes [S,H/64]
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
// act and y are written through the L2 (cache bits sc0 and sc1): their lines are not
// evicted among the weights' later, and the next launch finds more of them in the
// memory-side cache (combine of 16384 tokens 108 -> 99.5 us, 2048 tokens on 1792 experts
// 808 -> 798 us in all, against non-temporal stores; plain ones 101 and 804).
constexpr int kThrough = 17;
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

// The biased exponent of a block's power of two from its largest finite |v|, which is
// from 2^14 to 2^15 of it, and of fp16's range once rounded.
__device__ __forceinline__ uint32_t block16_scale(float most) {
  const int e = (int)(__float_as_uint(most) >> 23) - 14;
  return (uint32_t)(e < 1 ? 1 : e);
}

// f(integral_constant<int, nj>, g): a main loop for each number of row sub-tiles.
template <int TJ, typename F, typename G>
__device__ __forceinline__ void with_sub_tiles(int nj, F&& f, G&& g) {
  if constexpr (TJ > 1) {
    if (nj < TJ) return with_sub_tiles<TJ - 1>(nj, f, g);
  }
  f(std::integral_constant<int, TJ>{}, g);
}

// Waves a SIMD: 64 rows leave the registers and the LDS for three.
template <int BR> constexpr int kWavesSimd = BR <= 64 ? 3 : 2;

// NW waves, each with 64 weight rows of its own; STREAM: weights by non-temporal loads.
template <int BR, bool GATE, int NW, bool STREAM>
__global__ __launch_bounds__(64 * NW, kWavesSimd<BR>) void gemm4_kernel(Gemm4Args p) {
  constexpr int TJ = BR / 32;              // row sub-tiles, all of them every wave's
  constexpr int RPW = BR / 8 / NW;         // 1 KB DMA blocks of a stage's rows per wave
  constexpr int BC = 64 * NW;              // weight rows of a tile
  constexpr int OUT = GATE ? BC / 2 : BC;  // output columns of a tile
  static_assert(RPW >= 1, "DMA blocks per wave");
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wid = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int l32 = lane & 31, hl = lane >> 5;

  // The tiles are cut into eight ranges, one an XCD, so that the tiles that run at
  // a time share rows and weights in its L2.
  const int n_tiles = *p.tile_count * p.n_ct;
  const int xcd = blockIdx.x & 7, stride = gridDim.x >> 3, chunk = (n_tiles + 7) >> 3;
  const int t_end = min(n_tiles, (xcd + 1) * chunk);
  int t = xcd * chunk + (int)(blockIdx.x >> 3);
  if (t >= t_end) return;
  const int nk = (p.K + BK - 1) / BK;
  const uint32_t ebytes = (uint32_t)p.nt * p.kt * kPack4Q, sbytes = (uint32_t)p.nt * p.kt * kPack4S;

  const uint32_t lds0 = (uint32_t)(uintptr_t)(const lds_char_t*)smem;
  auto lds_at = [](uint32_t a) { return (lds_char_t*)(uintptr_t)a; };
  uint32_t b_off[4];  // of step j: row l32, chunk 4 hl + j
#pragma unroll
  for (int j = 0; j < 4; ++j)
    b_off[j] = lds0 + l32 * 128 + (((4 * hl + j) ^ ((l32 >> 1) & 7)) << 4);

  // ------------------------------------------------------------- operands
  struct Tile {
    int e, row0, row_end, ct;
  };
  auto tile_at = [&](int tt, const int4& ti) {
    return Tile{ti.x, ti.y, ti.z, tt % p.n_ct};
  };
  // What is computed once a tile is computed from the lane and the wave as the
  // optimizer does not know them: else it moves the addresses out of the tile loop,
  // or to the tile's beginning, and spills them (a reload waits for every load
  // before it).
  auto rows_load = [&](const int4& ti, int (&src)[RPW]) {  // their flat entries
    if constexpr (GATE) {
      int ln = lane, wd = wid;
      asm volatile("" : "+v"(ln), "+s"(wd));
#pragma unroll
      for (int i = 0; i < RPW; ++i)
        src[i] = p.row_src[min(ti.y + (wd + NW * i) * 8 + (ln >> 3), ti.z - 1)];
    }
  };
  const char *rptr = nullptr, *qptr = nullptr, *sptr = nullptr;
  uint32_t rbytes = 0, roff[RPW], qoff[2], soff[2];
  auto setup = [&](const Tile& d, int (&src)[RPW]) {
    int ln = lane, wd = wid, shift = p.tok_shift;
    uint32_t mul = p.tok_mul;
    asm volatile("" : "+v"(ln), "+s"(wd), "+s"(mul), "+s"(shift));
    if constexpr (GATE) {
#pragma unroll
      for (int i = 0; i < RPW; ++i) asm volatile("" : "+v"(src[i]));
    }
    rptr = (const char*)(GATE ? p.x : p.x + (int64_t)d.row0 * p.K);
    rbytes = GATE ? (uint32_t)(p.T * p.K * 2)
                  : (uint32_t)((int64_t)min(d.row_end - d.row0, BR) * p.K * 2);
#pragma unroll
    for (int i = 0; i < RPW; ++i) {
      const int f = (wd + NW * i) * 8 + (ln >> 3);
      const uint32_t c = ((ln & 7) ^ ((f >> 1) & 7)) * 16;
      int r = f;
      if constexpr (GATE) r = (int)(((uint64_t)(uint32_t)src[i] * mul) >> shift);
      roff[i] = d.row0 + f < d.row_end ? (uint32_t)r * (uint32_t)(p.K * 2) + c : kOOB;
    }
    // weight rows of the wave's two sub-tiles: gate and up of 32 features, or 64 columns
    qptr = p.q + (int64_t)d.e * ebytes;
    sptr = p.s + (int64_t)d.e * sbytes;
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const int f0 = d.ct * OUT + (GATE ? wd * 32 : wd * 64 + c * 32);
      const uint32_t tile = (uint32_t)(((GATE && c ? p.N : 0) + f0) / 16 + (ln >> 4 & 1)) * p.kt;
      qoff[c] = f0 < p.N ? tile * kPack4Q + (ln >> 5) * 256 + (ln & 15) * 16 : kOOB;
      soff[c] = f0 < p.N ? tile * kPack4S + (ln & 15) * 4 : kOOB;
    }
  };
  auto issue_rows = [&](int s) {
    const uint32_t adv = (uint32_t)s * (BK * 2);
    const auto rs = make_rsrc(
        rptr + adv, __builtin_amdgcn_readfirstlane(s < nk && adv < rbytes ? rbytes - adv : 0u));
    char* slot = smem + (s & 3) * kSlot<BR>;
#pragma unroll
    for (int i = 0; i < RPW; ++i) dma16(rs, roff[i], slot + (wid + NW * i) * 1024);
  };
  // The weights of four stages, the scales of their pairs.
  u32x4 wq[4][2];
  uint32_t ws[2][2];
  auto issue_codes = [&](int s, u32x4 (&w)[2]) {  // stage s: half a tile
    const uint32_t adv = (uint32_t)(s >> 1) * kPack4Q + (uint32_t)(s & 1) * 512;
    const auto rs = make_rsrc(qptr + adv, __builtin_amdgcn_readfirstlane(s < nk ? ebytes - adv : 0u));
#pragma unroll
    for (int c = 0; c < 2; ++c)
      w[c] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(rs, qoff[c], 0,
                                                                          STREAM ? 2 : 0));
  };
  auto issue_scales = [&](int pr, uint32_t (&w)[2]) {
    const uint32_t adv = (uint32_t)pr * kPack4S;
    const auto rs =
        make_rsrc(sptr + adv, __builtin_amdgcn_readfirstlane(pr < p.kt ? sbytes - adv : 0u));
#pragma unroll
    for (int c = 0; c < 2; ++c) w[c] = __builtin_amdgcn_raw_buffer_load_b32(rs, soff[c], 0, 0);
  };

  // ------------------------------------------------------------- main loop
  // Stages run in groups of four, the last one filled up to two or four with empty stages
  // (to four for gate and up of few rows, whose registers do not hold the branch: 22.0 us
  // become 24.4 for 509 tokens of 1024 columns; elsewhere 320 and 576 columns gain 5 to 10%).
  // A stage's rows, codes and (with odd ones) scales are asked for four stages ahead, in the last
  // group those of the next tile's first: so a tile begins with its loads under way.
  const int groups = (nk + 3) / 4;
  const bool half = (BR > 64 || !GATE) && nk - 4 * (groups - 1) <= 2;  // the last group
  f32x16 acc[2][TJ];
  auto fragment = [&](int s, int j, int r) {
    return *(const __attribute__((address_space(3))) bf16x8*)lds_at(
        (uint32_t)(s & 3) * kSlot<BR> + b_off[j] + r * 4096);
  };
  auto weights = [&](int u, int c, int j) {  // stage u of a group
    const uint32_t sc = ws[u / 2][c] >> (16 * (u & 1) + 8 * hl) & 0xffu;
    return __builtin_bit_cast(bf16x8, unpack4_eight(wq[u][c][j], unpack4_scale(sc)));
  };
  auto mma = [](const bf16x8& w, const bf16x8& x, const f32x16& c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(w, x, c, 0, 0, 0);
  };
  // Until the next stage's rows are there, and every wave has read all of this one's.
  // Asked for after them were two stages' rows, four loads of codes and two of scales
  // at least; in a tile's first stages, the previous one's stores too (`stored`
  // sub-tiles, kStores each), which may still be on their way (loads and stores
  // complete in order).
  constexpr int kStores = GATE ? 2 : 4, kAfter = 2 * RPW + 6;
  static_assert(kAfter + 4 * kStores <= 63 && TJ <= 4, "vmcnt");
  int stored = 0;
  auto wait_rows = [&](bool first_stages) {
    const int n = first_stages ? stored : 0;
    if (n == 0) __builtin_amdgcn_s_waitcnt(wait_imm(kAfter));
    else if (n == 1) __builtin_amdgcn_s_waitcnt(wait_imm(kAfter + kStores));
    else if (n == 2) __builtin_amdgcn_s_waitcnt(wait_imm(kAfter + 2 * kStores));
    else if (n == 3) __builtin_amdgcn_s_waitcnt(wait_imm(kAfter + 3 * kStores));
    else __builtin_amdgcn_s_waitcnt(wait_imm(kAfter + 4 * kStores));
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_sched_barrier(0);
  };
  // The second half of a group that has only one: the next tile's stages in its place, and
  // what the last one would have waited for, the next tile's first rows.
  auto leave_out = [&]() {
#pragma unroll
    for (int u = 2; u < 4; ++u) {
      if (u == 3) wait_rows(false);
      issue_rows(u);
      issue_codes(u, wq[u]);
      if (u & 1) issue_scales(u >> 1, ws[u / 2]);
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  // Many rows (bound by the matrix units): a stage's four steps, each reading and
  // converting the next one's fragments while it multiplies; before the last step the
  // next stage's rows are waited for, and behind that barrier stage `at`, the one four
  // on, is asked for in this one's place.
  auto many_rows = [&](auto nj_t, auto&& next_tile) {
    constexpr int NJ = decltype(nj_t)::value;
    bf16x8 fa[2][2], fb[2][NJ];
    auto read = [&](int buf, int u, int j) {
#pragma unroll
      for (int r = 0; r < NJ; ++r) fb[buf][r] = fragment(u, j, r);
#pragma unroll
      for (int c = 0; c < 2; ++c) fa[buf][c] = weights(u, c, j);
    };
    auto multiply = [&](int buf) {
#pragma unroll
      for (int r = 0; r < NJ; ++r)
#pragma unroll
        for (int c = 0; c < 2; ++c) acc[c][r] = mma(fa[buf][c], fb[buf][r], acc[c][r]);
    };
    // order within a step: loads, fragment reads and conversions between the MFMAs
    auto order = [&](auto loads_t) {
      constexpr int LOADS = decltype(loads_t)::value;
#pragma unroll
      for (int r = 0; r < NJ; ++r) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);  // MFMA
        if (LOADS) __builtin_amdgcn_sched_group_barrier(0x020, (LOADS + NJ - 1) / NJ, 0);  // VMEM
        __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);  // DS read
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x002, (16 + NJ - 1) / NJ, 0);  // VALU
      }
    };
    read(0, 0, 0);
    int group = 0;
    do {
      int at = 4 * group + 4;
      bool leave = false;
      if (group == groups - 1) {
        next_tile();
        at = 0;
        leave = half;
      }
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        if (u == 2 && leave) {
          leave_out();
          break;
        }
#pragma unroll
        for (int j = 0; j < 3; ++j) {
          read((j + 1) & 1, u, j + 1);
          multiply(j & 1);
          order(std::integral_constant<int, 0>{});
          __builtin_amdgcn_sched_barrier(0);
        }
        wait_rows(u < 3 && group == 0);
        issue_rows(at + u);
        issue_codes(at + u, wq[u]);
        if (u & 1) issue_scales((at + u) >> 1, ws[u / 2]);
        if (u < 3) read(0, u + 1, 0);
        else read(0, 0, 0);
        multiply(1);
        order(std::integral_constant<int, RPW + 4>{});
        __builtin_amdgcn_sched_barrier(0);
      }
    } while (++group < groups);
  };
  // Few rows (bound by the weights): a stage's fragments are all read a stage ahead, so
  // that a stage waits once.
  auto few_rows = [&](auto nj_t, auto&& next_tile) {
    constexpr int NJ = decltype(nj_t)::value;
    bf16x8 fb[2][4][NJ];
    auto read = [&](int buf, int u) {
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int r = 0; r < NJ; ++r) fb[buf][j][r] = fragment(u, j, r);
    };
    read(0, 0);
    int group = 0;
    do {
      int at = 4 * group + 4;
      bool leave = false;
      if (group == groups - 1) {
        next_tile();
        at = 0;
        leave = half;
      }
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        if (u == 2 && leave) {
          leave_out();
          break;
        }
        wait_rows(u < 3 && group == 0);
        issue_rows(at + u);
        __builtin_amdgcn_sched_barrier(0);
        read((u + 1) & 1, (u + 1) & 3);
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            const bf16x8 w = weights(u, c, j);
#pragma unroll
            for (int r = 0; r < NJ; ++r) acc[c][r] = mma(w, fb[u & 1][j][r], acc[c][r]);
          }
        __builtin_amdgcn_sched_barrier(0);
        issue_codes(at + u, wq[u]);
        if (u & 1) issue_scales((at + u) >> 1, ws[u / 2]);
        __builtin_amdgcn_sched_barrier(0);
      }
    } while (++group < groups);
  };

  // -------------------------------------------------------------- epilogue
  // Row sub-tiles through LDS to memory in row order, whole lines, while the next
  // tile's first stages are on their way.
  const uint32_t stage = lds0 + NSLOT * kSlot<BR>;
  typedef __attribute__((address_space(3))) u32x2 lds_u32x2_t;
  typedef __attribute__((address_space(3))) u32x4 lds_u32x4_t;
  auto lds_barrier = [&]() {  // (loads stay in flight)
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
  };
  auto turn = [&]() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront", "local");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront", "local");
  };
  auto epilogue = [&](const Tile& d, int nj) {
    int ln = lane, wd = wid;
    asm volatile("" : "+v"(ln), "+s"(wd));
    const int el32 = ln & 31, ehl = ln >> 5;
    const uint32_t rows = (uint32_t)min(d.row_end - d.row0, BR);
    if constexpr (GATE) {
      // a wave has 64 bytes of a row: the workgroup's waves write a sub-tile together,
      // in two halves of the staging by turns (and between two tiles lie the main
      // loop's barriers)
      constexpr int LINE = OUT * 2;            // bytes of a row
      constexpr int PER = 1024 / LINE;         // rows a store of a wave
      static_assert(kStores * NW * PER == 32, "a sub-tile's rows");
      const auto rs = make_rsrc(p.act + (int64_t)d.row0 * p.N, rows * (uint32_t)p.N * 2);
#pragma unroll
      for (int r = 0; r < TJ; ++r) {
        if (r >= nj) break;
        const uint32_t buf = stage + (r & 1) * (32 * LINE);
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          float v[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float g = acc[0][r][4 * q + i];
            v[i] = g * fast_sigmoid(g) * acc[1][r][4 * q + i];
          }
          *(lds_u32x2_t*)lds_at(buf + el32 * LINE + (((wd * 4 + q) ^ (el32 & 15)) << 4) + ehl * 8) =
              u32x2{pack_bf2(v[0], v[1]), pack_bf2(v[2], v[3])};
        }
        lds_barrier();
#pragma unroll
        for (int h = 0; h < kStores; ++h) {
          const int row = (h * NW + wd) * PER + ln / (LINE / 16), ch = ln % (LINE / 16);
          const int col = d.ct * OUT + ch * 8;
          const u32x4 v = *(const lds_u32x4_t*)lds_at(buf + row * LINE + ((ch ^ (row & 15)) << 4));
          __builtin_amdgcn_raw_buffer_store_b128(
              v, rs, col < p.N ? (uint32_t)(r * 32 + row) * (uint32_t)p.N * 2 + (uint32_t)col * 2 : kOOB,
              0, kThrough);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
    } else {
      const int f0 = d.ct * OUT + wd * 64;
      const auto rs = make_rsrc(p.y + (int64_t)d.row0 * p.N, rows * (uint32_t)p.N * 2);
      const uint32_t mine = stage + wd * 4096, scales = stage + NW * 4096;
      if (f0 < p.N) {
#pragma unroll
        for (int r = 0; r < TJ; ++r) {
          if (r >= nj) break;
          const auto row_most = [](float m) {  // of both lanes of a row
            const auto both = __builtin_amdgcn_permlane32_swap(__float_as_uint(m), __float_as_uint(m),
                                                               false, false);
            return __builtin_elementwise_maximum(__uint_as_float(both[0]), __uint_as_float(both[1]));
          };
          float m = 0.f;  // (maximum: NaN if any is)
#pragma unroll
          for (int c = 0; c < 2; ++c)
#pragma unroll
            for (int i = 0; i < 16; ++i)
              m = __builtin_elementwise_maximum(m, __builtin_fabsf(acc[c][r][i]));
          m = row_most(m);
          if (__builtin_amdgcn_ballot_w64(!(m < INFINITY))) {  // of those that are finite
            m = 0.f;
#pragma unroll
            for (int c = 0; c < 2; ++c)
#pragma unroll
              for (int i = 0; i < 16; ++i) {
                const float a = __builtin_fabsf(acc[c][r][i]);
                m = a < INFINITY && a > m ? a : m;
              }
            m = row_most(m);
          }
          const uint32_t sb = block16_scale(m);
          const float inv = __uint_as_float((254u - sb) << 23);
#pragma unroll
          for (int c = 0; c < 2; ++c)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
              const auto two = [&](int i) {
                const f16x2 v = {(_Float16)(acc[c][r][4 * q + i] * inv),
                                 (_Float16)(acc[c][r][4 * q + i + 1] * inv)};
                return __builtin_bit_cast(uint32_t, v);
              };
              *(lds_u32x2_t*)lds_at(mine + el32 * 128 + (((c * 4 + q) ^ (el32 & 7)) << 4) + ehl * 8) =
                  u32x2{two(0), two(2)};
            }
          if (ehl == 0)
            *(__attribute__((address_space(3))) uint8_t*)lds_at(scales + (r * 32 + el32) * NW + wd) =
                (uint8_t)sb;
          turn();
#pragma unroll
          for (int h = 0; h < 4; ++h) {
            const int row = h * 8 + (ln >> 3), ch = ln & 7;
            const u32x4 v = *(const lds_u32x4_t*)lds_at(mine + row * 128 + ((ch ^ (row & 7)) << 4));
            __builtin_amdgcn_raw_buffer_store_b128(
                v, rs, (uint32_t)(r * 32 + row) * (uint32_t)p.N * 2 + (uint32_t)(f0 + ch * 8) * 2, 0,
                kThrough);
          }
          turn();
          __builtin_amdgcn_sched_barrier(0);
        }
      }
      // a row's scale bytes together: one at a time they would be as many writes of memory
      lds_barrier();
      const int blocks = p.N / kBlock16, have = min(NW, blocks - d.ct * NW);
      for (uint32_t row = wd * 64 + ln; row < rows; row += 64 * NW) {
        uint8_t* at = p.ys + (int64_t)(d.row0 + row) * blocks + d.ct * NW;
        const lds_char_t* from = lds_at(scales + row * NW);
        if (have == NW && ((uintptr_t)at & 3) == 0) {
#pragma unroll
          for (int i = 0; i < NW / 4; ++i)
            ((uint32_t*)at)[i] = ((const __attribute__((address_space(3))) uint32_t*)from)[i];
        } else {
          for (int i = 0; i < have; ++i) at[i] = (uint8_t)from[i];
        }
      }
    }
  };

  // ------------------------------------------------------------- the tiles
  // (a table that no kernel writes meanwhile, read to scalar registers)
  typedef const __attribute__((address_space(4))) int const_int_t;
  const auto* infos = (const_int_t*)(uintptr_t)p.tile_info;
  auto info_at = [&](int tt) {
    const int64_t i = 4 * (int64_t)(min(tt, t_end - 1) / p.n_ct);
    return make_int4(infos[i], infos[i + 1], infos[i + 2], 0);
  };
  int4 ti = info_at(t), ti_next = info_at(t + stride);
  int src[RPW] = {};
  rows_load(ti, src);
  Tile d = tile_at(t, ti);
  setup(d, src);
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    issue_rows(u);
    issue_codes(u, wq[u]);
    if (u & 1) issue_scales(u >> 1, ws[u / 2]);
    __builtin_amdgcn_sched_barrier(0);
  }
  __builtin_amdgcn_s_waitcnt(wait_imm(3 * RPW));
  __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_sched_barrier(0);
  while (true) {
    const Tile done = d;
    const int nj = (min(d.row_end - d.row0, BR) + 31) / 32;
    t += stride;
    const bool more = t < t_end;
    ti = ti_next;
    ti_next = info_at(t + stride);
    rows_load(ti, src);  // (both land under the main loop)
#pragma unroll
    for (int c = 0; c < 2; ++c)
#pragma unroll
      for (int r = 0; r < TJ; ++r)
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[c][r][i] = 0.f;
    auto next_tile = [&]() {
      if (more) {
        d = tile_at(t, ti);
        setup(d, src);
      } else {  // loads as many as ever, of nothing
        rbytes = 0;
        qoff[0] = qoff[1] = soff[0] = soff[1] = kOOB;
      }
    };
    if constexpr (BR <= 64) with_sub_tiles<TJ>(nj, few_rows, next_tile);
    else with_sub_tiles<TJ>(nj, many_rows, next_tile);
    epilogue(done, nj);
    if (!more) return;
    // (a wave past the last column stores nothing)
    stored = GATE || done.ct * OUT + wid * 64 < p.N ? nj : 0;
  }
}

// ---------------------------------------------------------------- combine
// A wave a token, eight columns a lane, two pieces of 512 columns of up to eight rows
// of y in flight; the next token's rows and weights are read meanwhile.
constexpr int kCombineWaves = 4;
constexpr int kPieces = 2;
__global__ __launch_bounds__(64 * kCombineWaves, 4) void combine16_kernel(
    const _Float16* __restrict__ y, const uint8_t* __restrict__ ys, const int* __restrict__ slot,
    const int* __restrict__ offsets, const void* __restrict__ w, int wdt, int64_t T, int K, int E,
    int H, bf16* __restrict__ out) {
  const int lane = threadIdx.x & 63;
  const int nvalid = offsets[E], blocks = H / kBlock16;
  const int64_t nw = (int64_t)gridDim.x * kCombineWaves;
  const auto entry_load = [&](int64_t t, int kb, int& row, float& wk) {  // entries kb + lane
    const int64_t at = t * K + kb + lane;
    const bool in = t < T && kb + lane < K;
    row = in ? slot[at] : 0x7fffffff;
    wk = !in ? 0.f : wdt == MOE_DTYPE_BF16 ? bf2f(((const bf16*)w)[at]) : ((const float*)w)[at];
  };
  int64_t t = (int64_t)blockIdx.x * kCombineWaves + (threadIdx.x >> 6);
  int row, row_next;
  float wk, wk_next;
  entry_load(t, 0, row, wk);
  for (; t < T; t += nw) {
    entry_load(t + nw, 0, row_next, wk_next);
    for (int h0 = (int)blockIdx.y * 512 * kPieces; h0 < H; h0 += (int)gridDim.y * 512 * kPieces) {
      float o[kPieces][8] = {};
      for (int kb = 0; kb < K; kb += 64) {
        if (K > 64) entry_load(t, kb, row, wk);
        for (int k0 = 0; k0 < min(K - kb, 64); k0 += 8) {
          u32x4 v[kPieces][8];
          uint32_t sb[kPieces][8];
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            const int s = __builtin_amdgcn_readlane(row, k0 + k);
            if (s >= nvalid) continue;  // a sentinel, or none
#pragma unroll
            for (int c = 0; c < kPieces; ++c) {
              const int h = h0 + c * 512 + lane * 8;
              if (h < H) {
                v[c][k] = __builtin_nontemporal_load((const u32x4*)(y + (int64_t)s * H + h));
                sb[c][k] = ys[(int64_t)s * blocks + h / kBlock16];
              }
            }
          }
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            if (__builtin_amdgcn_readlane(row, k0 + k) >= nvalid) continue;
            const float f = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(wk), k0 + k));
#pragma unroll
            for (int c = 0; c < kPieces; ++c) {
              const float s = __uint_as_float(sb[c][k] << 23) * f;
              const f16x8 h = __builtin_bit_cast(f16x8, v[c][k]);
#pragma unroll
              for (int i = 0; i < 8; ++i) o[c][i] = fmaf((float)h[i], s, o[c][i]);
            }
          }
        }
      }
#pragma unroll
      for (int c = 0; c < kPieces; ++c) {
        const int h = h0 + c * 512 + lane * 8;
        if (h >= H) continue;
        u32x4 r;
#pragma unroll
        for (int i = 0; i < 4; ++i) r[i] = pack_bf2(o[c][2 * i], o[c][2 * i + 1]);
        __builtin_nontemporal_store(r, (u32x4*)(out + t * H + h));
      }
    }
    row = row_next;
    wk = wk_next;
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
  // a tile's rows and an expert's codes are read through descriptors of 32 bits
  MOE_REQUIRE(H <= kMostColumns && I <= kMostColumns, MOE_ERR_UNSUPPORTED,
              "%s: H=%d or I=%d above 2^22", who, H, I);
  MOE_REQUIRE(pack4_tiles(2 * (int64_t)I, H) * kPack4Q < ((int64_t)1 << 31) &&
                  pack4_tiles(H, I) * kPack4Q < ((int64_t)1 << 31),
              MOE_ERR_UNSUPPORTED, "%s: H=%d, I=%d: an expert's weights exceed 2 GB", who, H, I);
  return MOE_OK;
}

template <int BR, bool GATE, int NW, bool STREAM>
int launch4(Gemm4Args& a, int64_t S, int E, const void* tile_plan, int b, hipStream_t st,
            const char* who) {
  static_assert(kTileSizes[0] == 64 && kTileSizes[1] == 128, "the plan's row tiles");
  const char* pb = (const char*)tile_plan;
  a.tile_count = (const int*)pb + (size_t)b * (E + 1) + E;
  a.tile_info = (const int4*)(pb + plan_info_offset(S, E, b));
  constexpr int OUT = GATE ? 32 * NW : 64 * NW;
  a.n_ct = (a.N + OUT - 1) / OUT;
  const int64_t most = plan_max_tiles(S, E, b) * a.n_ct;
  MOE_REQUIRE(most <= (int64_t)1 << 30, MOE_ERR_UNSUPPORTED, "%s: too many tiles", who);
  // the ring of rows, and two halves of 32 rows or a part for each wave and the scales
  constexpr int lds = NSLOT * kSlot<BR> + (GATE ? 2 * 32 * OUT * 2 : NW * 4096 + BR * NW);
  static std::atomic<int> done[64];
  const hipError_t err = set_dynamic_lds_once(done, (const void*)gemm4_kernel<BR, GATE, NW, STREAM>, lds);
  MOE_REQUIRE(err == hipSuccess, MOE_ERR_HIP, "%s: HIP error %d (%s)", who, (int)err,
              hipGetErrorString(err));
  int64_t grid = (int64_t)num_cus() / 8 * 8 * (kWavesSimd<BR> * 4 / NW);
  if (grid > (most + 7) / 8 * 8) grid = (most + 7) / 8 * 8;
  if (grid < 8) grid = 8;
  gemm4_kernel<BR, GATE, NW, STREAM><<<(int)grid, 64 * NW, lds, st>>>(a);
  return check_launch(who);
}

// Row tiles by the mean rows of an expert (us at 2048 columns, I 768, top 8, three banks by
// turns; few: 64 rows, four waves; many: 128 rows, four waves for gate and up, eight, which
// read a row half as often, for down: its contraction is short):
//   mean rows, experts  8, 128  32, 128  40, 128  48, 128  64, 128  128, 128  512, 128  1024, 128  9, 1792
//   gate/up  few            40       49       54       62       79       121       385        716     524
//            many           42       49       56       61       68       125       370        684     567
//   down     few            23       28       32       35       41        68       221        419     314
//            many           25       30       34       37       43        71       210        373     306
// and many down's columns want to be a whole number of 512: where 256 do as well and the
// rest is more than a ninth, few (3000 tokens on 32 experts, top 6, I 320, 576 columns:
// 24.0 and 14.6; 8192 on 64, top 4, I 512, 1280 columns: 64.8 and 54.2).
// Few rows take half the registers, so that three workgroups share a CU where two do
// of many, which read the weights half as often.
// Few rows stream the codes of a bank that the memory-side cache cannot hold: 2048
// tokens on 1792 experts 524 and 314 us become 487 and 302, while with 300 on 128 the
// same bank's next call takes 45 and 26 us where it finds a part of it there in 41 and 23.
// The host knows the mean over all experts, not the counts: where all 2048 tokens go to
// 8, 16, 64 or 256 of the 1792 experts, gate/up and down take 99 + 57, 103 + 63, 113 + 68 and
// 151 + 85 us, the best of the three forms 84 + 50, 98 + 55, 107 + 63 and 138 + 81.
constexpr int64_t kMemoryCache = 256ll << 20;
template <bool GATE>
int launch4(Gemm4Args& a, int64_t S, int E, const void* tile_plan, hipStream_t st, const char* who) {
  const int quarters = (a.N + 255) / 256;
  if (S / E >= 40 && (GATE || quarters % 2 == 0 || quarters >= 9))
    return launch4<128, GATE, GATE ? 4 : 8, false>(a, S, E, tile_plan, 1, st, who);
  if (S / E < 40 && (int64_t)E * a.nt * a.kt * kPack4Q > kMemoryCache)
    return launch4<64, GATE, 4, true>(a, S, E, tile_plan, 0, st, who);
  return launch4<64, GATE, 4, false>(a, S, E, tile_plan, 0, st, who);
}

// moe_amd_experts4's workspace: each array 256-byte aligned.
struct Layout4 {
  size_t counts, offsets, row_src, slot, plan, sort, act, y, ys, bytes;
  size_t plan_bytes, sort_bytes;
};
Layout4 layout4(int64_t S, int E, int H, int I) {
  Layout4 l{};
  const auto take = [&](size_t n) {
    const size_t at = l.bytes;
    l.bytes += (n + 255) / 256 * 256;
    return at;
  };
  l.counts = take((size_t)E * 4);
  l.offsets = take((size_t)(E + 1) * 4);
  l.row_src = take((size_t)S * 4);
  l.slot = take((size_t)S * 4);
  l.plan = take(l.plan_bytes = moe_amd_tile_plan_size(S, E));
  l.sort = take(l.sort_bytes = moe_amd_permute_workspace_size(S, E));
  l.act = take((size_t)S * I * 2);
  l.y = take((size_t)S * H * 2);
  l.ys = take((size_t)S * (H / kBlock16));
  return l;
}

int check_experts4(int64_t T, int K, int E, int H, int I, const char* who) {
  MOE_REQUIRE(T >= 0 && K >= 1 && E <= kPermuteExperts, MOE_ERR_ARG, "%s: T=%lld, K=%d or E=%d out of range",
              who, (long long)T, K, E);
  MOE_REQUIRE(T < (int64_t)1 << 31, MOE_ERR_UNSUPPORTED, "%s: T=%lld too large", who, (long long)T);
  const int rc = check4(T * K, E, H, I, who);
  if (rc) return rc;
  MOE_REQUIRE(T * (int64_t)H * 2 < ((int64_t)1 << 31), MOE_ERR_UNSUPPORTED, "%s: T*H too large", who);
  return MOE_OK;
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
  a.y = (_Float16*)y_out;
  a.ys = (uint8_t*)y_scale_out;
  a.K = I;
  a.N = H;
  a.kt = (I + kPack4Cols - 1) / kPack4Cols;
  a.nt = H / kPack4Rows;
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
  MOE_REQUIRE(H <= kMostColumns, MOE_ERR_UNSUPPORTED, "%s: H=%d above 2^22", who, H);
  if (T == 0) return MOE_OK;
  MOE_REQUIRE(y && y_scale && slot && offsets && topk_weights && out, MOE_ERR_ARG,
              "%s: null pointer", who);
  MOE_ALIGNED(y, who);
  MOE_ALIGNED(out, who);
  // few tokens: a row's columns to several waves; many: as many waves as are resident
  int64_t gx = (T + kCombineWaves - 1) / kCombineWaves;
  const int gy = gx >= 1024 ? 1 : (H + 512 * kPieces - 1) / (512 * kPieces);
  if (gx > 1024) gx = 1024;
  combine16_kernel<<<dim3((unsigned)gx, (unsigned)gy), 64 * kCombineWaves, 0, (hipStream_t)stream>>>(
      (const _Float16*)y, (const uint8_t*)y_scale, slot, offsets, topk_weights, weights_dtype, T, K, E,
      H, (bf16*)out);
  return check_launch(who);
}

extern "C" size_t moe_amd_experts4_workspace_size(int64_t T, int E, int K, int H, int I) {
  if (check_experts4(T, K, E, H, I, "experts4_workspace_size") != MOE_OK) return 0;
  return layout4(T * K, E, H, I).bytes;
}

extern "C" int moe_amd_experts4(const void* hidden_states, const int64_t* topk_index,
                                const void* topk_weights, int weights_dtype, const void* gate_up_q,
                                const void* gate_up_scale, const void* down_q,
                                const void* down_scale, int64_t T, int K, int E, int H, int I,
                                void* workspace, size_t workspace_bytes, void* out, void* stream) {
  const char* who = "experts4";
  int rc = check_experts4(T, K, E, H, I, who);
  if (rc) return rc;
  if (T == 0) return MOE_OK;
  // all of it before the first launch
  MOE_REQUIRE(weights_dtype == MOE_DTYPE_F32 || weights_dtype == MOE_DTYPE_BF16, MOE_ERR_DTYPE,
              "%s: weights dtype %d", who, weights_dtype);
  MOE_REQUIRE(hidden_states && topk_index && topk_weights && gate_up_q && gate_up_scale && down_q &&
                  down_scale && out,
              MOE_ERR_ARG, "%s: null pointer", who);
  MOE_ALIGNED(hidden_states, who);
  MOE_ALIGNED(gate_up_q, who);
  MOE_ALIGNED(gate_up_scale, who);
  MOE_ALIGNED(down_q, who);
  MOE_ALIGNED(down_scale, who);
  MOE_ALIGNED(out, who);
  const int64_t S = T * K;
  const Layout4 l = layout4(S, E, H, I);
  MOE_REQUIRE(workspace && workspace_bytes >= l.bytes, MOE_ERR_WORKSPACE,
              "%s: workspace of %zu bytes, needs %zu", who, workspace_bytes, l.bytes);
  MOE_ALIGNED(workspace, who);
  char* const ws = (char*)workspace;
  int* const offsets = (int*)(ws + l.offsets);
  int* const row_src = (int*)(ws + l.row_src);
  int* const slot = (int*)(ws + l.slot);
  char* const plan = ws + l.plan;
  if ((rc = moe_amd_permute(topk_index, S, E, ws + l.sort, l.sort_bytes, (int*)(ws + l.counts),
                            offsets, row_src, slot, plan, l.plan_bytes, stream)) ||
      (rc = moe_amd_gemm_gate_up_swiglu4(hidden_states, row_src, K, offsets, plan, gate_up_q,
                                         gate_up_scale, T, S, E, H, I, ws + l.act, stream)) ||
      (rc = moe_amd_gemm_down4(ws + l.act, offsets, plan, down_q, down_scale, S, E, H, I, ws + l.y,
                               ws + l.ys, stream)))
    return rc;
  return moe_amd_combine16(ws + l.y, ws + l.ys, slot, offsets, topk_weights, weights_dtype, T, K, E,
                           H, out, stream);
}
