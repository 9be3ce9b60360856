// The expert layer for a few tokens on a bank in 4 bits (gfx950): few.hip's
// function and routing, gate_up_proj and down_proj packed (pack4.h), bf16 hidden
// states, forward only.
//
//   g, u = gate_up_proj[e] x_t,  act = silu(g) u     (few4_gate_up_kernel)
//   y = down_proj[e] act                              (few4_down_kernel)
//   out_t = sum_k w[t,k] y                            (few4_combine_kernel)
//
// Bound by reading each routed expert's weights once, now 17/32 of a byte each.
// A wave takes 1 KB tiles (16 features by 128 of the contraction) as they lie, 16
// bytes a lane, which are the A operand of four MFMAs once four conversions a
// MFMA have made them bf16; B are the expert's tokens, lane (l % 16, l / 16)
// holding 32 of token l % 16's values.  The operands' order along the contraction is
// the tile's: any order that A and B share gives the same sum.
//
// A CU takes in about 28 KB/us, tokens from L2 included, so these stay in registers
// while a wave walks along an expert's tile rows (loaded anew for each: 44 us where
// it takes 36, T = 64, H = 2048, E = 128, K = 8, I = 768).  Weights are asked for one
// item ahead; nothing that a step waits for is asked for behind them, since loads
// complete in order.
//
// H = 2048, E = 128, K = 8, I = 768: 22 us for one token, 75 for 64 (gate/up 5.8 TB/s,
// down 4.4); E = 1792: 181 us (6.5 and 5.6 TB/s).  few.hip: 23, 215 and 620.
// The tokens stay in registers up to H = 2048 and I = 768 (kGateUpTiles, kDownTiles); beyond,
// they are loaded anew for each tile row: 64 tokens at H = 4096 take gate/up to 4.7 TB/s,
// at I = 1024 down to 2.5, and the whole call (routing given) 141 and 114 us, where the
// grouped products of gemm4.hip take 122 and 100.
//
// Sums are fp32; act is rounded to bf16, the next product's operand type, once
// (not at all for up to 16 rows of 12288 values together: kSmallRows, kSmallValues); y
// and the routing weights stay fp32 and each output is rounded once.  Partial sums are added in a fixed order, so results do
// not depend on timing.
//
// Reference: src/models/modeling_qwen3_moe.py:266-289, src/models/router.py:103-152,
// transformers/integrations/moe.py:377-478.
#include "few.h"
#include "pack4.h"

namespace moe {
namespace {

struct Few4Args {
  FewArgs f;
  const char *q1, *s1;  // gate_up_proj: codes and scales in tiles
  const char *q2, *s2;  // down_proj
  int kt1, kt2;         // tiles along H and along I
  int act32;            // act is fp32 (for few4_down_small_kernel)
  float* y;             // workspace: [S][H] by flat entry
};

// A tile of weights on its way to the MFMA: the lane's 32 codes of one row, and
// the row's four scale bytes.
struct Tile4 {
  u32x4 q;
  uint32_t s;
};
// C tiles of a tile row, `left` of which are there (the others read as zeros, without
// memory access), from q and s on.
template <int C>
__device__ __forceinline__ void load_tiles(Tile4 (&w)[C], const char* q, const char* s, int left,
                                           int lane) {
  left = left > 0 ? left : 0;
  const auto rq = make_rsrc(q, (uint32_t)left * kPack4Q), rs = make_rsrc(s, (uint32_t)left * kPack4S);
#pragma unroll
  for (int i = 0; i < C; ++i) {
    w[i].q = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(
                                           rq, lane * 16 + i * kPack4Q, 0, 2));  // non-temporal
    w[i].s = __builtin_amdgcn_raw_buffer_load_b32(rs, (lane & 15) * 4 + i * kPack4S, 0, 0);
  }
}
// A tile's 128 values of each of up to 16 rows of a bf16 operand, the lane's 32
// from byte `at` on; zeros from kNowhere on, without memory access.
constexpr uint32_t kNowhere = 0x80000000u;
struct Rows4 {
  u32x4 v[4];
};
__device__ __forceinline__ Rows4 load_rows(__amdgpu_buffer_rsrc_t x, uint32_t at) {
  Rows4 r;
#pragma unroll
  for (int j = 0; j < 4; ++j)
    r.v[j] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(x, at + j * 16, 0, 0));
  return r;
}
__device__ __forceinline__ f32x4 mma_tile(const Tile4& w, const Rows4& x, int g, f32x4 acc) {
  const float s = unpack4_scale(w.s >> (8 * g) & 0xffu);
#pragma unroll
  for (int j = 0; j < 4; ++j) acc = mma_step(bf16{}, unpack4_eight(w.q[j], s), x.v[j], acc);
  return acc;
}
// C tiles of each of the rows of x from tile k on, the lane's of which begins at byte
// `row` (kNowhere: none); the tiles from k1 and columns from `columns` on are not there.
template <int C>
__device__ __forceinline__ void load_rows(Rows4 (&v)[C], __amdgpu_buffer_rsrc_t x, uint32_t row,
                                          int columns, int k, int k1, int g) {
#pragma unroll
  for (int i = 0; i < C; ++i) {
    const bool in = k + i < k1 && (k + i) * kPack4Cols + g * kPack4Block < columns;
    v[i] = load_rows(x, in ? row + (uint32_t)((k + i) * (kPack4Cols * 2) + g * 64) : kNowhere);
  }
}

// Waves a SIMD of the two kernels that stream weights, with 8 and 6 KB in flight each: three
// by their registers.
constexpr int kOccupancy = 3;

// The plan in LDS.  (Loads complete in order: a row's number that is read from
// memory behind weights is waited for with them.)
struct Plan4 {
  int4 list[kFewRows];
  int rows[kFewRows];
};
__device__ __forceinline__ int load_plan(const FewArgs& f, Plan4& plan) {
  const int nact = f.hdr[0], S = f.T * f.K;
  for (int i = threadIdx.x; i < S; i += blockDim.x) {
    plan.list[i] = f.list[i];  // past the active experts: anything
    plan.rows[i] = f.rows[i];
  }
  __syncthreads();
  return __builtin_amdgcn_readfirstlane(nact);
}
__device__ __forceinline__ int4 uniform(int4 v) {
  return make_int4(__builtin_amdgcn_readfirstlane(v.x), __builtin_amdgcn_readfirstlane(v.y),
                   __builtin_amdgcn_readfirstlane(v.z), 0);
}

// ------------------------------------------------------- gate/up + SwiGLU
// Item: 16 features of one entry of the list, a tile row of gate and one of up, which
// share the tokens; a workgroup's waves split H.  With the plan in memory (NV = 0)
// a workgroup takes a run of items, most of them of one entry, whose tokens then stay
// in registers, and asks for the next item's weights as soon as it has used its own;
// else (gate_up_entry's other NV) it has one item.
constexpr int kGateUpWaves = 4;
constexpr int kGateUpTiles = 4;  // of each tile row in flight
template <int NV>
__global__ __launch_bounds__(64 * kGateUpWaves, kOccupancy) void few4_gate_up_kernel(Few4Args p) {
  __shared__ f32x4 red[2][kGateUpWaves][2][64];
  __shared__ typename std::conditional<NV == 0, Plan4, SmallPlan>::type plan;
  __shared__ int s_ids[64];
  const FewArgs& f = p.f;
  const int nsl = f.I / 16;
  const int lane = threadIdx.x & 63, n = lane & 15, g = lane >> 4;
  const int wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int item, end;
  int4 info;
  if constexpr (NV == 0) {
    const int64_t items = load_plan(f, plan) * nsl;
    item = (int)(blockIdx.x * items / gridDim.x);
    end = (int)((blockIdx.x + 1) * items / gridDim.x);
    if (item >= end) return;
    info = uniform(plan.list[item / nsl]);
  } else {
    item = blockIdx.x;
    end = item + 1;
    if (!gate_up_entry<NV>(f, item / nsl, lane, wid, plan, s_ids, info)) return;
  }
  const auto entry = [&](const int4& at, int i) {  // of its row i
    if constexpr (NV == 0) return plan.rows[at.y + i];
    else return plan.row[i];
  };
  const int k0 = wid * p.kt1 / kGateUpWaves, k1 = (wid + 1) * p.kt1 / kGateUpWaves;
  const auto xs = make_rsrc(f.x, (uint32_t)f.T * f.H * 2);
  Tile4 w[2][kGateUpTiles];
  Rows4 v[kGateUpTiles];
  const auto load = [&](const int4& at, int f0, int k, int k_end) {
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const int64_t t = (((int64_t)at.x * 2 + r) * nsl + f0) * p.kt1 + k;
      load_tiles<kGateUpTiles>(w[r], p.q1 + t * kPack4Q, p.s1 + t * kPack4S, k_end - k, lane);
    }
  };
  const auto load_x = [&](const int4& at, int k) {
    const uint32_t row = n < at.z ? (uint32_t)(entry(at, n) / f.K) * f.H * 2 : kNowhere;
    load_rows<kGateUpTiles>(v, xs, row, f.H, k, k1, g);
  };
  load(info, item % nsl, k0, k1);
  load_x(info, k0);
  int k = k0, turn = 0;
  f32x4 acc[2] = {};
  while (true) {
#pragma unroll
    for (int i = 0; i < kGateUpTiles; ++i)
#pragma unroll
      for (int r = 0; r < 2; ++r) acc[r] = mma_tile(w[r][i], v[i], g, acc[r]);
    const bool last = k + kGateUpTiles >= k1, more = item + 1 < end;
    const int next = last ? item + 1 : item;
    const bool other = last && more && next % nsl == 0;  // another entry
    int4 info_next = info;
    if constexpr (NV == 0)
      if (other) info_next = uniform(plan.list[next / nsl]);
    k = last ? k0 : k + kGateUpTiles;
    load(info_next, next % nsl, k, !last || more ? k1 : 0);
    if (other || k1 - k0 > kGateUpTiles) load_x(info_next, k);
    if (!last) continue;
    red[turn][wid][0][lane] = acc[0];
    red[turn][wid][1][lane] = acc[1];
    // lgkmcnt alone: the next weights stay in flight (this half of red is written again
    // after the next barrier)
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
    const int c = threadIdx.x & 15, r = threadIdx.x >> 4, l = (c >> 2) * 16 + r;
    if (r < info.z) {
      float gs = 0.f, us = 0.f;
#pragma unroll
      for (int q = 0; q < kGateUpWaves; ++q) {
        gs += red[turn][q][0][l][c & 3];
        us += red[turn][q][1][l][c & 3];
      }
      const int64_t at = (int64_t)entry(info, r) * f.I + item % nsl * 16 + c;
      const float act = siluf_(gs) * us;
      if (p.act32) ((float*)f.act)[at] = act;
      else ((bf16*)f.act)[at] = f2bf(act);
    }
    if (!more) return;
    item = next;
    info = info_next;
    turn ^= 1;
    acc[0] = acc[1] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
}

// ------------------------------------------------------------------- down
// Item: a tile row, 16 columns of the output, of an entry of the list.  A wave takes
// a run of items, most of them of one entry, whose rows then stay in registers (where
// I is at most 768: kDownTiles), and asks for the next item's weights as soon as it has
// used its own; y of a row goes to the workspace, which few4_combine_kernel reads.
constexpr int kDownWaves = 4;
constexpr int kDownTiles = 6;
__global__ __launch_bounds__(64 * kDownWaves, kOccupancy) void few4_down_kernel(Few4Args p) {
  __shared__ Plan4 plan;
  const FewArgs& f = p.f;
  const int lane = threadIdx.x & 63, n = lane & 15, g = lane >> 4;
  const int wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int ncol = f.H / 16;
  const int64_t items = (int64_t)load_plan(f, plan) * ncol;
  const int wave = blockIdx.x * kDownWaves + wid, waves = gridDim.x * kDownWaves;
  int item = (int)(wave * items / waves);
  const int end = (int)((wave + 1) * items / waves);
  if (item >= end) return;
  const auto as = make_rsrc(f.act, (uint32_t)f.T * f.K * f.I * 2);
  int4 info = uniform(plan.list[item / ncol]);
  Tile4 w[kDownTiles];
  Rows4 v[kDownTiles];
  const auto row = [&](const int4& at) { return n < at.z ? plan.rows[at.y + n] : -1; };
  const auto load = [&](const int4& at, int col, int k, int k_end) {
    const int64_t t = ((int64_t)at.x * ncol + col) * p.kt2 + k;
    load_tiles<kDownTiles>(w, p.q2 + t * kPack4Q, p.s2 + t * kPack4S, k_end - k, lane);
  };
  const auto load_act = [&](const int4& at, int k) {
    const int s = row(at);
    load_rows<kDownTiles>(v, as, s < 0 ? kNowhere : (uint32_t)s * f.I * 2, f.I, k, p.kt2, g);
  };
  load(info, item % ncol, 0, p.kt2);
  load_act(info, 0);
  int k = 0;
  f32x4 y = {0.f, 0.f, 0.f, 0.f};
  while (true) {
#pragma unroll
    for (int i = 0; i < kDownTiles; ++i) y = mma_tile(w[i], v[i], g, y);
    const bool last = k + kDownTiles >= p.kt2, more = item + 1 < end;
    const int next = last ? item + 1 : item;
    const bool other = last && more && next % ncol == 0;  // another entry
    const int4 info_next = other ? uniform(plan.list[next / ncol]) : info;
    k = last ? 0 : k + kDownTiles;
    load(info_next, next % ncol, k, !last || more ? p.kt2 : 0);
    if (other || p.kt2 > kDownTiles) load_act(info_next, k);
    if (!last) continue;
    const int s = row(info);
    if (s >= 0) *(f32x4*)(p.y + (int64_t)s * f.H + item % ncol * 16 + 4 * g) = y;
    if (!more) return;
    y = f32x4{0.f, 0.f, 0.f, 0.f};
    item = next;
    info = info_next;
  }
}

// out = sum over k, in order, of w y; four columns of a token a thread.  (In the down
// kernel, by the last workgroup of a column slice to arrive, y written through to
// memory: 36 us for 64 tokens where the two kernels take 23 and 5.)
__global__ __launch_bounds__(256) void few4_combine_kernel(Few4Args p) {
  const FewArgs& f = p.f;
  const int quads = f.H / 4, i = blockIdx.x * 256 + threadIdx.x;
  const int t = i / quads, c = i % quads * 4;
  if (t >= f.T) return;
  f32x4 o = {0.f, 0.f, 0.f, 0.f};
  for (int k0 = 0; k0 < f.K; k0 += 8) {
    float w[8];
    f32x4 y[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const int s = t * f.K + min(k0 + k, f.K - 1);
      const bool real = k0 + k < f.K && f.real[s] >= 0;
      w[k] = f.w[s];
      y[k] = *(const f32x4*)(p.y + (int64_t)s * f.H + c);
      if (!real) {  // padding's y was never written
        w[k] = 0.f;
        y[k] = f32x4{0.f, 0.f, 0.f, 0.f};
      }
    }
#pragma unroll
    for (int k = 0; k < 8; ++k)
#pragma unroll
      for (int j = 0; j < 4; ++j) o[j] = fmaf(w[k], y[k][j], o[j]);
  }
  *(u32x2*)((bf16*)f.out + (int64_t)t * f.H + c) = u32x2{pack_bf2(o[0], o[1]), pack_bf2(o[2], o[3])};
}

// Up to kSmallRows entries (one token, or two): a workgroup takes a tile row of every
// one, two waves each, and combines them itself, which saves a launch.  Their rows go
// through LDS (a load of a few of a wave's lanes costs a CU as much as one of all).
// They are fp32, split into two bf16 terms for two MFMAs: act is not rounded, whose
// rounding would be as much as a single token's few outputs' own.
constexpr int kSmallWaves = 16;
constexpr int kSmallRows = 16;
constexpr int kSmallTiles = 3;
constexpr int kSmallValues = 12288;  // of all rows
// v as a + r, both bf16 values once r is rounded: a the nearest one, or where that is
// infinite and v is not, the one next to v towards 0.  Where v is not finite, a alone
// (inf - inf would be NaN).
__device__ __forceinline__ void two_terms(float v, float& a, float& r) {
  a = round_bf(v);
  if (!(__builtin_fabsf(a) < INFINITY)) a = __uint_as_float(__float_as_uint(v) & 0xffff0000u);
  r = __builtin_fabsf(a) < INFINITY ? v - a : 0.f;
}
__global__ __launch_bounds__(64 * kSmallWaves) void few4_down_small_kernel(Few4Args p) {
  __shared__ __attribute__((aligned(16))) bf16 s_act[2][kSmallValues];  // the two terms
  __shared__ float s_y[2][kSmallRows][16];
  __shared__ float s_w[kSmallRows];
  __shared__ int s_real[kSmallRows];
  const FewArgs& f = p.f;
  const int tid = threadIdx.x, lane = tid & 63, n = lane & 15, g = lane >> 4;
  const int wid = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int col = blockIdx.x, ncol = f.H / 16, S = f.T * f.K, half = wid & 1;
  const int k0 = half * p.kt2 / 2, k1 = (half + 1) * p.kt2 / 2;
  // the plan in one round trip: lane i holds rows[i]
  const int my_row = f.rows[min(n, S - 1)], nact = f.hdr[0];
  int4 info = f.list[min(wid >> 1, S - 1)];
  const int my_real = f.real[min(n, S - 1)];
  const float my_w = f.w[min(n, S - 1)];
  Tile4 w[kSmallTiles];
  const auto load = [&](int k) {
    const int64_t t = ((int64_t)info.x * ncol + col) * p.kt2 + k;
    load_tiles<kSmallTiles>(w, p.q2 + t * kPack4Q, p.s2 + t * kPack4S, k1 - k, lane);
  };
  int q = wid >> 1;
  info = uniform(info);
  if (q < nact) load(k0);
  __builtin_amdgcn_sched_barrier(0);
  for (int i = tid; i < S * f.I / 4; i += 64 * kSmallWaves) {
    const f32x4 v = ((const f32x4*)f.act)[i];
    float a[4], r[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) two_terms(v[j], a[j], r[j]);
    *(u32x2*)&s_act[0][i * 4] = u32x2{pack_bf2(a[0], a[1]), pack_bf2(a[2], a[3])};
    *(u32x2*)&s_act[1][i * 4] = u32x2{pack_bf2(r[0], r[1]), pack_bf2(r[2], r[3])};
  }
  if (tid < S) {
    s_w[tid] = my_w;
    s_real[tid] = my_real;
  }
  __syncthreads();
  while (q < nact) {
    const int at_row = __shfl(my_row, (info.y + n) & 15, 64), s = n < info.z ? at_row : -1;
    f32x4 y = {0.f, 0.f, 0.f, 0.f};
    for (int k = k0; k < k1; k += kSmallTiles) {
      if (k != k0) load(k);
#pragma unroll
      for (int i = 0; i < kSmallTiles; ++i) {
        const int c = (k + i) * kPack4Cols + g * kPack4Block;
        Rows4 v[2];
#pragma unroll
        for (int term = 0; term < 2; ++term)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            v[term].v[j] = u32x4{0, 0, 0, 0};
            if (s >= 0 && k + i < k1 && c < f.I)
              v[term].v[j] = *(const u32x4*)&s_act[term][s * f.I + c + j * 8];
          }
        y = mma_tile(w[i], v[0], g, y);
        y = mma_tile(w[i], v[1], g, y);
      }
    }
    if (s >= 0) *(f32x4*)&s_y[half][s][4 * g] = y;
    q += kSmallWaves / 2;
    if (q < nact) {
      info = uniform(f.list[q]);
      load(k0);
    }
  }
  __syncthreads();
  for (int i = tid; i < f.T * 16; i += 64 * kSmallWaves) {
    const int t = i >> 4, c = i & 15;
    float o = 0.f;
    for (int k = 0; k < f.K; ++k) {
      const int s = t * f.K + k;
      if (s_real[s] >= 0) o = fmaf(s_w[s], s_y[0][s][c] + s_y[1][s][c], o);
    }
    ((bf16*)f.out)[(int64_t)t * f.H + col * 16 + c] = f2bf(o);
  }
}

// ------------------------------------------------------------------- host
bool few4_small(int S, int I) { return S <= kSmallRows && (int64_t)S * I <= kSmallValues; }

struct Few4Layout {
  FewLayout few;
  size_t y, bytes;
};
Few4Layout few4_layout(int T, int E, int K, int H, int I) {
  const bool small = few4_small(T * K, I);
  Few4Layout l{few_layout(T, E, K, I, small ? 4 : 2), 0, 0};
  l.y = l.few.bytes;
  l.bytes = small ? l.y : align_up(l.y + (size_t)T * K * H * 4, 256);
  return l;
}

int few4_run(Few4Args& p, void* workspace, size_t workspace_bytes, hipStream_t st,
             const char* who) {
  FewArgs& f = p.f;
  const Few4Layout l = few4_layout(f.T, f.E, f.K, f.H, f.I);
  MOE_REQUIRE(workspace && workspace_bytes >= l.bytes, MOE_ERR_WORKSPACE,
              "%s: workspace of %zu bytes, needs %zu", who, workspace_bytes, l.bytes);
  MOE_REQUIRE(al16(f.x) && al16(f.wr) && al16(p.q1) && al16(p.s1) && al16(p.q2) && al16(p.s2) &&
                  al16(f.out) && al16(workspace),
              MOE_ERR_ALIGN, "%s: pointers must be 16-byte aligned", who);
  few_bind(f, l.few, workspace);
  p.y = (float*)((char*)workspace + l.y);
  p.kt1 = (f.H + kPack4Cols - 1) / kPack4Cols;
  p.kt2 = (f.I + kPack4Cols - 1) / kPack4Cols;
  p.act32 = few4_small(f.T * f.K, f.I);
  const int slots = few_slots(f);
  // runs: as many workgroups as are resident at a time, and an item each at least
  const int most = kOccupancy * 256;
  const auto runs = [&](int64_t items) { return (int)(items < most ? items : most); };
  few_route<bf16>(f, st, [&](auto nv) {
    constexpr int NV = decltype(nv)::value;
    const int items = slots * (f.I / 16);
    few4_gate_up_kernel<NV><<<NV == 0 ? runs(items) : items, 64 * kGateUpWaves, 0, st>>>(p);
  });
  if (p.act32) {
    few4_down_small_kernel<<<f.H / 16, 64 * kSmallWaves, 0, st>>>(p);
  } else {
    few4_down_kernel<<<runs((slots * (f.H / 16) + kDownWaves - 1) / kDownWaves), 64 * kDownWaves, 0,
                       st>>>(p);
    few4_combine_kernel<<<(f.T * (f.H / 4) + 255) / 256, 256, 0, st>>>(p);
  }
  return check_launch(who);
}

}  // namespace
}  // namespace moe

using namespace moe;

extern "C" size_t moe_amd_few4_workspace_size(int64_t T, int E, int K, int H, int I) {
  if (few_check(T, K, E, H, I, MOE_DTYPE_BF16, "few4_workspace_size") != MOE_OK) return 0;
  return few4_layout((int)T, E, K, H, I).bytes;
}

extern "C" int moe_amd_experts_few4(const void* hidden_states, const int64_t* topk_index,
                                    const void* topk_weights, int weights_dtype,
                                    const void* gate_up_q, const void* gate_up_scale,
                                    const void* down_q, const void* down_scale, int64_t T, int K,
                                    int E, int H, int I, void* workspace, size_t workspace_bytes,
                                    void* out, void* stream) {
  const char* who = "experts_few4";
  const int rc = few_check(T, K, E, H, I, MOE_DTYPE_BF16, who);
  if (rc) return rc;
  MOE_REQUIRE(weights_dtype == MOE_DTYPE_F32 || weights_dtype == MOE_DTYPE_BF16, MOE_ERR_DTYPE,
              "%s: weights dtype %d", who, weights_dtype);
  if (T == 0) return MOE_OK;
  MOE_REQUIRE(hidden_states && topk_index && topk_weights && gate_up_q && gate_up_scale && down_q &&
                  down_scale && out,
              MOE_ERR_ARG, "%s: null pointer", who);
  Few4Args p{};
  p.f.x = hidden_states;
  p.f.ids = topk_index;
  p.f.weights = topk_weights;
  p.f.weights_bf16 = weights_dtype == MOE_DTYPE_BF16;
  p.f.T = (int)T;
  p.f.E = E;
  p.f.K = K;
  p.f.H = H;
  p.f.I = I;
  p.f.out = out;
  p.q1 = (const char*)gate_up_q;
  p.s1 = (const char*)gate_up_scale;
  p.q2 = (const char*)down_q;
  p.s2 = (const char*)down_scale;
  return few4_run(p, workspace, workspace_bytes, (hipStream_t)stream, who);
}

extern "C" int moe_amd_moe_layer_few4(const void* hidden_states, const void* router_weight,
                                      const void* gate_up_q, const void* gate_up_scale,
                                      const void* down_q, const void* down_scale, int64_t T, int K,
                                      int E, int H, int I, int router, const float* offset_or_bias,
                                      int renormalize, float scaling_factor, int num_groups,
                                      int group_topk, void* workspace, size_t workspace_bytes,
                                      float* topk_weights, int64_t* topk_index, void* out,
                                      void* stream) {
  const char* who = "moe_layer_few4";
  int rc = few_check(T, K, E, H, I, MOE_DTYPE_BF16, who);
  if (rc) return rc;
  rc = few_check_router(router, K, E, num_groups, group_topk, who);
  if (rc) return rc;
  if (T == 0) return MOE_OK;
  MOE_REQUIRE(hidden_states && router_weight && gate_up_q && gate_up_scale && down_q && down_scale &&
                  out,
              MOE_ERR_ARG, "%s: null pointer", who);
  Few4Args p{};
  p.f.x = hidden_states;
  p.f.wr = router_weight;
  few_set_router(p.f, router, offset_or_bias, renormalize, scaling_factor, num_groups, group_topk);
  p.f.T = (int)T;
  p.f.E = E;
  p.f.K = K;
  p.f.H = H;
  p.f.I = I;
  p.f.out_w = topk_weights;
  p.f.out_idx = topk_index;
  p.f.out = out;
  p.q1 = (const char*)gate_up_q;
  p.s1 = (const char*)gate_up_scale;
  p.q2 = (const char*)down_q;
  p.s2 = (const char*)down_scale;
  return few4_run(p, workspace, workspace_bytes, (hipStream_t)stream, who);
}
