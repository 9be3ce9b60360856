// The expert layer for a few tokens (gfx950): router, experts and combine for
// T <= 64 tokens, forward only.
//
//   logits[t,e] = <x_t, W_r[e]>, then softmax or sigmoid top-K (few_plan_kernel)
//   g, u = gate_up_proj[e] x_t,  act = silu(g) u     (few_gate_up_kernel)
//   out_t = sum_k w[t,k] down_proj[e] act             (few_down_kernel)
//
// What bounds it is reading each routed expert's three matrices once: a few
// rows per expert leave the matrix units idle.  The weights therefore go from
// memory to the MFMA as the 16 rows of its A operand (output features), with
// the expert's tokens as the 16 columns of B, every wave's loads in flight
// together and the bytes dealt evenly to the CUs.  Partial sums are added in a
// fixed order, so results do not depend on timing.
//
// H = 2048, E = 128, K = 8, I = 768, bf16, fresh weights: 23 us for one token
// (75 MB), 215 us for 64 (1.18 GB: gate/up 5.9 TB/s, down 5.7); E = 1792, 64
// tokens 620 us (3.8 GB).  The layer by grouped GEMMs takes 95, 292 and 750.
//
// Sums are fp32 (the logits' across waves fp64); act is rounded to x's type,
// the next product's operand type, once; everything else is rounded once at
// the output.  The routing weights stay fp32.
//
// Reference: src/models/modeling_qwen3_moe.py:266-289 (router and block),
// src/models/router.py:103-152 (sigmoid router),
// transformers/integrations/moe.py:377-478 (experts).
#include "few.h"

namespace moe {
namespace {

// Blocks in flight of a gate/up wave: two leave room for four workgroups a CU (T = 64,
// E = 128: 218 us; four and two workgroups 228, one 219).
constexpr int kGateUpChunk = 2;
constexpr int kMaxLds = kWaves * kBlockLds + kFewRows * (16 + 64 + 12);  // of the down kernel

// ------------------------------------------------------- gate/up + SwiGLU
// Workgroup: 8 features of one entry of the list, their gate and up rows being
// the 16 rows of the A operand; the waves split H, CH blocks in flight each.  A
// CU takes in about 24 KB/us whatever else is idle, so the weights are dealt to
// all of them in small pieces: with 16 features a workgroup one token (K = 8,
// I = 768) has 384 for 256 CUs.
// NV: gate_up_entry's.
template <typename T, int CH, int NV>
__global__ __launch_bounds__(64 * kWaves) void few_gate_up_kernel(FewArgs p) {
  __shared__ __attribute__((aligned(16))) char turn[kWaves][kBlockLds];
  __shared__ SmallPlan small;
  __shared__ int s_ids[64];
  const int nsl = p.I / 8;
  const int slot = blockIdx.x / nsl, f0 = (blockIdx.x % nsl) * 8;
  const int lane = threadIdx.x & 63;
  const int wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int4 info;
  if (!gate_up_entry<NV>(p, slot, lane, wid, small, s_ids, info)) return;
  const int nb = p.H * (int)sizeof(T) / kBlock, row = lane >> 3;
  const uint32_t ld = (uint32_t)p.H * sizeof(T), j = (lane & 7) * 16;
  const char* wg = (const char*)p.w1 + ((int64_t)info.x * 2 * p.I + f0) * ld;
  const char* wu = wg + (int64_t)p.I * ld;
  const uint32_t wo = row * ld + j;
  const auto entry = [&](int i) {  // of row i, or the last
    i = min(i, info.z - 1);
    return NV != 0 ? small.row[i] : p.rows[info.y + i];
  };
  const uint32_t x0 = (uint32_t)(entry(row) / p.K) * ld + j;
  const uint32_t x1 = (uint32_t)(entry(row + 8) / p.K) * ld + j;
  f32x4 acc = {0.f, 0.f, 0.f, 0.f};
  chunks<CH>(wid * nb / kWaves, (wid + 1) * nb / kWaves, [&](auto ch, int s) {
    constexpr int C = decltype(ch)::value;
    const char *gs = wg + s * kBlock, *us = wu + s * kBlock, *xs = (const char*)p.x + s * kBlock;
    Block v[C];
#pragma unroll
    for (int i = 0; i < C; ++i) {
      v[i].a0 = ld16(gs, wo, i * kBlock);
      v[i].a1 = ld16(us, wo, i * kBlock);
    }
#pragma unroll
    for (int i = 0; i < C; ++i) {
      v[i].b0 = ld16(xs, x0, i * kBlock);
      v[i].b1 = ld16(xs, x1, i * kBlock);
    }
#pragma unroll
    for (int i = 0; i < C; ++i) acc = mma_block<T>(v[i], turn[wid], lane, acc);
  });
  f32x4(*red)[kBlockLds / 16] = (f32x4(*)[kBlockLds / 16])turn;  // in each wave's own part
  red[wid][lane] = acc;
  __syncthreads();
  if (threadIdx.x >= 128) return;
  const int f = threadIdx.x & 7, r = threadIdx.x >> 3, l = (f >> 2) * 16 + r;
  if (r >= info.z) return;
  float gs = 0.f, us = 0.f;
#pragma unroll
  for (int q = 0; q < kWaves; ++q) {
    gs += red[q][l][f & 3];
    us += red[q][l + 32][f & 3];
  }
  ((T*)p.act)[(int64_t)entry(r) * p.I + f0 + f] = (T)(siluf_(gs) * us);
}

// --------------------------------------------------------- down + combine
// Workgroup: C = 16 / parts columns of the output and every entry of the list; a
// wave takes the next one when it is done with its own (the oldest waves get
// their loads first: with a fixed share each, they end after half of the time
// and the rest finishes with too few loads in flight).  `parts` makes the column slices about as many
// as CUs where it divides the contraction's blocks: the A operand's 16 rows are
// C columns' weights for each of `parts` pieces of the contraction, B's 16
// columns C of the expert's rows for each of them, and the blocks of the product
// where the pieces match are added.
// A wave needs no other one: it reads CH blocks and the next CH before it
// multiplies these, and leaves y in LDS, where the workgroup then sums it with
// the routing weights, in k order.
template <typename T, int CH>
__global__ __launch_bounds__(64 * kWaves) void few_down_kernel(FewArgs p, int parts) {
  extern __shared__ __attribute__((aligned(16))) char lds[];
  const int S = p.T * p.K, C = 16 / parts;
  int4* s_list = (int4*)(lds + kWaves * kBlockLds);
  float* s_y = (float*)(s_list + S);   // [S][C]
  int* s_rows = (int*)(s_y + S * C);
  float* s_w = (float*)(s_rows + S);
  int* s_real = (int*)(s_w + S);
  __shared__ int s_next;
  const int h0 = blockIdx.x * C;
  const int tid = threadIdx.x, lane = tid & 63, n = lane & 15, g = lane >> 4;
  const int wid = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int nact = p.hdr[0];
  for (int i = tid; i < S; i += 64 * kWaves) {
    s_list[i] = p.list[i];  // past the active experts: anything
    s_rows[i] = p.rows[i];
    s_w[i] = p.w[i];
    s_real[i] = p.real[i];
  }
  if (tid == 0) s_next = kWaves;
  __syncthreads();
  const int nb = p.I * (int)sizeof(T) / kBlock / parts;  // of a piece
  const uint32_t ld = (uint32_t)p.I * sizeof(T);
  struct Pos {
    int q, rg, sb;
    bool more;
    int4 info;
    const char* w;
    uint32_t b0, b1;
  };
  // the lane's two rows of a tile: a column or an entry's row, and a piece
  const int c0 = (lane >> 3) % C, c1 = ((lane >> 3) + 8) % C;
  const uint32_t j = (lane & 7) * 16;
  const uint32_t p0 = (lane >> 3) / C * nb * kBlock + j, p1 = ((lane >> 3) + 8) / C * nb * kBlock + j;
  const uint32_t a0 = c0 * ld + p0, a1 = c1 * ld + p1;
  auto start = [&](Pos& c) {
    c.more = c.q < nact;
    if (!c.more) return;
    c.info = s_list[c.q];
    c.w = (const char*)p.w2 + ((int64_t)c.info.x * p.H + h0) * (int64_t)ld;
  };
  auto rows = [&](Pos& c) {
    const int left = c.info.z - c.rg - 1, at = c.info.y + c.rg;
    c.b0 = (uint32_t)s_rows[at + min(c0, left)] * ld + p0;
    c.b1 = (uint32_t)s_rows[at + min(c1, left)] * ld + p1;
  };
  auto next = [&](Pos c) {  // without one: more false, the addresses as they were
    if (c.sb + CH < nb) {
      c.sb += CH;
      return c;
    }
    c.sb = 0;
    c.rg += C;
    if (c.rg >= c.info.z) {
      c.rg = 0;
      int q = 0;
      if (lane == 0) q = atomicAdd(&s_next, 1);
      c.q = __builtin_amdgcn_readfirstlane(q);
      start(c);
    }
    if (c.more) rows(c);
    return c;
  };
  // The last chunk of a contraction that CH does not divide starts earlier: its
  // first blocks are the previous chunk's and are passed over.
  auto load = [&](const Pos& c, Block (&v)[CH]) {
    const int sb = min(c.sb, nb - CH);
    const char *ws = c.w + sb * kBlock, *as = (const char*)p.act + sb * kBlock;
#pragma unroll
    for (int i = 0; i < CH; ++i) {
      v[i].a0 = ld16(ws, a0, i * kBlock);
      v[i].a1 = ld16(ws, a1, i * kBlock);
    }
#pragma unroll
    for (int i = 0; i < CH; ++i) {
      v[i].b0 = ld16(as, c.b0, i * kBlock);
      v[i].b1 = ld16(as, c.b1, i * kBlock);
    }
  };
  f32x4 acc = {0.f, 0.f, 0.f, 0.f};
  auto step = [&](const Pos& c, const Block (&v)[CH]) {
    const int skip = c.sb - min(c.sb, nb - CH);
#pragma unroll
    for (int i = 0; i < CH; ++i)
      if (i >= skip) acc = mma_block<T>(v[i], lds + wid * kBlockLds, lane, acc);
    if (c.sb + CH < nb) return;
    // lane (n, g) holds rows 4g .. 4g+3 of column n: the block of piece f starts
    // 16 (C/4) + C = 5C lanes after that of piece f - 1
    f32x4 y = acc;
    for (int f = 1; f < parts; ++f)
#pragma unroll
      for (int i = 0; i < 4; ++i) y[i] += __shfl(acc[i], lane + 5 * C * f, 64);
    if (n < C && 4 * g < C && n < c.info.z - c.rg)
      *(f32x4*)&s_y[s_rows[c.info.y + c.rg + n] * C + 4 * g] = y;
    acc = f32x4{0.f, 0.f, 0.f, 0.f};
  };
  Pos c{};
  c.q = wid;
  start(c);
  if (c.more) {
    Block u[CH], v[CH];
    rows(c);
    load(c, u);
    // Past the wave's last entry the last addresses are loaded again, unused:
    // with a branch around the loads the compiler waits for all of them.
    while (true) {
      const Pos d = next(c);
      load(d, v);
      step(c, u);
      if (!d.more) break;
      c = next(d);
      load(c, u);
      step(d, v);
      if (!c.more) break;
    }
  }
  __syncthreads();
  for (int v = tid; v < p.T * C; v += 64 * kWaves) {
    const int t = v / C, h = v % C;
    float o = 0.f;
    for (int k0 = 0; k0 < p.K; k0 += 8) {
      float w[8], y[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const int s = t * p.K + min(k0 + k, p.K - 1);
        const bool real = k0 + k < p.K && s_real[s] >= 0;
        w[k] = s_w[s];
        y[k] = s_y[s * C + h];
        if (!real) w[k] = y[k] = 0.f;  // padding's y was never written
      }
#pragma unroll
      for (int k = 0; k < 8; ++k) o = fmaf(w[k], y[k], o);
    }
    ((T*)p.out)[(int64_t)t * p.H + h0 + h] = (T)o;
  }
}

// ------------------------------------------------------------------- host
template <typename T>
hipError_t few_launch(const FewArgs& p, hipStream_t st) {
  const int gu_grid = few_slots(p) * (p.I / 8);
  few_route<T>(p, st, [&](auto nv) {
    few_gate_up_kernel<T, kGateUpChunk, decltype(nv)::value><<<gu_grid, 64 * kWaves, 0, st>>>(p);
  });
  const int S = p.T * p.K;
  // Column slices of 16 / parts: about one for every CU, where the contraction has
  // a multiple of parts blocks.  With an odd number there are H / 16, too few below
  // H = 4096: bf16, E = 128, T = 64, I = 704 (11 blocks) and 768 (12), H = 1024:
  // 83 and 54 us (2.2 and 3.8 TB/s), H = 2048: 89 and 68 (4.1 and 5.9).
  int parts = p.H / 16 >= 256 ? 1 : p.H / 8 >= 256 ? 2 : 4;
  const int blocks = p.I * (int)sizeof(T) / kBlock;
  while (blocks % parts) parts /= 2;
  const int nb = blocks / parts;
  const int lds = kWaves * kBlockLds + S * (16 + 64 / parts + 12);
  // Two blocks in flight and the next two are enough (three, or four: the same at
  // T = 64, 0.5 of 25 us more at T = 1); never more than there are, as a block past
  // the end is another row's or nobody's.
  auto down = [&](auto c) -> hipError_t {
    static std::atomic<int> done[64];
    constexpr int CH = decltype(c)::value;
    const void* f = (const void*)few_down_kernel<T, CH>;
    if (lds > 65536) {
      const hipError_t err = set_dynamic_lds_once(done, f, kMaxLds);
      if (err != hipSuccess) return err;
    }
    few_down_kernel<T, CH><<<p.H * parts / 16, 64 * kWaves, lds, st>>>(p, parts);
    return hipSuccess;
  };
  if (nb >= 2) return down(std::integral_constant<int, 2>{});
  return down(std::integral_constant<int, 1>{});
}

int few_run(FewArgs& p, int dtype, void* workspace, size_t workspace_bytes, hipStream_t st,
            const char* who) {
  const FewLayout l = few_layout(p.T, p.E, p.K, p.I, dtype == MOE_DTYPE_BF16 ? 2 : 4);
  MOE_REQUIRE(workspace && workspace_bytes >= l.bytes, MOE_ERR_WORKSPACE,
              "%s: workspace of %zu bytes, needs %zu", who, workspace_bytes, l.bytes);
  MOE_REQUIRE(al16(p.x) && al16(p.wr) && al16(p.w1) && al16(p.w2) && al16(workspace),
              MOE_ERR_ALIGN, "%s: pointers must be 16-byte aligned", who);
  few_bind(p, l, workspace);
  const hipError_t err =
      dtype == MOE_DTYPE_BF16 ? few_launch<bf16>(p, st) : few_launch<float>(p, st);
  MOE_REQUIRE(err == hipSuccess, MOE_ERR_HIP, "%s: HIP error %d (%s)", who, (int)err,
              hipGetErrorString(err));
  return check_launch(who);
}

}  // namespace
}  // namespace moe

using namespace moe;

extern "C" size_t moe_amd_few_workspace_size(int64_t T, int E, int K, int H, int I, int dtype) {
  if (few_check(T, K, E, H, I, dtype, "few_workspace_size") != MOE_OK) return 0;
  return few_layout((int)T, E, K, I, dtype == MOE_DTYPE_BF16 ? 2 : 4).bytes;
}

extern "C" int moe_amd_experts_few(const void* hidden_states, const int64_t* topk_index,
                                   const void* topk_weights, int weights_dtype,
                                   const void* gate_up_proj, const void* down_proj, int64_t T,
                                   int K, int E, int H, int I, int dtype, void* workspace,
                                   size_t workspace_bytes, void* out, void* stream) {
  const char* who = "experts_few";
  int rc = few_check(T, K, E, H, I, dtype, who);
  if (rc) return rc;
  MOE_REQUIRE(weights_dtype == MOE_DTYPE_F32 || weights_dtype == MOE_DTYPE_BF16, MOE_ERR_DTYPE,
              "%s: weights dtype %d", who, weights_dtype);
  if (T == 0) return MOE_OK;
  MOE_REQUIRE(hidden_states && topk_index && topk_weights && gate_up_proj && down_proj && out,
              MOE_ERR_ARG, "%s: null pointer", who);
  FewArgs p{};
  p.x = hidden_states;
  p.w1 = gate_up_proj;
  p.w2 = down_proj;
  p.ids = topk_index;
  p.weights = topk_weights;
  p.weights_bf16 = weights_dtype == MOE_DTYPE_BF16;
  p.T = (int)T;
  p.E = E;
  p.K = K;
  p.H = H;
  p.I = I;
  p.out = out;
  return few_run(p, dtype, workspace, workspace_bytes, (hipStream_t)stream, who);
}

extern "C" int moe_amd_moe_layer_few(const void* hidden_states, const void* router_weight,
                                     const void* gate_up_proj, const void* down_proj, int64_t T,
                                     int K, int E, int H, int I, int dtype, int router,
                                     const float* offset_or_bias, int renormalize,
                                     float scaling_factor, int num_groups, int group_topk,
                                     void* workspace, size_t workspace_bytes, float* topk_weights,
                                     int64_t* topk_index, void* out, void* stream) {
  const char* who = "moe_layer_few";
  int rc = few_check(T, K, E, H, I, dtype, who);
  if (rc) return rc;
  rc = few_check_router(router, K, E, num_groups, group_topk, who);
  if (rc) return rc;
  if (T == 0) return MOE_OK;
  MOE_REQUIRE(hidden_states && router_weight && gate_up_proj && down_proj && out, MOE_ERR_ARG,
              "%s: null pointer", who);
  FewArgs p{};
  p.x = hidden_states;
  p.wr = router_weight;
  p.w1 = gate_up_proj;
  p.w2 = down_proj;
  few_set_router(p, router, offset_or_bias, renormalize, scaling_factor, num_groups, group_topk);
  p.T = (int)T;
  p.E = E;
  p.K = K;
  p.H = H;
  p.I = I;
  p.out_w = topk_weights;
  p.out_idx = topk_index;
  p.out = out;
  return few_run(p, dtype, workspace, workspace_bytes, (hipStream_t)stream, who);
}
