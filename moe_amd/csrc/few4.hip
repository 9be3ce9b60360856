// The expert layer for a few tokens on a bank in 4 bits (gfx950): few.hip's
// function and routing, gate_up_proj and down_proj packed (pack4.h), bf16 hidden
// states, forward only.
//
//   g, u = gate_up_proj[e] x_t,  act = silu(g) u     (few4_gate_up_kernel)
//   out_t = sum_k w[t,k] down_proj[e] act             (few4_down_kernel)
//
// Bound by reading each routed expert's weights once, now 17/32 of a byte each.
// A wave takes 1 KB tiles (16 features by 128 of the contraction) as they lie, 16
// bytes a lane, which are the A operand of four MFMAs once four conversions a
// MFMA have made them bf16; B are the expert's tokens, lane (l % 16, l / 16)
// holding eight of token l % 16's values, loaded only where there is a token.  The
// operands' order along the contraction is the tile's: any order that A and B
// share gives the same sum.
//
// Sums are fp32; act is rounded to bf16, the next product's operand type, once;
// y and the routing weights stay fp32 and each output is rounded once.  Partial
// sums are added in a fixed order, so results do not depend on timing.
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
  float* y;             // workspace: [S][H] by flat entry
  int* arrived;         // [H / 16] workgroups of a column slice that are done
};

// A tile of weights on its way to the MFMA: the lane's 32 codes of one row, and
// the row's four scale bytes.
struct Tile4 {
  u32x4 q;
  uint32_t s;
};
__device__ __forceinline__ Tile4 load_tile(const char* q, const char* s, int64_t tile, int lane) {
  return {__builtin_nontemporal_load((const u32x4*)(q + tile * kPack4Q + lane * 16)),
          *(const uint32_t*)(s + tile * kPack4S + (lane & 15) * 4)};
}
// A tile's 128 values of each of up to 16 rows of a bf16 operand, the lane's 32
// from `row` on; none of a row or block that is not there.
struct Rows4 {
  u32x4 v[4];
};
__device__ __forceinline__ Rows4 load_rows(const char* row, bool there) {
  Rows4 r;
#pragma unroll
  for (int j = 0; j < 4; ++j) r.v[j] = u32x4{0, 0, 0, 0};
  if (there) {
#pragma unroll
    for (int j = 0; j < 4; ++j) r.v[j] = *(const u32x4*)(row + j * 16);
  }
  return r;
}
__device__ __forceinline__ f32x4 mma_tile(const Tile4& w, const Rows4& x, int g, f32x4 acc) {
  const float s = unpack4_scale(w.s >> (8 * g) & 0xffu);
#pragma unroll
  for (int j = 0; j < 4; ++j) acc = mma_step(bf16{}, unpack4_eight(w.q[j], s), x.v[j], acc);
  return acc;
}

// ------------------------------------------------------- gate/up + SwiGLU
// Workgroup: 16 features of one entry of the list, a tile row of gate and one of
// up, which share the tokens; the waves split H.  NV: gate_up_entry's.
constexpr int kGateUpTiles = 2;  // of each of the two that a wave has in flight
template <int NV>
__global__ __launch_bounds__(64 * kWaves) void few4_gate_up_kernel(Few4Args p) {
  __shared__ f32x4 red[kWaves][2][64];
  __shared__ SmallPlan small;
  __shared__ int s_ids[64];
  const FewArgs& f = p.f;
  const int nsl = f.I / 16;
  const int slot = blockIdx.x / nsl, f0 = (blockIdx.x % nsl) * 16;
  const int lane = threadIdx.x & 63, n = lane & 15, g = lane >> 4;
  const int wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (blockIdx.x == 0)
    for (int i = threadIdx.x; i < f.H / 16; i += 64 * kWaves) p.arrived[i] = 0;
  int4 info;
  if (!gate_up_entry<NV>(f, slot, lane, wid, small, s_ids, info)) return;
  const auto entry = [&](int i) { return NV != 0 ? small.row[i] : f.rows[info.y + i]; };
  const bool there = n < info.z;
  const char* x = (const char*)f.x + (int64_t)(entry(there ? n : 0) / f.K) * f.H * 2 + g * 64;
  const int64_t tg = ((int64_t)info.x * 2 * f.I + f0) / 16 * p.kt1;
  const int64_t tu = tg + (int64_t)f.I / 16 * p.kt1;
  f32x4 ag = {0.f, 0.f, 0.f, 0.f}, au = ag;
  chunks<kGateUpTiles>(wid * p.kt1 / kWaves, (wid + 1) * p.kt1 / kWaves, [&](auto ch, int k0) {
    constexpr int C = decltype(ch)::value;
    Tile4 wg[C], wu[C];
    Rows4 v[C];
#pragma unroll
    for (int i = 0; i < C; ++i) {
      wg[i] = load_tile(p.q1, p.s1, tg + k0 + i, lane);
      wu[i] = load_tile(p.q1, p.s1, tu + k0 + i, lane);
    }
#pragma unroll
    for (int i = 0; i < C; ++i)
      v[i] = load_rows(x + (k0 + i) * 256, there && (k0 + i) * kPack4Cols + g * kPack4Block < f.H);
#pragma unroll
    for (int i = 0; i < C; ++i) {
      ag = mma_tile(wg[i], v[i], g, ag);
      au = mma_tile(wu[i], v[i], g, au);
    }
  });
  red[wid][0][lane] = ag;
  red[wid][1][lane] = au;
  __syncthreads();
  if (threadIdx.x >= 256) return;
  const int c = threadIdx.x & 15, r = threadIdx.x >> 4, l = (c >> 2) * 16 + r;
  if (r >= info.z) return;
  float gs = 0.f, us = 0.f;
#pragma unroll
  for (int q = 0; q < kWaves; ++q) {
    gs += red[q][0][l][c & 3];
    us += red[q][1][l][c & 3];
  }
  ((bf16*)f.act)[(int64_t)entry(r) * f.I + f0 + c] = f2bf(siluf_(gs) * us);
}

// --------------------------------------------------------- down + combine
// Workgroup: 16 columns of the output and every `groups`-th kDownWaves entries of
// the list, a wave each; y of a row goes to the workspace, and the last
// workgroup of a column slice to arrive adds them with the routing weights, in k
// order.
constexpr int kDownWaves = 4;
constexpr int kDownTiles = 3;
__global__ __launch_bounds__(64 * kDownWaves) void few4_down_kernel(Few4Args p, int groups) {
  __shared__ int box;
  const FewArgs& f = p.f;
  const int slice = blockIdx.x / groups, group = blockIdx.x % groups;
  const int lane = threadIdx.x & 63, n = lane & 15, g = lane >> 4;
  const int wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int nact = f.hdr[0];
  for (int q = group * kDownWaves + wid; q < nact; q += groups * kDownWaves) {
    const int4 info = f.list[q];
    const bool there = n < info.z;
    const int s = f.rows[info.y + (there ? n : 0)];
    const char* a = (const char*)f.act + (int64_t)s * f.I * 2 + g * 64;
    const int64_t t0 = ((int64_t)info.x * (f.H / 16) + slice) * p.kt2;
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
    chunks<kDownTiles>(0, p.kt2, [&](auto ch, int k0) {
      constexpr int C = decltype(ch)::value;
      Tile4 w[C];
      Rows4 v[C];
#pragma unroll
      for (int i = 0; i < C; ++i) w[i] = load_tile(p.q2, p.s2, t0 + k0 + i, lane);
#pragma unroll
      for (int i = 0; i < C; ++i)
        v[i] = load_rows(a + (k0 + i) * 256,
                         there && (k0 + i) * kPack4Cols + g * kPack4Block < f.I);
#pragma unroll
      for (int i = 0; i < C; ++i) acc = mma_tile(w[i], v[i], g, acc);
    });
    if (there) {  // columns 4g .. 4g + 3 of the entry's row n
      float* y = p.y + (int64_t)s * f.H + slice * 16 + 4 * g;
#pragma unroll
      for (int i = 0; i < 4; ++i) put_shared((int*)y + i, __float_as_int(acc[i]));
    }
  }
  if (!last_to_arrive(&p.arrived[slice], groups, &box)) return;
  for (int v = threadIdx.x; v < f.T * 16; v += 64 * kDownWaves) {
    const int t = v >> 4, h = slice * 16 + (v & 15);
    float o = 0.f;
    for (int k0 = 0; k0 < f.K; k0 += 8) {
      float w[8], y[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const int s = t * f.K + min(k0 + k, f.K - 1);
        const bool real = k0 + k < f.K && f.real[s] >= 0;  // padding's y was never written
        w[k] = real ? f.w[s] : 0.f;
        y[k] = real ? __int_as_float(get_shared((const int*)p.y + (int64_t)s * f.H + h)) : 0.f;
      }
#pragma unroll
      for (int k = 0; k < 8; ++k) o = fmaf(w[k], y[k], o);
    }
    ((bf16*)f.out)[(int64_t)t * f.H + h] = f2bf(o);
  }
}

// ------------------------------------------------------------------- host
struct Few4Layout {
  FewLayout few;
  size_t y, arrived, bytes;
};
Few4Layout few4_layout(int T, int E, int K, int H, int I) {
  Few4Layout l{few_layout(T, E, K, I, 2), 0, 0, 0};
  l.y = l.few.bytes;
  l.arrived = align_up(l.y + (size_t)T * K * H * 4, 256);
  l.bytes = align_up(l.arrived + (size_t)H / 16 * 4, 256);
  return l;
}

int few4_run(Few4Args& p, void* workspace, size_t workspace_bytes, hipStream_t st,
             const char* who) {
  FewArgs& f = p.f;
  const Few4Layout l = few4_layout(f.T, f.E, f.K, f.H, f.I);
  MOE_REQUIRE(workspace && workspace_bytes >= l.bytes, MOE_ERR_WORKSPACE,
              "%s: workspace of %zu bytes, needs %zu", who, workspace_bytes, l.bytes);
  MOE_REQUIRE(al16(f.x) && al16(f.wr) && al16(p.q1) && al16(p.s1) && al16(p.q2) && al16(p.s2) &&
                  al16(workspace),
              MOE_ERR_ALIGN, "%s: pointers must be 16-byte aligned", who);
  few_bind(f, l.few, workspace);
  p.y = (float*)((char*)workspace + l.y);
  p.arrived = (int*)((char*)workspace + l.arrived);
  p.kt1 = (f.H + kPack4Cols - 1) / kPack4Cols;
  p.kt2 = (f.I + kPack4Cols - 1) / kPack4Cols;
  const int slots = few_slots(f), slices = f.H / 16;
  few_route<bf16>(f, st, [&](auto nv) {
    few4_gate_up_kernel<decltype(nv)::value><<<slots * (f.I / 16), 64 * kWaves, 0, st>>>(p);
  });
  const int most = (slots + kDownWaves - 1) / kDownWaves;
  int groups = 2048 / slices;
  if (groups > most) groups = most;
  if (groups < 1) groups = 1;
  few4_down_kernel<<<slices * groups, 64 * kDownWaves, 0, st>>>(p, groups);
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
