// The expert layer for a few tokens (gfx950): router, experts and combine for
// T <= 64 tokens, forward only.
//
//   logits[t,e] = <x_t, W_r[e]>, then softmax or sigmoid top-K (few_plan_kernel)
//   g, u = gate_up_proj[e] x_t,  act = silu(g) u     (few_gate_up_kernel)
//   out_t = sum_k w[t,k] down_proj[e] act             (few_down_kernel)
//
// What bounds it is reading each routed expert's three matrices once: a few
// rows per expert leave the matrix units idle.  The weights therefore stream
// straight from memory into MFMA operands, as the 16 rows of the A operand
// (output features), with the expert's tokens as the 16 columns of B; no
// staging in LDS, every wave's loads in flight together.  A workgroup's eight
// waves split the contraction and add their partial sums in LDS in a fixed
// order, so results do not depend on timing.
//
// Sums are fp32 (the logits' across waves fp64); act is rounded to x's type,
// the next product's operand type, once; everything else is rounded once at
// the output.  The routing weights stay fp32.
//
// Reference: src/models/modeling_qwen3_moe.py:266-289 (router and block),
// src/models/router.py:103-152 (sigmoid router),
// transformers/integrations/moe.py:377-478 (experts).
#include "common.h"
#include "router_group.h"

namespace moe {
namespace {

constexpr int kFewTokens = MOE_FEW_MAX_TOKENS;
constexpr int kFewTopK = MOE_FEW_MAX_TOP_K;
constexpr int kFewExperts = 4096;
constexpr int kFewRows = kFewTokens * kFewTopK;
constexpr int kWaves = 8;        // waves per workgroup of the GEMV kernels
constexpr int kPlanWaves = 16;
constexpr int kRouteWaves = 4;   // tokens per workgroup of the routing
constexpr int kGroup = 4;        // experts per workgroup of the down kernel
constexpr int kParts = kWaves / kGroup;  // waves that split one expert's contraction there

struct FewArgs {
  const void* x;           // [T,H]
  const void* wr;          // [E,H] (null: routing given)
  const void* w1;          // [E,2I,H]
  const void* w2;          // [E,H,I]
  const float* offset;     // logit offset (softmax) or selection bias (sigmoid) [E], or null
  const int64_t* ids;      // given routing [T*K]
  const void* weights;     // given routing weights [T*K]
  int weights_bf16, sigmoid, renorm, ngroups, gtopk;
  float scaling;
  int T, E, K, H, I;
  float* logits;           // workspace from here on
  float* w;                // [S]
  int* hdr;                // [0] active experts, [1] finished routing workgroups
  int* arrived;            // [H/16] finished groups of the down kernel's column slices
  int4* list;              // {expert, first row, rows, 0} of the active experts
  int* rows;               // flat entries s = t*K + k by active expert, ascending
  void* act;               // [S,I] by flat entry
  float* y;                // [S,H]
  int* real;               // [S] the entry's expert, negative for padding
  float* out_w;            // routing out (may be null)
  int64_t* out_idx;
  void* out;
};

template <typename T> struct Mma;
// One step of a contraction: 64 bytes of each of 16 rows, lane l holding 16
// bytes of row l % 16 at chunk l / 16; A and B alike, so which k a lane's
// elements are does not matter.
template <> struct Mma<bf16> {
  static constexpr int kStep = 32;
  static __device__ __forceinline__ f32x4 step(const u32x4& a, const u32x4& b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a),
                                                   __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  }
};
template <> struct Mma<float> {
  static constexpr int kStep = 16;
  static __device__ __forceinline__ f32x4 step(const u32x4& a, const u32x4& b, f32x4 c) {
    const f32x4 fa = __builtin_bit_cast(f32x4, a), fb = __builtin_bit_cast(f32x4, b);
#pragma unroll
    for (int i = 0; i < 4; ++i)
      c = __builtin_amdgcn_mfma_f32_16x16x4f32(fa[i], fb[i], c, 0, 0, 0);
    return c;
  }
};

__device__ __forceinline__ u32x4 ld16(const char* p) { return *(const u32x4*)p; }
#ifndef FEW_NT
#define FEW_NT 0
#endif
__device__ __forceinline__ u32x4 ld16_w(const char* p) {
#if FEW_NT
  return __builtin_nontemporal_load((const u32x4*)p);
#else
  return *(const u32x4*)p;
#endif
}

template <typename T> __device__ __forceinline__ float few_round(float v) {
  if constexpr (sizeof(T) == 2) return round_bf(v);
  return v;
}

// The counters that workgroups of later launches finish by.
__device__ __forceinline__ void clear_counters(const FewArgs& p) {
  if (threadIdx.x == 0) p.hdr[1] = 0;
  for (int i = threadIdx.x; i < p.H / 16; i += blockDim.x) p.arrived[i] = 0;
}

// What one workgroup leaves for another of the same launch: written through to
// and read from the memory that all XCDs share, so that no cache has to be
// written back or invalidated.  A workgroup counts itself as arrived once its
// writes are there; the last one to arrive reads everybody's.
__device__ __forceinline__ void put_shared(float* p, float v) {
  __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ float get_shared(const float* p) {
  return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ void put_shared(int* p, int v) {
  __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ int get_shared(const int* p) {
  return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ bool last_to_arrive(int* counter, int of, int* box) {
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // this wave's writes are there
  __syncthreads();
  if (threadIdx.x == 0)
    *box = __hip_atomic_fetch_add(counter, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == of - 1;
  __syncthreads();
  return *box;
}

// ---------------------------------------------------------------- logits
// Workgroup: 16 experts and 16 tokens; the eight waves split H.  The first one
// clears the counters of the launches behind it.
template <typename T>
__global__ __launch_bounds__(64 * kWaves) void few_logits_kernel(FewArgs p) {
  __shared__ f32x4 red[kWaves][64];
  const int lane = threadIdx.x & 63, n = lane & 15, g = lane >> 4;
  const int wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int e0 = blockIdx.x * 16;
  const int ns = p.H / Mma<T>::kStep;
  const int s0 = wid * ns / kWaves, s1 = (wid + 1) * ns / kWaves;
  const int64_t ld = (int64_t)p.H * sizeof(T);
  const char* a = (const char*)p.wr + (int64_t)min(e0 + n, p.E - 1) * ld + g * 16;
  const int t0 = blockIdx.y * 16;
  const char* b = (const char*)p.x + (int64_t)min(t0 + n, p.T - 1) * ld + g * 16;
  f32x4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 8
  for (int s = s0; s < s1; ++s) acc = Mma<T>::step(ld16(a + s * 64), ld16(b + s * 64), acc);
  red[wid][lane] = acc;
  if (blockIdx.x == 0 && blockIdx.y == 0) clear_counters(p);
  __syncthreads();
  if (threadIdx.x < 256) {
    const int e = threadIdx.x & 15, t = threadIdx.x >> 4;
    double v = 0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) v += (double)red[w][(e >> 2) * 16 + t][e & 3];
    if (t0 + t < p.T && e0 + e < p.E) {
      const float f = (float)v;
      // the softmax router's logits have x's type, as the model's linear returns them
      p.logits[(int64_t)(t0 + t) * p.E + e0 + e] = p.sigmoid ? f : few_round<T>(f);
    }
  }
}

// ------------------------------------------------------- routing and plan
// The largest key of the wave below thr (0: none).
template <int NV>
__device__ __forceinline__ uint64_t wave_next_key(const uint64_t (&key)[NV], uint64_t thr) {
  const uint64_t b = group_max_key<16>(lane_next_key<NV>(key, thr));
  uint64_t w = readlane_u64(b, 0);
#pragma unroll
  for (int r = 16; r < 64; r += 16) {
    const uint64_t o = readlane_u64(b, r);
    w = o > w ? o : w;
  }
  return w;
}

// One token on one wave: lane k < K gets its k-th expert and weight.  The
// selections and the arithmetic are those of the router kernels.
template <int NV>
__device__ void route_token(const FewArgs& p, const float* logits, int lane, float& wk, int& ek) {
  const int E = p.E, K = p.K;
  uint64_t key[NV], kk;
  if (!p.sigmoid) {
    float v[NV];
    bool nan_here = false;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int e = j * 64 + lane;
      v[j] = e < E ? logits[e] + (p.offset ? p.offset[e] : 0.f) : -INFINITY;
      nan_here |= v[j] != v[j];
    }
    if (__ballot(nan_here)) {  // every prob of the row is NaN: they rank by index
#pragma unroll
      for (int j = 0; j < NV; ++j)
        if (j * 64 + lane < E) v[j] = __builtin_nanf("");
    }
    float m = -INFINITY;
#pragma unroll
    for (int j = 0; j < NV; ++j) m = fmaxf(m, v[j]);
    m = wave_max(m);
    float s = 0.f;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int e = j * 64 + lane;
      s += e < E ? expf(v[j] - m) : 0.f;
      key[j] = e < E ? rank_key(v[j], e) : 0ull;
    }
    s = wave_sum(s);
    ek = wave_topk_keys<NV>(key, lane, K, kk);
    wk = lane < K ? expf(key_value(kk) - m) / s : 0.f;
    if (p.renorm) wk = wk / wave_sum(wk);
    return;
  }
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int e = j * 64 + lane;
    key[j] = e < E ? rank_key(sigmoidf_(logits[e]) + (p.offset ? p.offset[e] : 0.f), e) : 0ull;
  }
  if (p.ngroups > 0) {
    // groups scored by the sum of their K / gtopk best biased scores, gtopk kept
    const int eg = E / p.ngroups, per = K / p.gtopk;
    float gv = -INFINITY;
    for (int q = 0; q < p.ngroups; ++q) {
      uint64_t gk[NV];
#pragma unroll
      for (int j = 0; j < NV; ++j) gk[j] = (j * 64 + lane) / eg == q ? key[j] : 0ull;
      float acc = 0.f;
      uint64_t thr = ~0ull;
      for (int r = 0; r < per; ++r) {
        thr = wave_next_key<NV>(gk, thr);
        acc += key_value(thr);
      }
      gv = lane == q ? acc : gv;
    }
    uint64_t gkey[1] = {lane < p.ngroups ? rank_key(gv, lane) : 0ull};
    uint64_t keep = 0, thr = ~0ull;
    for (int q = 0; q < p.gtopk; ++q) {
      thr = wave_next_key<1>(gkey, thr);
      keep |= 1ull << key_index(thr);
    }
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int e = j * 64 + lane;
      if (e < E && !((keep >> (e / eg)) & 1ull)) key[j] = 0ull;
    }
  }
  ek = wave_topk_keys<NV>(key, lane, K, kk);
  wk = lane < K ? sigmoidf_(logits[ek]) : 0.f;
  float ssum = 0.f;
  if (p.renorm)
    for (int k = 0; k < K; ++k) ssum += __shfl(wk, k, 64);
  wk = dsk_weight(wk, ssum, p.renorm, p.scaling, 0);
}

// The tokens' top-K, one token a wave, four a workgroup; the last workgroup to
// finish lists the active experts and their rows.  With the routing given there
// is one workgroup, which lists.  Every entry counts the entries of its expert
// and those before it by reading all ids from LDS (S <= 1024).
template <int NV>
__global__ __launch_bounds__(64 * kPlanWaves) void few_plan_kernel(FewArgs p) {
  __shared__ __attribute__((aligned(16))) int ids[kFewRows];
  __shared__ int row0_of[kFewRows];
  __shared__ int2 wsum[kPlanWaves];
  __shared__ int box;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wid = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int S = p.T * p.K;
  if (p.wr) {
    const int t = blockIdx.x * kRouteWaves + wid;
    if (wid < kRouteWaves && t < p.T) {
      float wk;
      int ek;
      route_token<NV>(p, p.logits + (int64_t)t * p.E, lane, wk, ek);
      if (lane < p.K) {
        const int s = t * p.K + lane;
        put_shared(&p.real[s], ek);
        p.w[s] = wk;
        if (p.out_w) p.out_w[s] = wk;
        if (p.out_idx) p.out_idx[s] = ek;
      }
    }
    if (gridDim.x > 1) {
      if (!last_to_arrive(&p.hdr[1], gridDim.x, &box)) return;
    } else {
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      __syncthreads();
    }
    if (tid < S) ids[tid] = get_shared(&p.real[tid]);
  } else {
    if (tid < S) {
      const int64_t e = p.ids[tid];
      ids[tid] = e >= 0 && e < p.E ? (int)e : -1;
      p.real[tid] = ids[tid];
      p.w[tid] = p.weights_bf16 ? bf2f(((const bf16*)p.weights)[tid])
                                : ((const float*)p.weights)[tid];
    }
    clear_counters(p);
  }
  for (int i = S + tid; i < kFewRows; i += 64 * kPlanWaves) ids[i] = -1;
  __syncthreads();
  const int e = ids[tid];
  int rank = 0, cnt = 0, first = S;
  for (int i = 0; i < S && wid * 64 < S; i += 4) {
    const int4 q = *(const int4*)&ids[i];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int o = j == 0 ? q.x : j == 1 ? q.y : j == 2 ? q.z : q.w;
      if (o == e) {
        ++cnt;
        rank += i + j < tid;
        first = min(first, i + j);
      }
    }
  }
  const bool lead = e >= 0 && rank == 0;
  // exclusive prefixes over the leaders: their number and their rows
  int2 v = lead ? make_int2(1, cnt) : make_int2(0, 0);
  int2 inc = v;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int a = __shfl_up(inc.x, o, 64), b = __shfl_up(inc.y, o, 64);
    if (lane >= o) {
      inc.x += a;
      inc.y += b;
    }
  }
  if (lane == 63) wsum[wid] = inc;
  __syncthreads();
  int2 base = make_int2(0, 0), all = make_int2(0, 0);
  for (int w = 0; w < kPlanWaves; ++w) {
    if (w == wid) base = all;
    all.x += wsum[w].x;
    all.y += wsum[w].y;
  }
  if (lead) {
    const int at = base.x + inc.x - 1, r0 = base.y + inc.y - cnt;
    p.list[at] = make_int4(e, r0, cnt, 0);
    row0_of[tid] = r0;
  }
  __syncthreads();
  if (e >= 0) p.rows[row0_of[first] + rank] = tid;
  if (tid == 0) p.hdr[0] = all.x;
}

// ------------------------------------------------------- gate/up + SwiGLU
// Workgroup: 16 features of one active expert; the waves split H, CH steps of
// gate and up rows in flight each.  An expert with more than 16 rows reads its
// weights again for the next 16, from L2.
template <typename T, int CH>
__global__ __launch_bounds__(64 * kWaves, 4) void few_gate_up_kernel(FewArgs p) {
  __shared__ f32x4 red[kWaves][2][64];
  const int nsl = p.I / 16;
  const int slot = blockIdx.x / nsl, f0 = (blockIdx.x % nsl) * 16;
  if (slot >= p.hdr[0]) return;
  const int4 info = p.list[slot];
  const int lane = threadIdx.x & 63, n = lane & 15, g = lane >> 4;
  const int wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int ns = p.H / Mma<T>::kStep;
  const int s0 = wid * ns / kWaves, s1 = (wid + 1) * ns / kWaves;
  const int64_t ld = (int64_t)p.H * sizeof(T);
  const char* wg = (const char*)p.w1 + ((int64_t)info.x * 2 * p.I + f0 + n) * ld + g * 16;
  const char* wu = wg + (int64_t)p.I * ld;
  for (int rg = 0; rg < info.z; rg += 16) {
    const int left = info.z - rg;
    const char* xr = (const char*)p.x +
                     (int64_t)(p.rows[info.y + rg + min(n, left - 1)] / p.K) * ld + g * 16;
    f32x4 ag = {0.f, 0.f, 0.f, 0.f}, au = ag;
    for (int sb = s0; sb < s1; sb += CH) {
      u32x4 a[CH], b[CH], c[CH];
#pragma unroll
      for (int i = 0; i < CH; ++i) {
        const int s = min(sb + i, s1 - 1);
        a[i] = ld16_w(wg + s * 64);
        b[i] = ld16_w(wu + s * 64);
      }
#pragma unroll
      for (int i = 0; i < CH; ++i) c[i] = ld16(xr + min(sb + i, s1 - 1) * 64);
#pragma unroll
      for (int i = 0; i < CH; ++i) {
        if (sb + i < s1) {
          ag = Mma<T>::step(a[i], c[i], ag);
          au = Mma<T>::step(b[i], c[i], au);
        }
      }
    }
    if (rg) __syncthreads();
    red[wid][0][lane] = ag;
    red[wid][1][lane] = au;
    __syncthreads();
    if (threadIdx.x < 256) {
      const int f = threadIdx.x & 15, r = threadIdx.x >> 4, l = (f >> 2) * 16 + r;
      if (r < left) {
        float gs = 0.f, us = 0.f;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) {
          gs += red[w][0][l][f & 3];
          us += red[w][1][l][f & 3];
        }
        const int s = p.rows[info.y + rg + r];
        ((T*)p.act)[(int64_t)s * p.I + f0 + f] = (T)(siluf_(gs) * us);
      }
    }
  }
}

// --------------------------------------------------------- down + combine
// Workgroup: 16 columns of the output and kGroup active experts, kParts waves
// an expert.  y rows go to the workspace; the workgroup that finishes a column
// slice's last group sums them with the routing weights, in k order.
template <typename T, int CH>
__global__ __launch_bounds__(64 * kWaves, 4) void few_down_kernel(FewArgs p) {
  __shared__ f32x4 red[kWaves][64];
  __shared__ int box;
  const int nh = p.H / 16;
  const int hs = blockIdx.x % nh, grp = blockIdx.x / nh, h0 = hs * 16;
  const int nact = p.hdr[0];
  const int ngrp = max(1, (nact + kGroup - 1) / kGroup);
  if (grp >= ngrp) return;
  const int tid = threadIdx.x, lane = tid & 63, n = lane & 15, g = lane >> 4;
  const int wid = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int j = wid / kParts, part = wid % kParts;
  int most = 0;
#pragma unroll
  for (int q = 0; q < kGroup; ++q)
    if (grp * kGroup + q < nact) most = max(most, p.list[grp * kGroup + q].z);
  int4 info = make_int4(0, 0, 0, 0);
  if (grp * kGroup + j < nact) info = p.list[grp * kGroup + j];
  const int ns = p.I / Mma<T>::kStep;
  const int s0 = part * ns / kParts, s1 = (part + 1) * ns / kParts;
  const int64_t ld = (int64_t)p.I * sizeof(T);
  const char* wd = (const char*)p.w2 + ((int64_t)info.x * p.H + h0 + n) * ld + g * 16;
  for (int rg = 0; rg < most; rg += 16) {
    const int left = info.z - rg;
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
    if (left > 0) {
      const char* ar =
          (const char*)p.act + (int64_t)p.rows[info.y + rg + min(n, left - 1)] * ld + g * 16;
      for (int sb = s0; sb < s1; sb += CH) {
        u32x4 a[CH], c[CH];
#pragma unroll
        for (int i = 0; i < CH; ++i) a[i] = ld16_w(wd + min(sb + i, s1 - 1) * 64);
#pragma unroll
        for (int i = 0; i < CH; ++i) c[i] = ld16(ar + min(sb + i, s1 - 1) * 64);
#pragma unroll
        for (int i = 0; i < CH; ++i)
          if (sb + i < s1) acc = Mma<T>::step(a[i], c[i], acc);
      }
    }
    if (rg) __syncthreads();
    red[wid][lane] = acc;
    __syncthreads();
    for (int v = tid; v < kGroup * 256; v += 64 * kWaves) {
      const int q = v >> 8, h = v & 15, r = (v >> 4) & 15, l = (h >> 2) * 16 + r;
      if (grp * kGroup + q >= nact) continue;
      const int4 iq = p.list[grp * kGroup + q];
      if (rg + r >= iq.z) continue;
      float sum = 0.f;
#pragma unroll
      for (int w = 0; w < kParts; ++w) sum += red[q * kParts + w][l][h & 3];
      put_shared(&p.y[(int64_t)p.rows[iq.y + rg + r] * p.H + h0 + h], sum);
    }
  }
  // the slice's last group combines
  if (!last_to_arrive(&p.arrived[hs], ngrp, &box)) return;
  const int h = h0 + (tid & 15);
  for (int t = tid >> 4; t < p.T; t += 4 * kWaves) {
    float o = 0.f;
    for (int k = 0; k < p.K; ++k) {
      const int s = t * p.K + k;
      if (p.real[s] >= 0) o = fmaf(p.w[s], get_shared(&p.y[(int64_t)s * p.H + h]), o);
    }
    ((T*)p.out)[(int64_t)t * p.H + h] = (T)o;
  }
}

// ------------------------------------------------------------------- host
struct FewLayout {
  size_t logits, w, hdr, arrived, list, rows, real, act, y, bytes;
};
FewLayout few_layout(int T, int E, int K, int H, int I, int elem) {
  const size_t S = (size_t)T * K;
  FewLayout l{};
  size_t at = 0;
  auto take = [&](size_t n) {
    const size_t o = at;
    at = align_up(at + n, 256);
    return o;
  };
  l.hdr = take(256);
  l.arrived = take((size_t)(H / 16) * 4);
  l.w = take(S * 4);
  l.rows = take(S * 4);
  l.real = take(S * 4);
  l.list = take(S * 16);
  l.logits = take((size_t)T * E * 4);
  l.act = take(S * I * elem);
  l.y = take(S * H * 4);
  l.bytes = at;
  return l;
}

int few_check(int64_t T, int K, int E, int H, int I, int dtype, const char* who) {
  MOE_REQUIRE(dtype == MOE_DTYPE_BF16 || dtype == MOE_DTYPE_F32, MOE_ERR_DTYPE,
              "%s: dtype %d is neither bf16 nor fp32", who, dtype);
  MOE_REQUIRE(T >= 0 && E >= 1 && K >= 1 && H > 0 && I > 0, MOE_ERR_ARG,
              "%s: T=%lld E=%d K=%d H=%d I=%d", who, (long long)T, E, K, H, I);
  MOE_REQUIRE(H % 64 == 0 && I % 64 == 0, MOE_ERR_ARG, "%s: H=%d, I=%d must be multiples of 64",
              who, H, I);
  MOE_REQUIRE(T <= kFewTokens && K <= kFewTopK && E <= kFewExperts && H <= (1 << 16) &&
                  I <= (1 << 16),
              MOE_ERR_UNSUPPORTED,
              "%s: T=%lld K=%d E=%d H=%d I=%d beyond %d tokens, top-%d, %d experts or 65536 "
              "features",
              who, (long long)T, K, E, H, I, kFewTokens, kFewTopK, kFewExperts);
  return MOE_OK;
}

template <typename T>
void few_launch(FewArgs& p, hipStream_t st) {
  const int S = p.T * p.K, slots = S < p.E ? S : p.E;
  if (p.wr) few_logits_kernel<T><<<dim3((p.E + 15) / 16, (p.T + 15) / 16), 64 * kWaves, 0, st>>>(p);
  const int nv = p.wr ? (p.E + 63) / 64 : 1;
  const int nr = p.wr ? (p.T + kRouteWaves - 1) / kRouteWaves : 1;
  if (nv <= 1) few_plan_kernel<1><<<nr, 64 * kPlanWaves, 0, st>>>(p);
  else if (nv <= 2) few_plan_kernel<2><<<nr, 64 * kPlanWaves, 0, st>>>(p);
  else if (nv <= 4) few_plan_kernel<4><<<nr, 64 * kPlanWaves, 0, st>>>(p);
  else if (nv <= 8) few_plan_kernel<8><<<nr, 64 * kPlanWaves, 0, st>>>(p);
  else if (nv <= 16) few_plan_kernel<16><<<nr, 64 * kPlanWaves, 0, st>>>(p);
  else if (nv <= 32) few_plan_kernel<32><<<nr, 64 * kPlanWaves, 0, st>>>(p);
  else few_plan_kernel<64><<<nr, 64 * kPlanWaves, 0, st>>>(p);
  few_gate_up_kernel<T, 8><<<slots * (p.I / 16), 64 * kWaves, 0, st>>>(p);
  few_down_kernel<T, 12>
      <<<(slots + kGroup - 1) / kGroup * (p.H / 16), 64 * kWaves, 0, st>>>(p);
}

int few_run(FewArgs& p, int dtype, void* workspace, size_t workspace_bytes, hipStream_t st,
            const char* who) {
  const FewLayout l = few_layout(p.T, p.E, p.K, p.H, p.I, dtype == MOE_DTYPE_BF16 ? 2 : 4);
  MOE_REQUIRE(workspace && workspace_bytes >= l.bytes, MOE_ERR_WORKSPACE,
              "%s: workspace of %zu bytes, needs %zu", who, workspace_bytes, l.bytes);
  MOE_REQUIRE(al16(p.x) && al16(p.wr) && al16(p.w1) && al16(p.w2) && al16(workspace),
              MOE_ERR_ALIGN, "%s: pointers must be 16-byte aligned", who);
  char* ws = (char*)workspace;
  p.hdr = (int*)(ws + l.hdr);
  p.arrived = (int*)(ws + l.arrived);
  p.w = (float*)(ws + l.w);
  p.rows = (int*)(ws + l.rows);
  p.real = (int*)(ws + l.real);
  p.list = (int4*)(ws + l.list);
  p.logits = (float*)(ws + l.logits);
  p.act = ws + l.act;
  p.y = (float*)(ws + l.y);
  if (dtype == MOE_DTYPE_BF16) few_launch<bf16>(p, st);
  else few_launch<float>(p, st);
  return check_launch(who);
}

}  // namespace
}  // namespace moe

using namespace moe;

extern "C" size_t moe_amd_few_workspace_size(int64_t T, int E, int K, int H, int I, int dtype) {
  if (few_check(T, K, E, H, I, dtype, "few_workspace_size") != MOE_OK) return 0;
  return few_layout((int)T, E, K, H, I, dtype == MOE_DTYPE_BF16 ? 2 : 4).bytes;
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
  MOE_REQUIRE(router == MOE_ROUTER_SOFTMAX || router == MOE_ROUTER_SIGMOID, MOE_ERR_ARG,
              "%s: router %d", who, router);
  MOE_REQUIRE(K <= E, MOE_ERR_ARG, "%s: K=%d outside [1,E=%d]", who, K, E);
  if (num_groups > 0) {
    MOE_REQUIRE(router == MOE_ROUTER_SIGMOID && num_groups <= 64 && E % num_groups == 0 &&
                    group_topk >= 1 && group_topk <= num_groups && K % group_topk == 0 &&
                    (E / num_groups) * group_topk >= K && K / group_topk <= E / num_groups,
                MOE_ERR_ARG, "%s: bad grouping (E=%d K=%d groups=%d group_topk=%d)", who, E, K,
                num_groups, group_topk);
  }
  if (T == 0) return MOE_OK;
  MOE_REQUIRE(hidden_states && router_weight && gate_up_proj && down_proj && out, MOE_ERR_ARG,
              "%s: null pointer", who);
  FewArgs p{};
  p.x = hidden_states;
  p.wr = router_weight;
  p.w1 = gate_up_proj;
  p.w2 = down_proj;
  p.offset = offset_or_bias;
  p.sigmoid = router == MOE_ROUTER_SIGMOID;
  p.renorm = renormalize;
  p.scaling = scaling_factor > 0.f ? scaling_factor : 0.f;
  p.ngroups = num_groups > 0 ? num_groups : 0;
  p.gtopk = group_topk;
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
