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
// Blocks in flight of a gate/up wave: two leave room for four workgroups a CU (T = 64,
// E = 128: 218 us; four and two workgroups 228, one 219).
constexpr int kGateUpChunk = 2;

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
  int* hdr;                // [0] entries of the list, [1] finished routing workgroups
  int4* list;              // {expert, first row, rows <= 16, 0} of the active experts
  int* rows;               // flat entries s = t*K + k by active expert, ascending
  void* act;               // [S,I] by flat entry
  int* real;               // [S] the entry's expert, negative for padding
  float* out_w;            // routing out (may be null)
  int64_t* out_idx;
  void* out;
};

// One step of a contraction: 64 bytes of each of 16 rows, lane l holding 16
// bytes of row l % 16 at chunk l / 16; A and B alike, so which k a lane's
// elements are does not matter.
__device__ __forceinline__ f32x4 mma_step(bf16, const u32x4& a, const u32x4& b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a),
                                                 __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mma_step(float, const u32x4& a, const u32x4& b, f32x4 c) {
  const f32x4 fa = __builtin_bit_cast(f32x4, a), fb = __builtin_bit_cast(f32x4, b);
#pragma unroll
  for (int i = 0; i < 4; ++i) c = __builtin_amdgcn_mfma_f32_16x16x4f32(fa[i], fb[i], c, 0, 0, 0);
  return c;
}

// A block of a contraction: 128 bytes, a whole line, of each operand's 16 rows.
// Lane l loads 16 bytes of rows l / 8 and 8 + l / 8, so that 16 lanes of a load
// cover two lines, and the wave turns the block to the MFMA's layout in 4 KB of
// LDS of its own (16-byte chunks XOR-swizzled by row: no bank conflicts).  Loaded
// straight into that layout, 16 lanes touch 16 lines and a CU takes in 38 KB/us
// of both operands together, 1 KB in 64 cycles.
constexpr int kBlock = 128;
constexpr int kBlockLds = 32 * kBlock;  // of a wave
constexpr int kMaxLds = kWaves * kBlockLds + kFewRows * (16 + 64 + 12);  // of the down kernel
struct Block {
  u32x4 a0, a1, b0, b1;
};
template <typename T>
__device__ __forceinline__ f32x4 mma_block(const Block& v, char* lds, int lane, f32x4 acc) {
  const int r = lane >> 3, n = lane & 15, g = lane >> 4;
  char* w = lds + r * kBlock + ((lane & 7) ^ r) * 16;
  *(u32x4*)w = v.a0;
  *(u32x4*)(w + 8 * kBlock) = v.a1;
  *(u32x4*)(w + 16 * kBlock) = v.b0;
  *(u32x4*)(w + 24 * kBlock) = v.b1;
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    const char* q = lds + n * kBlock + ((t * 4 + g) ^ (n & 7)) * 16;
    acc = mma_step(T{}, *(const u32x4*)q, *(const u32x4*)(q + 16 * kBlock), acc);
  }
  __builtin_amdgcn_wave_barrier();  // the next block's writes stay behind these reads
  return acc;
}

// 16 bytes of a row of a wave-uniform base: the lane's part of the address has
// 32 bits and a block's is an immediate, which keeps a chunk of loads short (a
// workgroup of these kernels runs each instruction once or twice, so fetching
// them is part of its time).
__device__ __forceinline__ u32x4 ld16(const char* base, uint32_t lane_off, int imm = 0) {
  return *(const u32x4*)(base + lane_off + imm);
}

// f(chunk length, first block) over the blocks [s, end): chunks of CH, then the
// rest in halves.
template <int CH, typename F>
__device__ __forceinline__ void chunks(int s, int end, F&& f) {
  for (; s + CH <= end; s += CH) f(std::integral_constant<int, CH>{}, s);
  if constexpr (CH > 1) chunks<CH / 2>(s, end, f);
}

template <typename T> __device__ __forceinline__ float few_round(float v) {
  if constexpr (sizeof(T) == 2) return round_bf(v);
  return v;
}

// What one workgroup leaves for another of the same launch: written through to
// and read from the memory that all XCDs share, so that no cache has to be
// written back or invalidated.  A workgroup counts itself as arrived once its
// writes are there; the last one to arrive reads everybody's.
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
// clears the counter that the routing workgroups finish by.
template <typename T>
__global__ __launch_bounds__(64 * kWaves) void few_logits_kernel(FewArgs p) {
  __shared__ __attribute__((aligned(16))) char turn[kWaves][kBlockLds];
  __shared__ f32x4 red[kWaves][64];
  const int lane = threadIdx.x & 63, r = lane >> 3;
  const int wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int e0 = blockIdx.x * 16, t0 = blockIdx.y * 16;
  const int nb = p.H * (int)sizeof(T) / kBlock;
  const uint32_t ld = (uint32_t)p.H * sizeof(T), j = (lane & 7) * 16;
  const uint32_t a0 = min(r, p.E - 1 - e0) * ld + j, a1 = min(r + 8, p.E - 1 - e0) * ld + j;
  const uint32_t b0 = min(t0 + r, p.T - 1) * ld + j, b1 = min(t0 + r + 8, p.T - 1) * ld + j;
  const char* a = (const char*)p.wr + (int64_t)e0 * ld;
  f32x4 acc = {0.f, 0.f, 0.f, 0.f};
  chunks<4>(wid * nb / kWaves, (wid + 1) * nb / kWaves, [&](auto ch, int s) {
    constexpr int C = decltype(ch)::value;
    const char *as = a + s * kBlock, *bs = (const char*)p.x + s * kBlock;
    Block v[C];
#pragma unroll
    for (int i = 0; i < C; ++i) {
      v[i].a0 = ld16(as, a0, i * kBlock);
      v[i].a1 = ld16(as, a1, i * kBlock);
      v[i].b0 = ld16(bs, b0, i * kBlock);
      v[i].b1 = ld16(bs, b1, i * kBlock);
    }
#pragma unroll
    for (int i = 0; i < C; ++i) acc = mma_block<T>(v[i], turn[wid], lane, acc);
  });
  red[wid][lane] = acc;
  if (blockIdx.x == 0 && blockIdx.y == 0 && threadIdx.x == 0) p.hdr[1] = 0;
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
// The order of wave_topk.h's rank_key in 32 bits, by value alone; 0 is below
// every value.
__device__ __forceinline__ uint32_t value_key(float v) { return (uint32_t)(rank_key(v, 0) >> 32); }
__device__ __forceinline__ float value_of(uint32_t key) {
  return key_value((uint64_t)key << 32);
}

// The waves that route one token: one, which holds entry j*64 + lane of its
// experts in slot j, or (BLOCK) all of a workgroup's kPlanWaves, wave w holding
// the experts from w * chunk on.  They share the largest keys of their parts
// through LDS, in two places by turns, so that a round needs one barrier.
struct RouteShared {
  uint32_t key[2][kPlanWaves];
  float part[2][kPlanWaves];
  int entry[64];
};
template <int NV, bool BLOCK>
struct Router {
  RouteShared* sh;
  int lane, wid, base, count, turn = 0;

  __device__ __forceinline__ Router(RouteShared* sh_, int E, int wid_, int lane_)
      : sh(sh_), lane(lane_), wid(wid_) {
    const int chunk = BLOCK ? (E + kPlanWaves - 1) / kPlanWaves : E;
    base = BLOCK ? wid * chunk : 0;
    count = min(chunk, E - base);  // none, or fewer, of a last wave's
  }
  __device__ __forceinline__ bool has(int j) const { return j * 64 + lane < count; }
  __device__ __forceinline__ int expert(int j) const { return base + j * 64 + lane; }

  // Over all entries: whether any, maximum, sum.
  __device__ __forceinline__ bool any(bool v) {
    if constexpr (BLOCK) return all_max(v ? 1.f : 0.f) > 0.f;
    return __ballot(v) != 0;
  }
  __device__ __forceinline__ float all_max(float v) {
    v = group_max<16>(v);
    v = fmaxf(fmaxf(lane_of(v, 0), lane_of(v, 16)), fmaxf(lane_of(v, 32), lane_of(v, 48)));
    if constexpr (BLOCK) v = group_max<16>(exchange(v));
    return v;
  }
  __device__ __forceinline__ float all_sum(float v) {
    v = group_sum<16>(v);
    v = (lane_of(v, 0) + lane_of(v, 16)) + (lane_of(v, 32) + lane_of(v, 48));
    if constexpr (BLOCK) v = group_sum<16>(exchange(v));
    return v;
  }
  static __device__ __forceinline__ float lane_of(float v, int l) {
    return __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(v), l));
  }
  __device__ __forceinline__ float exchange(float v) {  // wave (lane % 16)'s v
    float* at = sh->part[turn ^= 1];
    if (lane == 0) at[wid] = v;
    __syncthreads();
    return at[lane & 15];
  }

  // Takes the largest key out and returns it: the value by DPP, its holder (of
  // equal ones the lowest expert) by ballots.  (64-bit keys that hold the index
  // too need four times the instructions.)  `entry`, in its holder's wave alone
  // where BLOCK: the expert, else negative.
  __device__ __forceinline__ uint32_t take(uint32_t (&key)[NV], int& entry) {
    uint32_t m = key[0];
#pragma unroll
    for (int j = 1; j < NV; ++j) m = max(m, key[j]);
    m = group_max_key<16>(m);
    m = max(max((uint32_t)__builtin_amdgcn_readlane(m, 0),
                (uint32_t)__builtin_amdgcn_readlane(m, 16)),
            max((uint32_t)__builtin_amdgcn_readlane(m, 32),
                (uint32_t)__builtin_amdgcn_readlane(m, 48)));
    entry = -1;
    if constexpr (BLOCK) {
      uint32_t* at = sh->key[turn ^= 1];
      if (lane == 0) at[wid] = m;
      __syncthreads();
      const uint32_t other = at[lane & 15];
      m = __builtin_amdgcn_readfirstlane(group_max_key<16>(other));
      if (__builtin_ctzll(__ballot(other == m)) != wid) return m;
    }
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const uint64_t here = __ballot(key[j] == m);
      if (entry < 0 && here) {
        const int l = __builtin_ctzll(here);
        entry = base + j * 64 + l;
        if (lane == l) key[j] = 0;
      }
    }
    return m;
  }
};

// One token: lane k < K gets its k-th expert and weight (of every wave that
// routes it).  The selections and the arithmetic are those of the router
// kernels.
template <int NV, bool BLOCK>
__device__ __forceinline__ void route_token(const FewArgs& p, const float* logits,
                                            RouteShared* sh, int wid, int lane, float& wk,
                                            int& ek) {
  const int E = p.E, K = p.K;
  Router<NV, BLOCK> r(sh, E, wid, lane);
  uint32_t key[NV];
  float m = 0.f, s = 0.f;
  if (!p.sigmoid) {
    float v[NV];
    bool nan_here = false;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      v[j] = r.has(j) ? logits[r.expert(j)] + (p.offset ? p.offset[r.expert(j)] : 0.f) : -INFINITY;
      nan_here |= v[j] != v[j];
    }
    if (r.any(nan_here)) {  // every prob of the row is NaN: they rank by index
#pragma unroll
      for (int j = 0; j < NV; ++j)
        if (r.has(j)) v[j] = __builtin_nanf("");
    }
    m = -INFINITY;
#pragma unroll
    for (int j = 0; j < NV; ++j) m = fmaxf(m, v[j]);
    m = r.all_max(m);
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      s += r.has(j) ? expf(v[j] - m) : 0.f;
      key[j] = r.has(j) ? value_key(v[j]) : 0u;
    }
    s = r.all_sum(s);
  } else {
#pragma unroll
    for (int j = 0; j < NV; ++j)
      key[j] = r.has(j) ? value_key(sigmoidf_(logits[r.expert(j)]) +
                                    (p.offset ? p.offset[r.expert(j)] : 0.f))
                        : 0u;
  }
  if (p.ngroups > 0) {
    // groups scored by the sum of their K / gtopk best biased scores, gtopk kept
    const int eg = E / p.ngroups, per = K / p.gtopk;
    float gv = -INFINITY;
    for (int q = 0; q < p.ngroups; ++q) {
      uint32_t gk[NV];
#pragma unroll
      for (int j = 0; j < NV; ++j) gk[j] = r.expert(j) / eg == q ? key[j] : 0u;
      float acc = 0.f;
      int e;
      for (int i = 0; i < per; ++i) acc += value_of(r.take(gk, e));
      gv = lane == q ? acc : gv;
    }
    uint32_t gkey[1] = {lane < p.ngroups ? value_key(gv) : 0u};
    Router<1, false> groups(sh, 64, 0, lane);  // every wave for itself
    uint64_t keep = 0;
    for (int q = 0; q < p.gtopk; ++q) {
      int e;
      groups.take(gkey, e);
      keep |= 1ull << e;
    }
#pragma unroll
    for (int j = 0; j < NV; ++j)
      if (r.has(j) && !((keep >> (r.expert(j) / eg)) & 1ull)) key[j] = 0u;
  }
  uint32_t kk = 0;
  ek = 0;
  for (int k = 0; k < K; ++k) {
    int e;
    const uint32_t top = r.take(key, e);
    kk = lane == k ? top : kk;
    if constexpr (BLOCK) {
      if (e >= 0 && lane == 0) sh->entry[k] = e;
    } else {
      ek = lane == k ? e : ek;
    }
  }
  if constexpr (BLOCK) {
    __syncthreads();
    ek = lane < K ? sh->entry[lane] : 0;
  }
  if (!p.sigmoid) {
    wk = lane < K ? expf(value_of(kk) - m) / s : 0.f;
    if (p.renorm) wk = wk / group_sum<16>(wk);  // K <= 16: the other rows of lanes divide by 0
  } else {
    wk = lane < K ? sigmoidf_(logits[ek]) : 0.f;
    float ssum = 0.f;
    if (p.renorm)
      for (int k = 0; k < K; ++k) ssum += __shfl(wk, k, 64);
    wk = dsk_weight(wk, ssum, p.renorm, p.scaling, 0);
  }
}

// Leaves token t's routing, held by lanes 0 .. K-1, for later launches.
__device__ __forceinline__ void store_route(const FewArgs& p, int t, int lane, float wk, int ek) {
  if (lane >= p.K) return;
  const int s = t * p.K + lane;
  put_shared(&p.real[s], ek);
  p.w[s] = wk;
  if (p.out_w) p.out_w[s] = wk;
  if (p.out_idx) p.out_idx[s] = ek;
}

// Entry s of a given routing: its expert, negative for padding, and weight.
__device__ __forceinline__ int given_route(const FewArgs& p, int s, float& w) {
  const int64_t id = p.ids[s];
  w = p.weights_bf16 ? bf2f(((const bf16*)p.weights)[s]) : ((const float*)p.weights)[s];
  return id >= 0 && id < p.E ? (int)id : -1;
}

// The tokens' top-K, one token a wave or (BLOCK) a workgroup; the last
// workgroup to finish lists the active experts and their rows, at most 16 (an
// MFMA's columns) an entry: an expert with more has several entries, which run
// side by side and find its weights in L2.  (One after the other in a workgroup:
// 61 us for 64 rows in each of 4 experts, H = 2048, I = 768.)  With the routing
// given there is one workgroup, which lists.  Places in the list and
// among an expert's rows are taken with LDS atomics: their order may differ
// from call to call, which no result depends on (rows are computed apart, and
// combined by their number).
template <int NV, bool BLOCK>
__global__ __launch_bounds__(64 * kPlanWaves) void few_plan_kernel(FewArgs p) {
  __shared__ RouteShared sh;
  __shared__ int count[kFewExperts];   // rows of an expert, then its first row
  __shared__ int ids[kFewRows];
  __shared__ int total, box;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wid = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int S = p.T * p.K;
  for (int i = tid; i < p.E; i += blockDim.x) count[i] = 0;
  if (tid == 0) total = 0;
  int e = -1;
  if (p.wr) {
    const int t = BLOCK ? blockIdx.x : blockIdx.x * kPlanWaves + wid;
    const bool one = gridDim.x == 1;
    if (t < p.T) {  // uniform over the workgroup where BLOCK
      float wk;
      int ek;
      route_token<NV, BLOCK>(p, p.logits + (int64_t)t * p.E, &sh, wid, lane, wk, ek);
      if (!BLOCK || wid == 0) {
        store_route(p, t, lane, wk, ek);
        if (one && lane < p.K) ids[t * p.K + lane] = ek;
      }
    }
    if (!one && !last_to_arrive(&p.hdr[1], gridDim.x, &box)) return;
    __syncthreads();
    if (tid < S) e = one ? ids[tid] : get_shared(&p.real[tid]);
  } else {
    if (tid < S) {
      float w;
      e = given_route(p, tid, w);
      p.real[tid] = e;
      p.w[tid] = w;
    }
    __syncthreads();
  }
  const int rank = e >= 0 ? atomicAdd(&count[e], 1) : 0;
  __syncthreads();
  const bool lead = e >= 0 && rank == 0;
  const int cnt = lead ? count[e] : 0, n = (cnt + 15) / 16;
  // entries (high half) and rows before it: the wave's by a scan, one atomic a
  // wave for the others' (with one a leader, all of the same word, this kernel took
  // 9.8 us for 64 tokens and 128 experts and 13.7 for 1792, with the scan 8.5 and 11.4)
  const int own = n << 16 | cnt;
  int upto = own;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int v = __shfl_up(upto, o, 64);
    if (lane >= o) upto += v;
  }
  int at = 0;
  if (lane == 63) at = atomicAdd(&total, upto);
  at = __builtin_amdgcn_readlane(at, 63) + upto - own;
  if (lead) {  // the one that reads or writes count[e] until the next barrier
    const int r0 = at & 0xffff;
    for (int i = 0; i < n; ++i)
      p.list[(at >> 16) + i] = make_int4(e, r0 + 16 * i, min(16, cnt - 16 * i), 0);
    count[e] = r0;
  }
  __syncthreads();
  if (e >= 0) p.rows[count[e] + rank] = tid;
  if (tid == 0) p.hdr[0] = total >> 16;
}

// ------------------------------------------------------- gate/up + SwiGLU
// Workgroup: 8 features of one entry of the list, their gate and up rows being
// the 16 rows of the A operand; the waves split H, CH blocks in flight each.  A
// CU takes in about 24 KB/us whatever else is idle, so the weights are dealt to
// all of them in small pieces: with 16 features a workgroup one token (K = 8,
// I = 768) has 384 for 256 CUs.
// NV != 0: at most 64 entries, which every workgroup lists for itself; the first
// one leaves the plan for the down kernel.  NV > 0: it routes the tokens too, a
// wave each, up to 64 NV experts; kGiven: the routing is given.
constexpr int kGiven = -1;

// The list and rows of few_plan_kernel from up to 64 entries on one wave, lane s
// holding entry s's expert (negative: padding): `slot`'s expert and rows (n = 0:
// no such entry), and the whole plan where `leave`.
struct SmallPlan {
  int e, n;
  int row[16];
};
__device__ __forceinline__ void small_plan(const FewArgs& p, int e, int lane, int slot, bool leave,
                                           SmallPlan* out) {
  const uint64_t before = (1ull << lane) - 1;
  if (p.T == 1) {
    // slot k is entry k, padding included; an expert named twice is read twice
    // (the general form costs one token 0.7 of 24 us)
    const int expert = __builtin_amdgcn_readlane(e, slot);
    if (lane == 0) {
      out->e = expert;
      out->n = expert >= 0;
      out->row[0] = slot;
    }
    if (!leave) return;
    const uint64_t real = __ballot(e >= 0);
    if (e >= 0) p.list[__popcll(real & before)] = make_int4(e, lane, 1, 0);
    if (lane < p.K) p.rows[lane] = lane;
    if (lane == 0) p.hdr[0] = __popcll(real);
    return;
  }
  uint64_t peers = __ballot(e >= 0);  // entries of the same expert
#pragma unroll
  for (int b = 0; b < 12; ++b) {
    const uint64_t one = __ballot(e >> b & 1);
    peers &= e >> b & 1 ? one : ~one;
  }
  static_assert(kFewExperts <= 1 << 12, "a ballot for each bit of an id");
  const int rank = __popcll(peers & before);
  const bool lead = e >= 0 && (rank & 15) == 0;  // begins a list entry
  const uint64_t leads = __ballot(lead);
  const int at = __popcll(leads & before);
  const uint64_t mine = __ballot(lead && at == slot);
  if (mine) {
    const int l = __builtin_ctzll(mine);
    const bool member = e >= 0 && peers == readlane_u64(peers, l) &&
                        rank >> 4 == __builtin_amdgcn_readlane(rank, l) >> 4;
    if (member) out->row[rank & 15] = lane;
    const int n = __popcll(__ballot(member)), expert = __builtin_amdgcn_readlane(e, l);
    if (lane == 0) {
      out->e = expert;
      out->n = n;
    }
  } else if (lane == 0) {
    out->n = 0;
  }
  if (!leave) return;
  const int count = e >= 0 && rank == 0 ? __popcll(peers) : 0;
  int upto = count;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int v = __shfl_up(upto, o, 64);
    if (lane >= o) upto += v;
  }
  const int row0 = __shfl(upto - count, e >= 0 ? __builtin_ctzll(peers) : 0, 64);
  if (e >= 0) p.rows[row0 + rank] = lane;
  if (lead) p.list[at] = make_int4(e, row0 + rank, min(16, __popcll(peers) - rank), 0);
  if (lane == 0) p.hdr[0] = __popcll(leads);
}

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
  if constexpr (NV != 0) {
    const bool first = blockIdx.x == 0;
    if constexpr (NV > 0) {
      if (wid < p.T) {
        float wk;
        int ek;
        route_token<NV, false>(p, p.logits + (int64_t)wid * p.E, nullptr, 0, lane, wk, ek);
        if (lane < p.K) s_ids[wid * p.K + lane] = ek;
        if (first) store_route(p, wid, lane, wk, ek);
      }
      if (p.T > 1) __syncthreads();
    }
    if (wid == 0) {
      const int S = p.T * p.K;
      int e = -1;
      if constexpr (NV > 0) {
        if (lane < S) e = s_ids[lane];
      } else if (lane < S) {
        float wk;
        e = given_route(p, lane, wk);
        if (first) {
          p.real[lane] = e;
          p.w[lane] = wk;
        }
      }
      small_plan(p, e, lane, slot, first, &small);
    }
    __syncthreads();
    info = make_int4(__builtin_amdgcn_readfirstlane(small.e), 0,
                     __builtin_amdgcn_readfirstlane(small.n), 0);
    if (info.z == 0) return;
  } else {
    const int nact = p.hdr[0];
    info = p.list[slot];  // a slot past the active experts holds anything
    if (slot >= nact) return;
  }
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
struct FewLayout {
  size_t logits, w, hdr, list, rows, real, act, bytes;
};
FewLayout few_layout(int T, int E, int K, int I, int elem) {
  const size_t S = (size_t)T * K;
  FewLayout l{};
  size_t at = 0;
  auto take = [&](size_t n) {
    const size_t o = at;
    at = align_up(at + n, 256);
    return o;
  };
  l.hdr = take(256);
  l.w = take(S * 4);
  l.rows = take(S * 4);
  l.real = take(S * 4);
  l.list = take(S * 16);
  l.logits = take((size_t)T * E * 4);
  l.act = take(S * I * elem);
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
hipError_t few_launch(const FewArgs& p, hipStream_t st) {
  // entries of the list: an expert's last one may be short, the others are full
  // (one token's are its own)
  const int S = p.T * p.K, slots = p.T == 1 || S < p.E + S / 16 ? S : p.E + S / 16;
  if (p.wr) few_logits_kernel<T><<<dim3((p.E + 15) / 16, (p.T + 15) / 16), 64 * kWaves, 0, st>>>(p);
  // One wave routes a token of up to 256 experts, a workgroup one of more (with
  // 28 entries a lane, one wave took 46 us for each of 64 tokens, E = 1792).
  const bool wide = p.wr && p.E > 256;
  const int threads = 64 * kWaves, gu_grid = slots * (p.I / 8);
  const auto plan = [&](auto nv) {
    constexpr int NV = decltype(nv)::value;
    // Few entries are listed by the gate/up workgroups themselves, which saves a
    // launch of 4 us; so is the routing of one or two tokens (two: 4 of 38 us),
    // whose instructions every workgroup repeats.
    if (S <= 64 && !p.wr) {
      few_gate_up_kernel<T, kGateUpChunk, kGiven><<<gu_grid, threads, 0, st>>>(p);
      return;
    }
    if (S <= 64 && p.T <= 2 && !wide) {
      few_gate_up_kernel<T, kGateUpChunk, NV><<<gu_grid, threads, 0, st>>>(p);
      return;
    }
    if (wide) {
      few_plan_kernel<NV, true><<<p.T, 64 * kPlanWaves, 0, st>>>(p);
    } else {
      // a wave for every 64 entries, and for each of the tokens that it routes
      const int nr = p.wr ? (p.T + kPlanWaves - 1) / kPlanWaves : 1;
      const int tokens = p.wr ? (p.T < kPlanWaves ? p.T : kPlanWaves) : 1;
      const int entries = (S + 63) / 64;
      few_plan_kernel<NV, false><<<nr, 64 * (tokens > entries ? tokens : entries), 0, st>>>(p);
    }
    few_gate_up_kernel<T, kGateUpChunk, 0><<<gu_grid, threads, 0, st>>>(p);
  };
  const int part = wide ? (p.E + kPlanWaves - 1) / kPlanWaves : p.wr ? p.E : 1;
  if (part <= 64) plan(std::integral_constant<int, 1>{});
  else if (part <= 128) plan(std::integral_constant<int, 2>{});
  else plan(std::integral_constant<int, 4>{});
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
  char* ws = (char*)workspace;
  p.hdr = (int*)(ws + l.hdr);
  p.w = (float*)(ws + l.w);
  p.rows = (int*)(ws + l.rows);
  p.real = (int*)(ws + l.real);
  p.list = (int4*)(ws + l.list);
  p.logits = (float*)(ws + l.logits);
  p.act = ws + l.act;
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
