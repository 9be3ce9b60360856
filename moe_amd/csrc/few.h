// What the few-token kernels of exact and of 4-bit banks share (gfx950): the
// gating product, the routing and the plan, and the MFMA step of exact operands.
#pragma once
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

// A gate/up workgroup's entry of the list, {expert, first row, rows <= 16}, false
// where there is none.  NV != 0: at most 64 entries, which every workgroup lists
// for itself into `small`; the first one leaves the plan for the down kernel.  NV > 0:
// it routes the tokens too, a wave each, up to 64 NV experts; kGiven: the routing
// is given.
template <int NV>
__device__ __forceinline__ bool gate_up_entry(const FewArgs& p, int slot, int lane, int wid,
                                              SmallPlan& small, int* s_ids, int4& info) {
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
    return info.z != 0;
  } else {
    const int nact = p.hdr[0];
    info = p.list[slot];  // a slot past the active experts holds anything
    return slot < nact;
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

// Entries of the list: an expert's last one may be short, the others are full
// (one token's are its own).
int few_slots(const FewArgs& p) {
  const int S = p.T * p.K;
  return p.T == 1 || S < p.E + S / 16 ? S : p.E + S / 16;
}

// Launches the router and the plan, where they need launches of their own, and
// gate_up(std::integral_constant<int, NV>), NV being gate_up_entry's.
template <typename T, typename F>
void few_route(const FewArgs& p, hipStream_t st, F&& gate_up) {
  const int S = p.T * p.K;
  if (p.wr) few_logits_kernel<T><<<dim3((p.E + 15) / 16, (p.T + 15) / 16), 64 * kWaves, 0, st>>>(p);
  // One wave routes a token of up to 256 experts, a workgroup one of more (with
  // 28 entries a lane, one wave took 46 us for each of 64 tokens, E = 1792).
  const bool wide = p.wr && p.E > 256;
  const auto plan = [&](auto nv) {
    constexpr int NV = decltype(nv)::value;
    // Few entries are listed by the gate/up workgroups themselves, which saves a
    // launch of 4 us; so is the routing of one or two tokens (two: 4 of 38 us),
    // whose instructions every workgroup repeats.
    if (S <= 64 && !p.wr) {
      gate_up(std::integral_constant<int, kGiven>{});
      return;
    }
    if (S <= 64 && p.T <= 2 && !wide) {
      gate_up(nv);
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
    gate_up(std::integral_constant<int, 0>{});
  };
  const int part = wide ? (p.E + kPlanWaves - 1) / kPlanWaves : p.wr ? p.E : 1;
  if (part <= 64) plan(std::integral_constant<int, 1>{});
  else if (part <= 128) plan(std::integral_constant<int, 2>{});
  else plan(std::integral_constant<int, 4>{});
}

void few_bind(FewArgs& p, const FewLayout& l, void* workspace) {
  char* ws = (char*)workspace;
  p.hdr = (int*)(ws + l.hdr);
  p.w = (float*)(ws + l.w);
  p.rows = (int*)(ws + l.rows);
  p.real = (int*)(ws + l.real);
  p.list = (int4*)(ws + l.list);
  p.logits = (float*)(ws + l.logits);
  p.act = ws + l.act;
}

int few_check_router(int router, int K, int E, int num_groups, int group_topk, const char* who) {
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
  return MOE_OK;
}

void few_set_router(FewArgs& p, int router, const float* offset_or_bias, int renormalize,
                    float scaling_factor, int num_groups, int group_topk) {
  p.offset = offset_or_bias;
  p.sigmoid = router == MOE_ROUTER_SIGMOID;
  p.renorm = renormalize;
  p.scaling = scaling_factor > 0.f ? scaling_factor : 0.f;
  p.ngroups = num_groups > 0 ? num_groups : 0;
  p.gtopk = group_topk;
}
}  // namespace
}  // namespace moe
