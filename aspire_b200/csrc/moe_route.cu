// Router top-k and the sort of the tokens by expert.
//
// One warp per token, two tokens at a time (a round's latency is that of two
// warp reductions, and the second token's fill it).  Lane l holds the logits of
// experts l, l + 32, ... as order-preserving integers, sorted; each of the
// top_k rounds takes the maximum of the lanes' heads and, among equals, the
// lowest expert index.  A NaN or -inf logit is
// never chosen: a token with fewer than top_k others gets expert -1 and
// weight 0 for the rest.  The weights are the softmax over all experts at the
// chosen ones or, renormalised, the softmax over the chosen ones.
//
// The sort counts: within a block of slots each warp ranks its 32 slots among
// those of the same expert (a warp match), per-warp counts are summed over
// the block's warps and the earlier blocks' counts, so the order is stable
// and no atomic decides it.  A cluster of up to 8 blocks routes a decode step
// and sorts it in the same launch, its counts exchanged in distributed shared
// memory; more than 8 x 1024 slots take a second launch after every block's
// counts are known.  Both are bound by latency, as the bytes are a few megabytes
// at most: 72 tokens over 128 experts 5.5 us (9.9 in one block), 8192 tokens
// 18 us.
#include <cooperative_groups.h>

#include "moe.cuh"

namespace aspire {

namespace {

namespace cg = cooperative_groups;

__device__ __forceinline__ float load_logit(const void* p, int32_t type, int64_t i) {
  if (type == ASPIRE_T_F32) return static_cast<const float*>(p)[i];
  if (type == ASPIRE_T_BF16) return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
  return __half2float(static_cast<const __half*>(p)[i]);
}

// Integers in the order of the floats (-0 just below 0; equal floats compare
// equal after adding 0, which turns -0 into 0).  0 stands for "never chosen".
__device__ __forceinline__ uint32_t order_of(float v) {
  if (!(v > -INFINITY)) return 0u;  // NaN, -inf
  const uint32_t b = __float_as_uint(v + 0.0f);
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ float value_of(uint32_t o) {
  return __uint_as_float((o & 0x80000000u) ? (o & 0x7FFFFFFFu) : ~o);
}
// exp(v - m) with m the row's maximum; two infinities count as equal.
__device__ __forceinline__ float exp_below(float v, float m) { return v == m ? 1.0f : expf(v - m); }

struct SortShared {
  uint16_t count[32][kMoeMaxExperts];  // per warp: slots of the expert, then the warps before it
  int32_t base[kMoeMaxExperts];        // the block's first row of the expert
  int32_t part[2][kMoeSlotsBlock];     // several blocks: sums of a share of their counts (all, earlier)
  int32_t scan[32];
  int16_t ids[kMoeSlotsOne];           // the block's choices
};

// Sorts the block's slots (thread = slot, expert id or -1).
// ONE: the blocks are one cluster; otherwise their counts are in p.counts.
template <bool ONE>
__device__ void sort_block(const MoeRouteParams& p, SortShared& sh, int32_t id, int64_t slot, bool live) {
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int warps = blockDim.x >> 5, E = p.num_experts;
  for (int w = warp; w < 32; w += warps)  // (all 32: the sums below are unrolled)
    for (int e = lane; e < E; e += 32) sh.count[w][e] = 0;
  if constexpr (!ONE) {
    // The blocks' counts, a share of the blocks for every blockDim / E threads.
    const int shares = blockDim.x / E, share = tid / E, e = tid - share * E;
    int32_t all = 0, earlier = 0;
    if (share < shares) {
      const int blocks = gridDim.x, self = blockIdx.x;
#pragma unroll 8
      for (int b = share; b < blocks; b += shares) {
        const int32_t n = p.counts[int64_t(b) * E + e];
        all += n;
        earlier += b < self ? n : 0;
      }
    }
    sh.part[0][tid] = all;
    sh.part[1][tid] = earlier;
  }
  __syncthreads();
  const unsigned peers = __match_any_sync(0xffffffffu, id);
  const int rank = __popc(peers & ((1u << lane) - 1));
  if (id >= 0 && rank == 0) sh.count[warp][id] = uint16_t(__popc(peers));
  __syncthreads();
  // Thread e: the warps' counts become offsets within the block; then the
  // experts' totals are scanned over all threads (E <= blockDim).
  int32_t total = 0, earlier = 0;
  if (tid < E) {
    uint16_t n[32];
#pragma unroll
    for (int w = 0; w < 32; ++w) n[w] = sh.count[w][tid];
#pragma unroll
    for (int w = 0; w < 32; ++w) {
      sh.count[w][tid] = uint16_t(total);
      total += n[w];
    }
    if constexpr (ONE) {
      sh.base[tid] = total;
    } else {
      total = 0;
      for (int i = tid; i < int(blockDim.x) / E * E; i += E) {
        total += sh.part[0][i];
        earlier += sh.part[1][i];
      }
    }
  }
  if constexpr (ONE) {
    const int blocks = gridDim.x;
    if (blocks > 1) {
      cg::cluster_group cluster = cg::this_cluster();
      cluster.sync();
      int32_t n[kMoeCluster] = {};
      if (tid < E) {
#pragma unroll
        for (int b = 0; b < kMoeCluster; ++b)
          if (b < blocks) n[b] = cluster.map_shared_rank(sh.base, b)[tid];
      }
      cluster.sync();  // before the totals make way for the bases
      total = 0;
#pragma unroll
      for (int b = 0; b < kMoeCluster; ++b) {
        total += n[b];
        earlier += b < int(blockIdx.x) ? n[b] : 0;
      }
    }
  }
  int32_t incl = total;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int32_t v = __shfl_up_sync(0xffffffffu, incl, d);
    if (lane >= d) incl += v;
  }
  if (lane == 31) sh.scan[warp] = incl;
  __syncthreads();
  // Every warp scans the warps' sums.
  const int32_t mine = lane < warps ? sh.scan[lane] : 0;
  int32_t sums = mine;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int32_t v = __shfl_up_sync(0xffffffffu, sums, d);
    if (lane >= d) sums += v;
  }
  const int32_t all = __shfl_sync(0xffffffffu, sums, 31);
  const int32_t before = __shfl_sync(0xffffffffu, sums - mine, warp);
  if (tid < E) {
    sh.base[tid] = before + incl - total + earlier;
    if (blockIdx.x == 0) {
      p.offsets[tid + 1] = before + incl;
      if (tid == 0) p.offsets[0] = 0;
    }
  }
  __syncthreads();
  if (live) {
    int32_t pos = -1;
    if (id >= 0) {
      pos = sh.base[id] + sh.count[warp][id] + rank;
      p.source[pos] = int32_t(slot);
    }
    p.position[slot] = pos;
    if (slot >= all) p.source[slot] = -1;  // rows past the last expert's
  }
}

// Routes N tokens (token + i * step, those below `end`) with the calling warp.
// The choices also go to `ids` (the block's, from its first token on).
template <int EPL, int N>
__device__ __forceinline__ void route_tokens(const MoeRouteParams& p, int64_t token, int64_t step, int64_t end,
                                             int lane, int16_t* ids, int64_t first) {
  uint32_t o[N][EPL];  // sorted, largest first; equal ones by expert
  uint8_t at[N][EPL];  // expert = lane + 32 at
#pragma unroll
  for (int n = 0; n < N; ++n)
#pragma unroll
    for (int i = 0; i < EPL; ++i) {
      const int e = lane + 32 * i;
      at[n][i] = uint8_t(i);
      o[n][i] = 0u;
      if (token + n * step < end && e < p.num_experts)
        o[n][i] = order_of(load_logit(p.logits, p.logits_type, (token + n * step) * p.logits_stride + e));
    }
  float all[N];  // softmax denominator over all experts
  uint32_t top[N];
#pragma unroll
  for (int n = 0; n < N; ++n) {
    all[n] = 0.f;
    uint32_t best = 0;
#pragma unroll
    for (int i = 0; i < EPL; ++i) best = max(best, o[n][i]);
    top[n] = __reduce_max_sync(0xffffffffu, best);
    if (!p.renormalize && top[n] != 0) {
      const float mv = value_of(top[n]);
#pragma unroll
      for (int i = 0; i < EPL; ++i)
        if (o[n][i] != 0) all[n] += exp_below(value_of(o[n][i]), mv);
#pragma unroll
      for (int d = 16; d > 0; d >>= 1) all[n] += __shfl_xor_sync(0xffffffffu, all[n], d);
    }
    // Insertion sort; strict comparisons keep equal ones in order.
#pragma unroll
    for (int i = 1; i < EPL; ++i)
#pragma unroll
      for (int j = i; j > 0; --j)
        if (o[n][j] > o[n][j - 1]) {
          const uint32_t t = o[n][j];
          o[n][j] = o[n][j - 1];
          o[n][j - 1] = t;
          const uint8_t u = at[n][j];
          at[n][j] = at[n][j - 1];
          at[n][j - 1] = u;
        }
  }
  uint32_t mine_o[N];
  int32_t mine_e[N];  // lane j keeps choice j
#pragma unroll
  for (int n = 0; n < N; ++n) {
    mine_o[n] = 0;
    mine_e[n] = -1;
  }
  for (int j = 0; j < p.top_k; ++j) {
#pragma unroll
    for (int n = 0; n < N; ++n) {
      const uint32_t m = __reduce_max_sync(0xffffffffu, o[n][0]);
      const uint32_t own = o[n][0] == m ? uint32_t(lane) + 32u * at[n][0] : 0xffffffffu;
      const uint32_t e = __reduce_min_sync(0xffffffffu, own);
      if (lane == j && m != 0) {  // 0: nothing left to choose
        mine_o[n] = m;
        mine_e[n] = int32_t(e);
      }
      if (own == e) {
#pragma unroll
        for (int i = 0; i + 1 < EPL; ++i) {
          o[n][i] = o[n][i + 1];
          at[n][i] = at[n][i + 1];
        }
        o[n][EPL - 1] = 0;
      }
    }
  }
#pragma unroll
  for (int n = 0; n < N; ++n) {
    float w = mine_e[n] >= 0 ? exp_below(value_of(mine_o[n]), value_of(top[n])) : 0.f;
    if (p.renormalize) {
      all[n] = w;
#pragma unroll
      for (int d = 16; d > 0; d >>= 1) all[n] += __shfl_xor_sync(0xffffffffu, all[n], d);
    }
    const int64_t t = token + n * step;
    if (t < end && lane < p.top_k) {
      p.weights[t * p.top_k + lane] = mine_e[n] >= 0 ? w / all[n] : 0.f;
      p.experts[t * p.top_k + lane] = mine_e[n];
      ids[(t - first) * p.top_k + lane] = int16_t(mine_e[n]);
    }
  }
}

// EPL: experts per lane; 0: the experts are given.
template <int EPL>
__global__ void __launch_bounds__(kMoeSlotsOne) aspire_moe_route_kernel(MoeRouteParams p) {
  pdl_begin();
  __shared__ SortShared sh;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int64_t t0 = int64_t(blockIdx.x) * p.block_tokens;
  const int nt = int(min(int64_t(p.block_tokens), p.tokens - t0));
  if constexpr (EPL > 0) {
    const int warps = blockDim.x >> 5;
    constexpr int N = EPL <= 4 ? 2 : 1;
    for (int t = warp; t < nt; t += N * warps) route_tokens<EPL, N>(p, t0 + t, warps, t0 + nt, lane, sh.ids, t0);
    __syncthreads();
  }
  const bool live = tid < nt * p.top_k;
  const int64_t slot = t0 * p.top_k + tid;
  int32_t id = live ? (EPL > 0 ? int32_t(sh.ids[tid]) : p.experts[slot]) : -1;
  if (id >= p.num_experts || id < 0) id = -1;
  if (p.counts == nullptr) {
    sort_block<true>(p, sh, id, slot, live);
    return;
  }
  int32_t* count = sh.base;
  for (int e = tid; e < p.num_experts; e += blockDim.x) count[e] = 0;
  __syncthreads();
  const unsigned peers = __match_any_sync(0xffffffffu, id);
  if (id >= 0 && (peers & ((1u << lane) - 1)) == 0) atomicAdd(count + id, __popc(peers));
  __syncthreads();
  for (int e = tid; e < p.num_experts; e += blockDim.x) p.counts[int64_t(blockIdx.x) * p.num_experts + e] = count[e];
}

}  // namespace

__global__ void __launch_bounds__(kMoeSlotsBlock) aspire_moe_sort_kernel(MoeRouteParams p) {
  pdl_begin();
  __shared__ SortShared sh;
  const int64_t t0 = int64_t(blockIdx.x) * p.block_tokens;
  const int nt = int(min(int64_t(p.block_tokens), p.tokens - t0));
  const bool live = int(threadIdx.x) < nt * p.top_k;
  const int64_t slot = t0 * p.top_k + threadIdx.x;
  int32_t id = live ? p.experts[slot] : -1;
  if (id >= p.num_experts || id < 0) id = -1;
  sort_block<false>(p, sh, id, slot, live);
}

MoeRouteKernel moe_route_kernel(int32_t num_experts) {
  if (num_experts <= 0) return aspire_moe_route_kernel<0>;
  if (num_experts <= 32) return aspire_moe_route_kernel<1>;
  if (num_experts <= 64) return aspire_moe_route_kernel<2>;
  if (num_experts <= 128) return aspire_moe_route_kernel<4>;
  if (num_experts <= 256) return aspire_moe_route_kernel<8>;
  return aspire_moe_route_kernel<16>;
}

// Gradient of the weights to the logits, one warp per token.  Renormalised:
// d logit = w_j (g_j - sum_i w_i g_i) at choice j and 0 elsewhere.  Not
// renormalised (w_j = p_j of the softmax over all): d logit_e =
// p_e ([e chosen] g_e - sum_j p_j g_j), p_e computed again from the logits.
__global__ void __launch_bounds__(256) aspire_moe_route_grad_kernel(MoeRouteGradParams p) {
  pdl_begin();
  const int lane = threadIdx.x & 31;
  const int64_t token = int64_t(blockIdx.x) * (blockDim.x >> 5) + (threadIdx.x >> 5);
  if (token >= p.tokens) return;
  int32_t e = -1;
  float w = 0.f, g = 0.f;
  if (lane < p.top_k) {
    e = p.experts[token * p.top_k + lane];
    if (e >= 0 && e < p.num_experts) {
      w = p.weights[token * p.top_k + lane];
      g = p.grad_weights[token * p.top_k + lane];
    } else {
      e = -1;
    }
  }
  float inner = w * g;
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) inner += __shfl_xor_sync(0xffffffffu, inner, d);
  float m = -INFINITY, sum = 0.f;
  if (!p.renormalize) {
    for (int i = lane; i < p.num_experts; i += 32) {
      const float v = load_logit(p.logits, p.logits_type, token * p.logits_stride + i);
      if (v > m) m = v;  // NaN never wins
    }
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, d));
    if (m > -INFINITY) {
      for (int i = lane; i < p.num_experts; i += 32) {
        const float v = load_logit(p.logits, p.logits_type, token * p.logits_stride + i);
        if (v > -INFINITY) sum += exp_below(v, m);
      }
    }
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
  }
  for (int i0 = 0; i0 < p.num_experts; i0 += 32) {
    const int i = i0 + lane;
    float d = 0.f;
    for (int j = 0; j < p.top_k; ++j) {
      const int32_t ej = __shfl_sync(0xffffffffu, e, j);
      const float wj = __shfl_sync(0xffffffffu, w, j), gj = __shfl_sync(0xffffffffu, g, j);
      if (ej == i) d = p.renormalize ? wj * (gj - inner) : wj * gj;
    }
    if (i >= p.num_experts) continue;
    if (!p.renormalize) {
      const float v = load_logit(p.logits, p.logits_type, token * p.logits_stride + i);
      if (v > -INFINITY && sum > 0.f) d -= exp_below(v, m) / sum * inner;
    }
    const int64_t at = token * p.num_experts + i;
    if (p.logits_type == ASPIRE_T_F32)
      static_cast<float*>(p.grad_logits)[at] = d;
    else if (p.logits_type == ASPIRE_T_BF16)
      static_cast<__nv_bfloat16*>(p.grad_logits)[at] = __float2bfloat16_rn(d);
    else
      static_cast<__half*>(p.grad_logits)[at] = __float2half_rn(d);
  }
}

}  // namespace aspire
