// Router top-k and the sort of the tokens by expert.
//
// One warp per token.  Lane l holds the logits of experts l, l + 32, ... as
// order-preserving integers; each of the top_k rounds takes the warp's
// maximum and, among equals, the lowest expert index.  A NaN or -inf logit is
// never chosen: a token with fewer than top_k others gets expert -1 and
// weight 0 for the rest.  The weights are the softmax over all experts at the
// chosen ones or, renormalised, the softmax over the chosen ones.
//
// The sort counts: within a block of slots each warp ranks its 32 slots among
// those of the same expert (a warp match), per-warp counts are summed over
// the block's warps and the earlier blocks' counts, so the order is stable
// and no atomic decides it.  One block sorts a decode step in the launch that
// routes it; more tokens take a second launch after every block's counts are
// known.  Both are bound by latency: the bytes are a few megabytes at most.
#include "moe.cuh"

namespace aspire {

namespace {

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
  int32_t scan[32];
};

// Sorts the block's slots (thread = slot, expert id or -1).  earlier[e] /
// total[e]: slots of expert e in earlier blocks / all blocks; with one block
// they are 0 and the block's own counts.
__device__ void sort_block(const MoeRouteParams& p, SortShared& sh, int32_t id, int64_t slot, bool live, bool one) {
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int warps = blockDim.x >> 5, E = p.num_experts;
  for (int i = tid; i < warps * E; i += blockDim.x) sh.count[i / E][i % E] = 0;
  __syncthreads();
  const unsigned peers = __match_any_sync(0xffffffffu, id);
  const int rank = __popc(peers & ((1u << lane) - 1));
  if (id >= 0 && rank == 0) sh.count[warp][id] = uint16_t(__popc(peers));
  __syncthreads();
  // Thread e: the warps' counts become offsets within the block; then the
  // experts' totals are scanned over all threads (E <= blockDim).
  int32_t total = 0, earlier = 0;
  if (tid < E) {
    int32_t run = 0;
    for (int w = 0; w < warps; ++w) {
      const int32_t n = sh.count[w][tid];
      sh.count[w][tid] = uint16_t(run);
      run += n;
    }
    if (one) {
      total = run;
    } else {
      const int blocks = gridDim.x, self = blockIdx.x;
      for (int b = 0; b < blocks; ++b) {
        const int32_t n = p.counts[int64_t(b) * E + tid];
        total += n;
        earlier += b < self ? n : 0;
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
  int32_t before = 0, all = 0;
  for (int w = 0; w < warps; ++w) {
    before += w < warp ? sh.scan[w] : 0;
    all += sh.scan[w];
  }
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

// Routes one token with the calling warp.
template <int EPL>
__device__ __forceinline__ void route_token(const MoeRouteParams& p, int64_t token, int lane) {
  uint32_t o[EPL];
#pragma unroll
  for (int i = 0; i < EPL; ++i) {
    const int e = lane + 32 * i;
    o[i] = e < p.num_experts ? order_of(load_logit(p.logits, p.logits_type, token * p.logits_stride + e)) : 0u;
  }
  uint32_t top = 0;  // the row's maximum
  float all = 0.f;   // softmax denominator over all experts
  uint32_t mine_o = 0;
  int32_t mine_e = -1;  // lane j keeps choice j
  for (int j = 0; j < p.top_k; ++j) {
    uint32_t best = 0;
    int at = 0;
#pragma unroll
    for (int i = EPL - 1; i >= 0; --i)
      if (o[i] >= best) {
        best = o[i];
        at = i;
      }
    const uint32_t m = __reduce_max_sync(0xffffffffu, best);
    if (j == 0) {
      top = m;
      if (!p.renormalize && m != 0) {
        const float mv = value_of(m);
#pragma unroll
        for (int i = 0; i < EPL; ++i)
          if (o[i] != 0) all += exp_below(value_of(o[i]), mv);
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) all += __shfl_xor_sync(0xffffffffu, all, d);
      }
    }
    if (m == 0) break;  // nothing left to choose
    const uint32_t e = __reduce_min_sync(0xffffffffu, best == m ? uint32_t(lane + 32 * at) : 0xffffffffu);
    if (lane == j) {
      mine_o = m;
      mine_e = int32_t(e);
    }
#pragma unroll
    for (int i = 0; i < EPL; ++i)
      if (uint32_t(lane + 32 * i) == e) o[i] = 0;
  }
  float w = mine_e >= 0 ? exp_below(value_of(mine_o), value_of(top)) : 0.f;
  if (p.renormalize) {
    all = w;
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) all += __shfl_xor_sync(0xffffffffu, all, d);
  }
  if (lane < p.top_k) {
    p.weights[token * p.top_k + lane] = mine_e >= 0 ? w / all : 0.f;
    p.experts[token * p.top_k + lane] = mine_e;
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
    for (int t = warp; t < nt; t += blockDim.x >> 5) route_token<EPL>(p, t0 + t, lane);
    __syncthreads();  // the block reads its own choices back
  }
  const bool live = tid < nt * p.top_k;
  const int64_t slot = t0 * p.top_k + tid;
  int32_t id = live ? p.experts[slot] : -1;
  if (id >= p.num_experts || id < 0) id = -1;
  if (gridDim.x == 1) {
    sort_block(p, sh, id, slot, live, true);
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
  sort_block(p, sh, id, slot, live, false);
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
