// The accepted path of each row's tree, and its keys and values moved to their
// committed places in every layer's cache:
//
//   node_0 = 0;  node_{d+1} = the first child of node_d whose token is
//   targets[node_d], the target's choice after node_d; the walk ends where no
//   child has it, or at max_path nodes;
//   count = nodes walked, tokens_d = targets[node_d] (the accepted drafts,
//   then the target's next token), length + count committed tokens;
//   cache place length + node_d  ->  length + d  (K and V, all heads).
//
// A CTA serves one row of one layer: its first warp walks (all layers' CTAs
// walk alike, which is a few L1-resident reads, against a second launch), then
// each thread moves the same 16 bytes of one token after another.  node_d
// grows with d and is at least d, so a place is written only after the same
// thread has read it.
#include "tree.cuh"

namespace aspire {

namespace {

__device__ __forceinline__ int64_t place_offset(const AcceptParams& p, int b, int64_t pos, uint32_t& bad) {
  const int64_t col = pos / p.page_size;
  const int32_t page = col < p.table_cols ? p.table[b * p.table_stride + col] : -1;
  if (page < 0 || page >= p.pages) {
    bad |= ASPIRE_STATUS_BAD_PAGE;
    return -1;
  }
  return (int64_t(page) * 2 * p.page_size + pos % p.page_size) * p.token_bytes;
}

}  // namespace

__global__ void __launch_bounds__(kAcceptThreads) aspire_tree_accept_kernel(const __grid_constant__ AcceptParams p) {
  pdl_begin();
  __shared__ int32_t path[kAcceptMaxPath];
  __shared__ int64_t from[kAcceptMaxPath], to[kAcceptMaxPath];
  __shared__ int walked;
  const int tid = threadIdx.x, lane = tid & 31;
  const int b = blockIdx.x;
  const bool writer = blockIdx.y == 0;  // the row's outputs come from one CTA
  int64_t lo = p.indptr[b], hi = p.indptr[b + 1];
  uint32_t bad = 0;
  if (lo < 0 || hi < lo || hi > p.total) {
    bad = ASPIRE_STATUS_BAD_ROW;
    hi = lo = 0;
  }
  if (tid < 32) {
    int count = 0;
    int32_t node = 0;
    bool more = hi > lo;
    while (more) {
      if (lane == 0) path[count] = node;
      ++count;
      more = false;
      if (count == p.max_path) break;
      const int32_t want = p.targets[lo + node];
      // Children come after their parent.
      for (int64_t c0 = int64_t(node) + 1; c0 < hi - lo; c0 += 32) {
        const int64_t c = c0 + lane;
        const bool hit = c < hi - lo && p.parents[lo + c] == node && p.tokens[lo + c] == want;
        const uint32_t found = __ballot_sync(0xffffffffu, hit);
        if (found) {
          node = int32_t(c0) + __ffs(int(found)) - 1;
          more = true;
          break;
        }
      }
    }
    if (lane == 0) walked = count;
  }
  __syncthreads();
  const int count = walked;
  const int64_t length = max(p.lengths[b], 0);
  if (writer) {
    for (int d = tid; d < p.max_path; d += kAcceptThreads) {
      p.path[int64_t(b) * p.max_path + d] = d < count ? path[d] : -1;
      p.out_tokens[int64_t(b) * p.max_path + d] = d < count ? p.targets[lo + path[d]] : -1;
    }
    if (tid == 0) {
      p.count[b] = count;
      p.new_lengths[b] = int32_t(min(length + count, int64_t(INT32_MAX)));
    }
  }
  if (p.num_caches > 0) {
    for (int d = tid; d < count; d += kAcceptThreads) {
      from[d] = to[d] = -1;
      if (path[d] != d) {
        from[d] = place_offset(p, b, length + path[d], bad);
        to[d] = place_offset(p, b, length + d, bad);
      }
    }
    __syncthreads();
    const int64_t value_at = int64_t(p.page_size) * p.token_bytes;  // from a token's K to its V
    const int pieces = int(p.token_bytes / 16);
    for (int layer = blockIdx.y; layer < p.num_caches; layer += gridDim.y) {
      for (int i = tid; i < 2 * pieces; i += kAcceptThreads) {
        char* base = p.caches[layer] + (i < pieces ? int64_t(i) * 16 : value_at + int64_t(i - pieces) * 16);
        for (int d = 1; d < count; ++d)
          if (from[d] >= 0 && to[d] >= 0)
            *reinterpret_cast<uint4*>(base + to[d]) = *reinterpret_cast<const uint4*>(base + from[d]);
      }
    }
  }
  if (bad && writer) record_status(p.status, bad);
}

}  // namespace aspire
