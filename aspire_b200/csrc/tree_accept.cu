// The accepted path of each row's tree, and its keys and values moved to their
// committed places in every layer's cache:
//
//   node_0 = 0;  node_{d+1} = the first child of node_d whose token is
//   targets[node_d], the target's choice after node_d; the walk ends where no
//   child has it, at max_path nodes, or before a node without a choice
//   (targets[node] < 0): what is committed are tokens, and -1 is none;
//   count = nodes walked, tokens_d = targets[node_d] (the accepted drafts,
//   then the target's next token), length + count committed tokens;
//   cache place length + node_d  ->  length + d  (K and V, all heads).
//
// Given the step's key counts (kv_len), the walk keeps to nodes whose keys the
// cache holds: those at places below kv_len, none of a row that got no pages,
// up to the first whose place has no page.
//
// A CTA serves one row and some of the layers.  Its tree is read to shared
// memory at once and walked there by the first warp; every CTA of the row walks
// alike, which costs less than a second launch.  Then each thread moves the
// same 16 bytes of up to kBatch tokens at a time, all read before the first is
// written.  node_d grows with d and is at least d, so no place is written
// before it is read.  Bound by latency (the tree, the walk, the pages, the
// move); 64 rows of 36 layers with 8 heads move 17 MB: 14.4 us, one row of 28
// layers 6.3.
#include "tree.cuh"

namespace aspire {

namespace {

constexpr int kTree = 1024;  // nodes held in shared memory; larger trees are walked where they are
constexpr int kBatch = 8;    // tokens moved together

__device__ __forceinline__ int64_t place_offset(const AcceptParams& p, int b, int64_t pos, uint32_t& bad) {
  const int64_t col = pos / p.page_size;
  const int32_t page = col < p.table_cols ? p.table[b * p.table_stride + col] : -1;
  if (page < 0 || page >= p.pages) {
    bad |= ASPIRE_STATUS_BAD_PAGE;
    return -1;
  }
  return (int64_t(page) * 2 * p.page_size + pos % p.page_size) * p.token_bytes;
}

// The walk, by one warp; `path` gets the nodes.  `dead` is set where it ends before a node without a choice.
__device__ __forceinline__ int walk(const int32_t* tokens, const int32_t* parents, const int32_t* targets, int n,
                                    int max_path, int lane, int32_t* path, bool& dead) {
  int count = 0, node = 0;
  bool more = n > 0;
  while (more) {
    const int32_t want = targets[node];
    if (want < 0) {
      dead = true;
      break;
    }
    if (lane == 0) path[count] = node;
    ++count;
    more = false;
    if (count == max_path) break;
    for (int c0 = node + 1; c0 < n; c0 += 32) {  // children come after their parent
      const int c = c0 + lane;
      const uint32_t found = __ballot_sync(0xffffffffu, c < n && parents[c] == node && tokens[c] == want);
      if (found) {
        node = c0 + __ffs(int(found)) - 1;
        more = true;
        break;
      }
    }
  }
  return count;
}

}  // namespace

__global__ void __launch_bounds__(kAcceptThreads) aspire_tree_accept_kernel(const __grid_constant__ AcceptParams p) {
  pdl_begin();
  __shared__ int32_t tokens[kTree], parents[kTree], targets[kTree];
  __shared__ int32_t path[kAcceptMaxPath];
  __shared__ int64_t from[kAcceptMaxPath], to[kAcceptMaxPath];
  __shared__ int walked, moves;
  const int tid = threadIdx.x, lane = tid & 31;
  const int b = blockIdx.x;
  const bool writer = blockIdx.y == 0;  // the row's outputs come from one CTA
  int64_t lo = p.indptr[b], hi = p.indptr[b + 1];
  const int64_t length = max(p.lengths[b], 0);
  uint32_t bad = 0;
  if (lo < 0 || hi < lo || hi > p.total) {
    bad = ASPIRE_STATUS_BAD_ROW;
    hi = lo = 0;
  }
  int n = int(hi - lo);
  if (p.kv_len) n = int(min(int64_t(n), max(int64_t(p.kv_len[b]) - length, int64_t(0))));
  const bool held = n <= kTree;
  if (held)
    for (int i = tid; i < n; i += kAcceptThreads) {
      tokens[i] = p.tokens[lo + i];
      parents[i] = p.parents[lo + i];
      targets[i] = p.targets[lo + i];
    }
  __syncthreads();
  const int32_t* want = held ? targets : p.targets + lo;
  if (tid < 32) {
    bool dead = false;
    const int count =
        walk(held ? tokens : p.tokens + lo, held ? parents : p.parents + lo, want, n, p.max_path, lane, path, dead);
    if (dead) bad |= ASPIRE_STATUS_NO_TOKEN;
    __syncwarp();
    // The moves: nodes that lie behind their places, all of a path's from the first such on.
    int first = count, kept = count;
    for (int d = lane; d < count; d += 32) {
      if (path[d] != d) first = min(first, d);
      if (p.num_caches > 0 && (path[d] != d || p.kv_len)) {
        from[d] = place_offset(p, b, length + path[d], bad);
        to[d] = place_offset(p, b, length + d, bad);
        if (from[d] < 0) to[d] = -1;
        if (p.kv_len && to[d] < 0) kept = min(kept, d);
      }
    }
    first = __reduce_min_sync(0xffffffffu, first);
    kept = __reduce_min_sync(0xffffffffu, kept);
    if (lane == 0) {
      walked = kept;
      moves = min(first, kept);
    }
  }
  __syncthreads();
  const int count = walked;
  if (writer) {
    for (int d = tid; d < p.max_path; d += kAcceptThreads) {
      p.path[int64_t(b) * p.max_path + d] = d < count ? path[d] : -1;
      p.out_tokens[int64_t(b) * p.max_path + d] = d < count ? want[path[d]] : -1;
    }
    if (tid == 0) {
      p.count[b] = count;
      p.new_lengths[b] = int32_t(min(length + count, int64_t(INT32_MAX)));
    }
    if (bad) record_status(p.status, bad);
  }
  if (p.num_caches == 0 || moves == count) return;
  const int64_t value_at = int64_t(p.page_size) * p.token_bytes;  // from a token's K to its V
  const int pieces = int(p.token_bytes / 16);
  const int layers = (p.num_caches - int(blockIdx.y) + gridDim.y - 1) / gridDim.y;
  for (int64_t u = tid; u < int64_t(layers) * 2 * pieces; u += kAcceptThreads) {
    const int layer = int(u / (2 * pieces)), i = int(u - int64_t(layer) * 2 * pieces);
    char* base = p.caches[blockIdx.y + layer * gridDim.y] +
                 (i < pieces ? int64_t(i) * 16 : value_at + int64_t(i - pieces) * 16);
    for (int d0 = moves; d0 < count; d0 += kBatch) {
      uint4 v[kBatch];
#pragma unroll
      for (int k = 0; k < kBatch; ++k)
        if (d0 + k < count && to[d0 + k] >= 0) v[k] = *reinterpret_cast<const uint4*>(base + from[d0 + k]);
#pragma unroll
      for (int k = 0; k < kBatch; ++k)
        if (d0 + k < count && to[d0 + k] >= 0) *reinterpret_cast<uint4*>(base + to[d0 + k]) = v[k];
    }
  }
}

}  // namespace aspire
