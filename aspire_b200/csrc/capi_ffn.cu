// extern "C" entry points of the feed-forward operators: 4-bit products and
// the tokens' way to their experts and back (declared in
// include/aspire_b200.h).  Argument checking and launch configuration; no
// entry point allocates device memory or synchronises, and none lets a C++
// exception out.
#include <algorithm>
#include <atomic>
#include <cstdint>
#include <string>

#include "errors.h"
#include "launch.cuh"
#include "moe.cuh"
#include "w4.cuh"

namespace aspire {
namespace {

// Runs an entry point's body; an exception (out of host memory while a message
// is built) becomes an error code.
template <typename F>
int guarded(F&& body) noexcept {
  try {
    clear_error();
    return body();
  } catch (...) {
    return ASPIRE_ERR_CAPACITY;
  }
}

int invalid(const char* who, const char* what) {
  return set_error(ASPIRE_ERR_INVALID, std::string(who) + ": " + what);
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

int ceil32(int v) { return (v + 31) / 32 * 32; }

// Rows up to which the kernel for few tokens runs: 16 of one matrix (16 rows
// 12288 -> 4096: 17.8 us against 25.4 on tcgen05; 32 rows 4096 -> 2 x 12288:
// 55 against 30), 8 on average of an expert (10 and 16 on average over 128
// experts 2048 -> 2 x 768: 90 and 117 us against 72 and 80; 4: 55 us).
constexpr int64_t kW4SmallRows = 16;
constexpr int64_t kW4SmallExpertRows = 8;
constexpr int64_t kMaxTileTokens = 128;

// Opt-in caches of the small kernel's variants: [type][tokens 8, 16]
// [groups 1, 2, 4][swiglu].
SmemOptIn g_w4_small[2][2][3][2];

int index_of(int v) { return v <= 1 ? 0 : (v == 2 ? 1 : 2); }

// Launch with a programmatic dependency and, for cluster > 1, clusters along x.
template <typename... KArgs, typename... Args>
int cluster_launch(void (*kernel)(KArgs...), dim3 grid, int cluster, int threads, size_t smem, cudaStream_t stream,
              const char* what, const Args&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = unsigned(cluster);
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = cluster > 1 ? 2 : 1;
  return check_cuda(cudaLaunchKernelEx(&cfg, kernel, args...), what);
}

// Clusters of 2, 4 and 8 CTAs that are resident at once (index log2 - 1), per
// device; 0: not asked yet.  (A GPC's SMs are no multiple of 8: 15 clusters of
// 8 CTAs with an SM each fit on 148 SMs, 33 of 4, 74 of 2.)
struct ClusterCounts {
  std::atomic<int> n[kMaxDevices][3];
  ClusterCounts() {
    for (auto& d : n)
      for (auto& c : d) c.store(0);
  }
};

template <typename Kernel>
int cluster_count(Kernel kernel, int threads, size_t smem, int cluster, ClusterCounts& cache, int* out) {
  int dev = 0;
  int rc = check_cuda(cudaGetDevice(&dev), "cudaGetDevice");
  if (rc) return rc;
  const int at = cluster == 2 ? 0 : (cluster == 4 ? 1 : 2);
  const bool cached = dev >= 0 && dev < kMaxDevices;
  int n = cached ? cache.n[dev][at].load(std::memory_order_relaxed) : 0;
  if (n == 0) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(unsigned(cluster));
    cfg.blockDim = dim3(unsigned(threads));
    cfg.dynamicSmemBytes = smem;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = unsigned(cluster);
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    rc = check_cuda(cudaOccupancyMaxActiveClusters(&n, kernel, &cfg), "cudaOccupancyMaxActiveClusters");
    if (rc) return rc;
    if (cached) cache.n[dev][at].store(n, std::memory_order_relaxed);
  }
  *out = n;
  return ASPIRE_OK;
}

ClusterCounts g_w4_small_clusters;

// CTAs that split a tile's K: the size whose waves of tiles take the fewest
// stages one after the other, a join of partials counted as `join` tenths of a
// stage.  `slots`: CTAs resident at once without clusters.
template <typename Kernel>
int pick_cluster(Kernel kernel, int threads, size_t smem, int64_t tiles, int64_t stages, int64_t slots, int64_t join,
                 ClusterCounts& cache, int* out) {
  *out = 1;
  if (2 * tiles > slots) return ASPIRE_OK;  // the rest would not hold a second wave
  int64_t best = (tiles + slots - 1) / slots * stages * 10;
  for (int c = 2; c <= 8 && c <= stages; c *= 2) {
    int n = 0;
    const int rc = cluster_count(kernel, threads, smem, c, cache, &n);
    if (rc) return rc;
    if (n <= 0) break;
    const int64_t cost = (tiles + n - 1) / n * ((stages + c - 1) / c * 10 + join);
    if (cost < best) {
      best = cost;
      *out = c;
    }
  }
  return ASPIRE_OK;
}

// Upper bound of the token tiles of `rows` rows in `experts` ranges, those of the
// rows before the first and past the last range included: a range of c rows has
// at most 1 + (c - 1) / width, and there are no more ranges than rows.
int64_t tiles_bound(int64_t rows, int32_t experts, bool grouped, int width) {
  if (!grouped) return (rows + width - 1) / width;
  return std::min<int64_t>(rows, int64_t(experts) + 2) + rows / width;
}

// Rows an ordinary tile has to hold: all of them, or an expert's average share.
int64_t typical_rows(const AspireW4Args* a) {
  return a->offsets ? (a->rows + a->experts - 1) / a->experts : a->rows;
}

int w4_small(const AspireW4Args* a, const W4Params& p, cudaStream_t stream) {
  const bool grouped = a->offsets != nullptr;
  // Tokens per tile: the fewest columns that hold the rows.
  const int64_t typical = typical_rows(a);
  const int tokens = typical <= 8 ? 8 : 16;
  const int groups = a->group == 32 ? 4 : (a->group == 64 ? 2 : 1);
  const int features = a->swiglu ? w4::kRows / 2 : w4::kRows;
  const int64_t ny = (int64_t(a->n) + features - 1) / features;
  const int64_t nz = tiles_bound(a->rows, a->experts, grouped, tokens);
  if (ny > 65535 || nz > 65535) return invalid("aspire_w4_linear", "n or rows too large");
  int sms = 0;
  int rc = current_sm_count(&sms);
  if (rc) return rc;
  W4Kernel kernel = w4_small_kernel(a->type == ASPIRE_T_BF16, tokens, groups, a->swiglu != 0);
  const size_t smem = w4_small_smem(tokens, groups);
  rc = ensure_smem(reinterpret_cast<const void*>(kernel), smem,
                   g_w4_small[a->type == ASPIRE_T_BF16][tokens != 8][index_of(groups)][a->swiglu != 0]);
  if (rc) return rc;
  // Two CTAs per SM; a join takes about 1.5 us, a stage 0.6.
  int cluster = 1;
  rc = pick_cluster(kernel, kW4SmallThreads, smem, ny * nz, (a->k + 255) / 256, 2 * sms, 25, g_w4_small_clusters,
                    &cluster);
  if (rc) return rc;
  return cluster_launch(kernel, dim3(unsigned(cluster), unsigned(ny), unsigned(nz)), cluster, kW4SmallThreads, smem, stream,
                   "aspire_w4_small_kernel launch", p);
}

int encode_map(CUtensorMap* map, CUtensorMapDataType type, int dims, const void* base, const cuuint64_t* size,
               const cuuint64_t* strides, const cuuint32_t* box) {
  PFN_cuTensorMapEncodeTiled_v12000 enc = tensor_map_encoder();
  if (!enc) return set_error(ASPIRE_ERR_CUDA, "cuTensorMapEncodeTiled entry point unavailable");
  const cuuint32_t ones[3] = {1, 1, 1};
  const CUresult r = enc(map, type, cuuint32_t(dims), const_cast<void*>(base), size, strides, box, ones,
                         CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                         CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS)
    return set_error(ASPIRE_ERR_INVALID,
                     "aspire_w4_linear: cuTensorMapEncodeTiled failed with code " + std::to_string(int(r)));
  return ASPIRE_OK;
}

SmemOptIn g_w4_tc[2][3][3][2];
ClusterCounts g_w4_tc_clusters;

int w4_tc(const AspireW4Args* a, const W4Params& p, cudaStream_t stream) {
  const bool grouped = a->offsets != nullptr;
  const int64_t typical = typical_rows(a);
  const int tokens = typical <= 32 ? 32 : (typical <= 64 ? 64 : 128);
  const int groups = a->group == 32 ? 4 : (a->group == 64 ? 2 : 1);
  const int features = a->swiglu ? w4::kRows : 2 * w4::kRows;
  const int64_t tiles = (int64_t(a->n) + features - 1) / features * tiles_bound(a->rows, a->experts, grouped, tokens);
  // (The second: ranges that overlap, which the kernel reports, count more tiles.)
  if (tiles > INT32_MAX || (grouped && a->experts * ((a->rows + tokens - 1) / tokens) > INT32_MAX))
    return invalid("aspire_w4_linear", "n or rows too large");
  int sms = 0;
  int rc = current_sm_count(&sms);
  if (rc) return rc;
  W4TcKernel kernel = w4_tc_kernel(a->type == ASPIRE_T_BF16, tokens, groups, a->swiglu != 0);
  const size_t smem = w4_tc_smem(tokens);
  rc = ensure_smem(reinterpret_cast<const void*>(kernel), smem,
                   g_w4_tc[a->type == ASPIRE_T_BF16][tokens == 32 ? 0 : (tokens == 64 ? 1 : 2)][index_of(groups)]
                          [a->swiglu != 0]);
  if (rc) return rc;
  // One CTA per SM; a join takes about 3 us, a stage 1.1.
  int cluster = 1;
  rc = pick_cluster(kernel, kW4TcThreads, smem, tiles, (a->k + 255) / 256, sms, 30, g_w4_tc_clusters, &cluster);
  if (rc) return rc;
  const int64_t ctas = cluster > 1 ? tiles : std::min<int64_t>(tiles, sms);
  CUtensorMap codes_map, x_map;
  {
    const cuuint64_t size[3] = {cuuint64_t(a->k / 8), cuuint64_t(a->n) * (a->swiglu ? 2 : 1),
                                cuuint64_t(grouped ? a->experts : 1)};
    const cuuint64_t strides[2] = {cuuint64_t(a->codes_stride) * 4,
                                   cuuint64_t(grouped && a->experts > 1 ? a->codes_stride_e : a->codes_stride) * 4};
    const cuuint32_t box[3] = {32, cuuint32_t(w4::kRows), 1};
    rc = encode_map(&codes_map, CU_TENSOR_MAP_DATA_TYPE_INT32, 3, a->codes, size, strides, box);
    if (rc) return rc;
  }
  {
    const cuuint64_t size[2] = {cuuint64_t(a->k), cuuint64_t(a->rows)};
    const cuuint64_t strides[1] = {cuuint64_t(a->x_stride) * 2};
    const cuuint32_t box[2] = {64, cuuint32_t(tokens)};
    rc = encode_map(&x_map,
                    a->type == ASPIRE_T_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2,
                    a->x, size, strides, box);
    if (rc) return rc;
  }
  return cluster_launch(kernel, dim3(unsigned(cluster), unsigned(ctas)), cluster, kW4TcThreads, smem, stream,
                   "aspire_w4_tc_kernel launch", p, codes_map, x_map);
}

int64_t elem_bytes(int32_t type) { return type == ASPIRE_T_F32 ? 4 : 2; }

bool known_type(int32_t t) { return t == ASPIRE_T_F32 || t == ASPIRE_T_BF16 || t == ASPIRE_T_F16; }

// Tokens per block of the sort, its blocks, and whether they are one cluster.
// A cluster takes a block per 8 tokens, so that its warps have one or two each
// (72 tokens of 128 experts: 9.9 us in one block, 5.5 in eight).
void route_blocks(int64_t tokens, int32_t top_k, int64_t* block_tokens, int64_t* blocks, bool* one) {
  *one = tokens <= int64_t(kMoeCluster) * (kMoeSlotsOne / top_k);
  if (*one) {
    *blocks = 1;
    while (*blocks < kMoeCluster && *blocks * 8 < tokens) *blocks *= 2;
    *block_tokens = (tokens + *blocks - 1) / *blocks;
  } else {
    *block_tokens = kMoeSlotsBlock / top_k;
    *blocks = (tokens + *block_tokens - 1) / *block_tokens;
  }
}

int check_permute(const AspireMoePermuteArgs* a, const char* who, bool grad) {
  if (!a) return invalid(who, "null argument");
  if (!known_type(a->type)) return invalid(who, "type must be ASPIRE_T_F32, ASPIRE_T_BF16 or ASPIRE_T_F16");
  if (a->tokens < 0 || a->top_k <= 0 || a->top_k > kMoeMaxTopK) return invalid(who, "bad token count or top_k");
  if (a->num_experts < 0 || a->width <= 0) return invalid(who, "bad expert count or width");
  if (a->tokens == 0) return ASPIRE_OK;
  if (a->tokens > INT32_MAX / a->top_k) return invalid(who, "too many tokens");
  if (!a->position || !a->offsets) return invalid(who, "null position or offsets");
  const int64_t vec = 16 / elem_bytes(a->type);
  if (a->width % vec) return invalid(who, "rows must be a multiple of 16 bytes");
  if ((a->in && (a->in_stride % vec || a->in_stride < a->width)) ||
      (a->out && (a->out_stride % vec || a->out_stride < a->width)) ||
      (a->residual && (a->residual_stride % vec || a->residual_stride < a->width)) ||
      (a->grad && (a->grad_stride % vec || a->grad_stride < a->width)))
    return invalid(who, "row strides must be multiples of 16 bytes and at least the width");
  if (!aligned16(a->in) || !aligned16(a->out) || !aligned16(a->residual) || !aligned16(a->grad))
    return invalid(who, "tensors must be 16-byte aligned");
  if (grad) {
    if (!a->grad) return invalid(who, "null gradient");
    if (a->grad_weights && !a->in) return invalid(who, "the weights' gradient needs the rows");
  } else if (!a->in || !a->out) {
    return invalid(who, "null tensor pointer");
  }
  return ASPIRE_OK;
}

MoePermuteParams permute_params(const AspireMoePermuteArgs* a) {
  MoePermuteParams p = {};
  p.in = a->in;
  p.in_stride = a->in_stride;
  p.residual = a->residual;
  p.residual_stride = a->residual_stride;
  p.weights = a->weights;
  p.position = a->position;
  p.offsets = a->offsets;
  p.num_experts = a->num_experts;
  p.tokens = int32_t(a->tokens);
  p.top_k = a->top_k;
  p.width = a->width;
  p.out = a->out;
  p.out_stride = a->out_stride;
  p.grad = a->grad;
  p.grad_stride = a->grad_stride;
  p.grad_weights = a->grad_weights;
  p.status = a->status;
  return p;
}

}  // namespace
}  // namespace aspire

using namespace aspire;

extern "C" {

int aspire_w4_linear(const AspireW4Args* a, void* stream) {
  return guarded([&]() -> int {
    const char* who = "aspire_w4_linear";
    if (!a) return invalid(who, "null argument");
    if (a->type != ASPIRE_T_BF16 && a->type != ASPIRE_T_F16)
      return invalid(who, "type must be ASPIRE_T_BF16 or ASPIRE_T_F16");
    // (Row counts are rounded up to tiles in 32 bits.)
    if (a->rows < 0 || a->rows > INT32_MAX - kMaxTileTokens || a->n <= 0 || a->k <= 0 || a->n > (1 << 29) || a->k > (1 << 29))
      return invalid(who, "bad sizes");
    if (a->group != 32 && a->group != 64 && (a->group <= 0 || a->group % 128))
      return invalid(who, "group must be 32, 64 or a multiple of 128");
    if (a->k % 32 || a->k % a->group) return invalid(who, "k must be a multiple of 32 and of group");
    // Up to here the group of a block is exact (group_recip).
    if (int64_t(a->k / 128) * (a->group / 128) > int64_t(1) << 32) return invalid(who, "k times group past 2^46");
    if (a->offsets && a->experts <= 0) return invalid(who, "offsets need experts > 0");
    if (a->offsets && a->experts > kW4MaxExperts) return invalid(who, "at most 1024 experts are supported");
    if (a->swiglu && a->residual) return invalid(who, "the gated form takes no residual");
    if (a->rows == 0) return ASPIRE_OK;
    if (!a->x || !a->codes || !a->scales || !a->out) return invalid(who, "null tensor pointer");
    const int64_t groups = a->k / a->group;
    if (a->x_stride < a->k || a->codes_stride < a->k / 8 || a->scales_stride < groups || a->out_stride < a->n ||
        (a->zeros && a->zeros_stride < groups) || (a->residual && a->residual_stride < a->n))
      return invalid(who, "a row stride is shorter than its row");
    if (!aligned16(a->x) || !aligned16(a->codes)) return invalid(who, "x and codes must be 16-byte aligned");
    if ((a->x_stride & 7) || (a->codes_stride & 3) || (a->offsets && (a->codes_stride_e & 3)))
      return invalid(who, "x rows must be multiples of 8 elements and codes rows of 4 words apart");
    W4Params p = {};
    p.x = static_cast<const uint16_t*>(a->x);
    p.x_stride = a->x_stride;
    p.rows = int32_t(a->rows);
    p.codes = a->codes;
    p.codes_stride = a->codes_stride;
    p.codes_stride_e = a->codes_stride_e;
    p.scales = static_cast<const uint16_t*>(a->scales);
    p.scales_stride = a->scales_stride;
    p.scales_stride_e = a->scales_stride_e;
    p.zeros = a->zeros;
    p.zeros_stride = a->zeros_stride;
    p.zeros_stride_e = a->zeros_stride_e;
    p.residual = static_cast<const uint16_t*>(a->residual);
    p.residual_stride = a->residual_stride;
    p.out = static_cast<uint16_t*>(a->out);
    p.out_stride = a->out_stride;
    p.out_quads = ((reinterpret_cast<uintptr_t>(a->out) & 7) | uintptr_t(a->out_stride & 3) | uintptr_t(a->n & 3)) == 0;
    p.n = a->n;
    p.k = a->k;
    p.group_blocks = std::max(a->group / 128, 1);
    p.group_recip = p.group_blocks > 1 ? uint32_t((uint64_t(1) << 32) / uint64_t(p.group_blocks)) + 1u : 0u;
    // 256 weights have 8, 4 or 2 groups: 16, 8 or 4 bytes of scales, and 8 or 4
    // of zero points (two groups' are half a word).
    const uintptr_t sb = a->group == 32 ? 16 : (a->group == 64 ? 8 : 4), zb = a->group == 32 ? 8 : 4;
    p.scales_vec = a->group <= 128 && (reinterpret_cast<uintptr_t>(a->scales) | uintptr_t(a->scales_stride * 2) |
                                       uintptr_t(a->offsets ? a->scales_stride_e * 2 : 0)) % sb == 0;
    p.zeros_vec = a->group <= 128 && (reinterpret_cast<uintptr_t>(a->zeros) | uintptr_t(a->zeros_stride) |
                                      uintptr_t(a->offsets ? a->zeros_stride_e : 0)) % zb == 0;
    p.offsets = a->offsets;
    p.num_experts = a->offsets ? a->experts : 0;
    p.status = a->status;
    p.wait_ns = wait_limit_ns();
    return typical_rows(a) <= (a->offsets ? kW4SmallExpertRows : kW4SmallRows)
               ? w4_small(a, p, static_cast<cudaStream_t>(stream))
               : w4_tc(a, p, static_cast<cudaStream_t>(stream));
  });
}

size_t aspire_moe_route_workspace(int64_t tokens, int32_t num_experts, int32_t top_k) {
  if (tokens <= 0 || top_k <= 0 || top_k > kMoeMaxTopK || num_experts <= 0 || tokens > INT32_MAX / top_k) return 0;
  int64_t bt, nb;
  bool one;
  route_blocks(tokens, top_k, &bt, &nb, &one);
  return one ? 0 : size_t(nb) * size_t(num_experts) * sizeof(int32_t);
}

int aspire_moe_route(const AspireMoeRouteArgs* a, void* stream) {
  return guarded([&]() -> int {
    const char* who = "aspire_moe_route";
    if (!a) return invalid(who, "null argument");
    if (a->num_experts <= 0 || a->num_experts > kMoeMaxExperts) return invalid(who, "num_experts must be in [1, 512]");
    if (a->top_k <= 0 || a->top_k > kMoeMaxTopK) return invalid(who, "top_k must be in [1, 32]");
    if (a->logits && a->top_k > a->num_experts) return invalid(who, "top_k must not exceed num_experts");
    if (a->tokens < 0 || a->tokens > INT32_MAX / a->top_k) return invalid(who, "bad token count");
    if (a->logits && !known_type(a->logits_type)) return invalid(who, "bad logits type");
    if (a->logits && a->tokens > 1 && a->logits_stride < a->num_experts)
      return invalid(who, "logits rows are shorter than num_experts");
    if (!a->offsets) return invalid(who, "null offsets");
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (a->tokens == 0)
      return check_cuda(cudaMemsetAsync(a->offsets, 0, sizeof(int32_t) * (size_t(a->num_experts) + 1), st),
                        "aspire_moe_route memset");
    if (!a->experts || !a->position || !a->source || (a->logits && !a->weights)) return invalid(who, "null pointer");
    int64_t bt, nb;
    bool one;
    route_blocks(a->tokens, a->top_k, &bt, &nb, &one);
    if (!one && (!a->workspace || a->workspace_bytes < aspire_moe_route_workspace(a->tokens, a->num_experts, a->top_k)))
      return set_error(ASPIRE_ERR_CAPACITY, "aspire_moe_route: workspace too small");
    MoeRouteParams p = {};
    p.logits = a->logits;
    p.logits_type = a->logits_type;
    p.logits_stride = a->logits_stride;
    p.tokens = int32_t(a->tokens);
    p.num_experts = a->num_experts;
    p.top_k = a->top_k;
    p.renormalize = a->renormalize ? 1 : 0;
    p.weights = a->weights;
    p.experts = a->experts;
    p.position = a->position;
    p.source = a->source;
    p.offsets = a->offsets;
    p.counts = one ? nullptr : a->workspace;
    p.block_tokens = int32_t(bt);
    if (one) {  // a thread per slot and per expert, a warp per token
      int threads = std::max(ceil32(int(bt * a->top_k)), ceil32(a->num_experts));
      if (a->logits) threads = std::max(threads, 32 * int(std::min<int64_t>(bt, 32)));
      return cluster_launch(moe_route_kernel(a->logits ? a->num_experts : 0), dim3(unsigned(nb)), int(nb), threads, 0,
                            st, "aspire_moe_route_kernel launch", p);
    }
    int rc = launch(moe_route_kernel(a->logits ? a->num_experts : 0), dim3(unsigned(nb)), dim3(kMoeSlotsBlock), 0, st,
                    "aspire_moe_route_kernel launch", p);
    if (rc) return rc;
    return launch(aspire_moe_sort_kernel, dim3(unsigned(nb)), dim3(kMoeSlotsBlock), 0, st,
                  "aspire_moe_sort_kernel launch", p);
  });
}

int aspire_moe_route_grad(const AspireMoeRouteGradArgs* a, void* stream) {
  return guarded([&]() -> int {
    const char* who = "aspire_moe_route_grad";
    if (!a) return invalid(who, "null argument");
    if (a->num_experts <= 0 || a->num_experts > kMoeMaxExperts || a->top_k <= 0 || a->top_k > kMoeMaxTopK ||
        a->top_k > a->num_experts || a->tokens < 0 || a->tokens > INT32_MAX / a->top_k)
      return invalid(who, "bad sizes");
    if (!known_type(a->logits_type)) return invalid(who, "bad logits type");
    if (a->tokens == 0) return ASPIRE_OK;
    if (!a->weights || !a->experts || !a->grad_weights || !a->grad_logits || (!a->renormalize && !a->logits))
      return invalid(who, "null pointer");
    if (!a->renormalize && a->tokens > 1 && a->logits_stride < a->num_experts)
      return invalid(who, "logits rows are shorter than num_experts");
    MoeRouteGradParams p = {};
    p.logits = a->logits;
    p.logits_type = a->logits_type;
    p.logits_stride = a->logits_stride;
    p.weights = a->weights;
    p.experts = a->experts;
    p.grad_weights = a->grad_weights;
    p.tokens = int32_t(a->tokens);
    p.num_experts = a->num_experts;
    p.top_k = a->top_k;
    p.renormalize = a->renormalize ? 1 : 0;
    p.grad_logits = a->grad_logits;
    return launch(aspire_moe_route_grad_kernel, dim3(unsigned((a->tokens + 7) / 8)), dim3(256), 0,
                  static_cast<cudaStream_t>(stream), "aspire_moe_route_grad_kernel launch", p);
  });
}

int aspire_moe_dispatch(const AspireMoePermuteArgs* a, void* stream) {
  return guarded([&]() -> int {
    int rc = check_permute(a, "aspire_moe_dispatch", false);
    if (rc || a->tokens == 0) return rc;
    return launch(moe_dispatch_kernel(a->type), dim3(unsigned(a->tokens)), dim3(kMoeThreads), 0,
                  static_cast<cudaStream_t>(stream), "aspire_moe_dispatch_kernel launch", permute_params(a));
  });
}

int aspire_moe_combine(const AspireMoePermuteArgs* a, void* stream) {
  return guarded([&]() -> int {
    int rc = check_permute(a, "aspire_moe_combine", false);
    if (rc || a->tokens == 0) return rc;
    return launch(moe_combine_kernel(a->type), dim3(unsigned(a->tokens)), dim3(kMoeThreads), 0,
                  static_cast<cudaStream_t>(stream), "aspire_moe_combine_kernel launch", permute_params(a));
  });
}

int aspire_moe_combine_grad(const AspireMoePermuteArgs* a, void* stream) {
  return guarded([&]() -> int {
    int rc = check_permute(a, "aspire_moe_combine_grad", true);
    if (rc || a->tokens == 0) return rc;
    if (!a->out && !a->grad_weights) return ASPIRE_OK;
    return launch(moe_combine_grad_kernel(a->type), dim3(unsigned(a->tokens)), dim3(kMoeThreads), 0,
                  static_cast<cudaStream_t>(stream), "aspire_moe_combine_grad_kernel launch", permute_params(a));
  });
}

}  // extern "C"
