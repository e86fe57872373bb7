// Routing of tokens to experts: parameters of the kernels in moe_route.cu
// (top-k, sort by expert) and moe_permute.cu (the way there and back).
//
// A slot is a (token, choice) pair, numbered token * top_k + choice.  The
// sort puts the slots in order of (expert, slot): position[slot] is a slot's
// row among the sorted ones (-1: no expert), source[row] the slot of a row
// (-1 past the last one), offsets[e] the first row of expert e.
#pragma once

#include "kernels.cuh"

namespace aspire {

constexpr int kMoeMaxExperts = 512;
constexpr int kMoeMaxTopK = 32;
// One launch routes and sorts up to 8 x 1024 slots: a cluster of up to 8 blocks
// of up to 1024.  More slots go in blocks of 512 and take two launches.
constexpr int kMoeCluster = 8;
constexpr int kMoeSlotsOne = 1024;
constexpr int kMoeSlotsBlock = 512;

struct MoeRouteParams {
  const void* logits;      // [tokens, experts] fp32, bf16 or fp16; NULL: `experts` is an input
  int32_t logits_type;     // ASPIRE_T_*
  int64_t logits_stride;
  int32_t tokens, num_experts, top_k;
  int32_t renormalize;
  float* weights;          // [tokens, top_k]
  int32_t* experts;        // [tokens, top_k]
  int32_t* position;       // [tokens * top_k]
  int32_t* source;         // [tokens * top_k]
  int32_t* offsets;        // [num_experts + 1]
  int32_t* counts;         // [blocks, num_experts] with two launches, else NULL
  int32_t block_tokens;    // tokens of a block
};
// Top-k and, with `counts`, the block's expert counts; without it the sort of
// the one cluster's slots.
using MoeRouteKernel = void (*)(MoeRouteParams);
MoeRouteKernel moe_route_kernel(int32_t num_experts);
// Sort of one block's slots, from every block's counts.
__global__ void aspire_moe_sort_kernel(MoeRouteParams p);

struct MoeRouteGradParams {
  const void* logits;      // read only without renormalisation
  int32_t logits_type;
  int64_t logits_stride;
  const float* weights;
  const int32_t* experts;
  const float* grad_weights;  // contiguous [tokens, top_k]
  int32_t tokens, num_experts, top_k, renormalize;
  void* grad_logits;       // contiguous [tokens, experts], the logits' type
};
__global__ void aspire_moe_route_grad_kernel(MoeRouteGradParams p);

struct MoePermuteParams {
  const void* in;          // dispatch: x [tokens, width]; combine and its gradient: rows [tokens * top_k, width]
  int64_t in_stride;
  const void* residual;    // combine: [tokens, width] or NULL
  int64_t residual_stride;
  const float* weights;    // [tokens, top_k] or NULL: 1
  const int32_t* position;
  const int32_t* offsets;
  int32_t num_experts, tokens, top_k, width;
  void* out;               // dispatch: rows; combine: [tokens, width]
  int64_t out_stride;
  // Combine's gradient: `out` is the gradient of the rows (or NULL), this the
  // outputs' gradient and the weights' (or NULL).
  const void* grad;
  int64_t grad_stride;
  float* grad_weights;
  uint32_t* status;
};
constexpr int kMoeThreads = 128;
using MoePermuteKernel = void (*)(MoePermuteParams);
MoePermuteKernel moe_dispatch_kernel(int32_t type);
MoePermuteKernel moe_combine_kernel(int32_t type);
MoePermuteKernel moe_combine_grad_kernel(int32_t type);

}  // namespace aspire
