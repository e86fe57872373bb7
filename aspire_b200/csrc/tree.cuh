// Parameter blocks of the operators of a tree-speculation step: step tables
// (step_tables.cu), logits (logits.cu) and the accepted path
// (tree_accept.cu).
#pragma once

#include "kernels.cuh"

namespace aspire {

struct StepTablesParams {
  const int32_t* lengths;     // [rows]
  const int32_t* new_tokens;  // [rows], or NULL: none
  int32_t rows;
  int32_t page_size;
  int32_t* table;             // [rows, table_stride], table_cols used
  int64_t table_stride;
  int32_t table_cols;
  int32_t* held;              // [rows]
  int32_t* free_pages;        // [free_capacity]
  int32_t* free_count;        // [1]
  int64_t free_capacity;
  const int32_t* parents;     // [tokens] or NULL
  int32_t mask_words;         // 0 without parents
  int64_t tokens;
  int32_t* qo_indptr;         // [rows + 1]
  int32_t* kv_indptr;         // [rows + 1]
  int32_t* kv_len;            // [rows]
  int32_t* last_page_len;     // [rows]
  int32_t* positions;         // [tokens]
  int64_t* slots;             // [tokens]
  int32_t* tree_mask;         // [tokens, mask_words]
  uint32_t* status;
};
constexpr int kTablesThreads = 1024;
__global__ void aspire_step_tables_kernel(StepTablesParams p);
constexpr int kStepTokensThreads = 256;
__global__ void aspire_step_tokens_kernel(StepTablesParams p);

struct LogitsParams {
  const void* logits;
  int64_t logits_stride;      // elements between tokens
  void* out;                  // NULL: pick only
  int64_t out_stride;
  int64_t tokens;
  int32_t vocab;
  int32_t rows;
  const int32_t* indptr;      // [rows + 1] or NULL: token t is row t's
  const int32_t* history;     // [rows, history_stride]
  int64_t history_stride;
  int32_t history_cols;
  const int32_t* history_len; // [rows]
  const int32_t* prompt_len;  // [rows] or NULL
  const int32_t* step_tokens; // [tokens] or NULL
  const int32_t* tree_mask;   // [tokens, mask_words] or NULL
  int32_t mask_words;
  const float* repetition;    // [rows] or NULL each
  const float* frequency;
  const float* presence;
  const int32_t* bias_indptr; // [rows + 1] or NULL
  const int32_t* bias_ids;
  const float* bias_values;
  int64_t bias_entries;
  const int32_t* allowed;     // [tokens, allowed_stride] words or NULL
  int64_t allowed_stride;
  int32_t slice;              // vocabulary entries of a CTA
  int32_t slices;
  float* best_value;          // [tokens, slices], NULL: no pick
  int32_t* best_id;
  int32_t* ids;               // [tokens]
  uint32_t* status;
};
constexpr int kLogitsThreads = 256;
using LogitsKernel = void (*)(LogitsParams);
LogitsKernel logits_kernel(int type);  // aspire_logits_kernel of an ASPIRE_T_*
__global__ void aspire_pick_kernel(LogitsParams p);
constexpr int kPickThreads = 128;

constexpr int kAcceptCaches = 128;
struct AcceptParams {
  const int32_t* tokens;   // [total]
  const int32_t* parents;
  const int32_t* targets;
  const int32_t* indptr;   // [rows + 1]
  const int32_t* lengths;  // [rows]
  int64_t total;
  int32_t rows;
  int32_t max_path;
  int32_t* count;          // [rows]
  int32_t* path;           // [rows, max_path]
  int32_t* out_tokens;     // [rows, max_path]
  int32_t* new_lengths;    // [rows]
  const int32_t* table;    // [rows, table_stride]
  int64_t table_stride;
  int32_t table_cols;
  int32_t page_size;
  int64_t pages;
  int64_t token_bytes;     // bytes of one token's K (or V) of all heads, a multiple of 16
  int32_t num_caches;
  uint32_t* status;
  char* caches[kAcceptCaches];
};
constexpr int kAcceptThreads = 256;
constexpr int kAcceptMaxPath = 64;
__global__ void aspire_tree_accept_kernel(const __grid_constant__ AcceptParams p);

}  // namespace aspire
