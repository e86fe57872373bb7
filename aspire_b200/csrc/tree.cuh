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
constexpr int kFewTokens = 4096;  // that the tables' kernel does itself, if their rows are one tile
using TablesKernel = void (*)(StepTablesParams);
TablesKernel step_tables_kernel(bool few);  // aspire_step_tables_kernel
constexpr int kStepTokensThreads = 256;
__global__ void aspire_step_tokens_kernel(StepTablesParams p);

struct LogitsParams {
  const void* logits;
  int64_t logits_stride;      // elements between tokens
  void* out;
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
  int32_t* ids;               // [tokens]: the best tokens, or NULL: adjusted logits to out
  // Workspace.  Where the marking CTAs' lists lie: list_base.
  unsigned long long* keys;   // [tokens], with ids
  uint32_t* arrived;          // [tokens], with ids: slices done
  int2* list;                 // touched ids with their counts and flags; NULL: nothing touches the logits
  uint2* list_bias;           // with biases, of ids that have one: 1 + the entry's number, the bias
  int2* table;                // [rows, blocks * kLogitsBlock / kLogitsUnit]: a unit's part of the list
  uint32_t* touched;          // [rows, blocks, kLogitsBlock / 32] bitmap
  int32_t mark_ranks;         // CTAs that mark a row
  int32_t mark_blocks;        // blocks of each
  int32_t list_stride;        // entries from a marking CTA's list to the next, or 0: as many as its row can touch
  uint32_t* status;
};
constexpr int kLogitsBlock = 4096;  // vocabulary entries, the steps of a marking CTA's share
constexpr int kLogitsUnit = 512;    // vocabulary entries that share an entry of the table
constexpr int kMarkThreads = 1024;
constexpr int kMarkMaxBlocks = 21;  // of a CTA with 16-bit counts: 216 KB of counts and bits
constexpr int kMarkMaxWide = 12;    // with 32-bit ones: 219 KB
constexpr int kMarkNarrow = 65535;  // history up to which 16 bits count
using LogitsKernel = void (*)(LogitsParams);
LogitsKernel mark_kernel(bool wide);  // aspire_logits_mark_kernel
size_t mark_smem_bytes(int blocks, bool wide);
constexpr int kLogitsThreads = 256;
constexpr int kLogitsCtas = 3;  // of an SM
LogitsKernel logits_kernel(int type, bool pick);  // aspire_logits_kernel of an ASPIRE_T_*
int logits_slice(int type);                       // vocabulary entries of one of its CTAs at a time
size_t logits_smem_bytes();

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
  const int32_t* kv_len;   // [rows] or NULL
  char* caches[kAcceptCaches];
};
constexpr int kAcceptThreads = 256;
constexpr int kAcceptMaxPath = 64;
__global__ void aspire_tree_accept_kernel(const __grid_constant__ AcceptParams p);

}  // namespace aspire
