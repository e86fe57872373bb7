// extern "C" entry points of a tree-speculation step (declared in
// include/aspire_b200.h): argument checking and launch configuration.  No
// entry point allocates device memory or synchronises, and none lets a C++
// exception out.  (The attention under a tree mask is in capi.cu.)
#include <algorithm>
#include <cstdint>
#include <string>

#include "errors.h"
#include "launch.cuh"
#include "tree.cuh"

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

SmemOptIn g_logits_smem[3];  // by ASPIRE_T_*

// Vocabulary entries of a CTA and how many CTAs share a row.
struct Slicing {
  int32_t slice, slices;
};

// Shared memory of a slice: a bit and a count an entry, with biases an entry's number too.
size_t slice_bytes(int64_t slice, bool bias) { return size_t((slice + 31) / 32 * 4 + slice * (bias ? 8 : 4)); }

constexpr int64_t kSliceStep = 256;
constexpr int64_t kMostSlice = 25600;  // 103 KB: two CTAs fit an SM

Slicing slicing(int32_t rows, int32_t vocab, bool bias, int sms) {
  const int64_t most = bias ? kMostSlice / 2 : kMostSlice;
  const int64_t least = (int64_t(vocab) + most - 1) / most;
  int64_t n = std::max<int64_t>(least, (2 * int64_t(sms) + rows - 1) / std::max(rows, 1));
  n = std::min<int64_t>(n, (int64_t(vocab) + kSliceStep - 1) / kSliceStep);
  const int64_t slice = ((int64_t(vocab) + n - 1) / n + kSliceStep - 1) / kSliceStep * kSliceStep;
  return {int32_t(slice), int32_t((int64_t(vocab) + slice - 1) / slice)};
}

int step_tables(const AspireStepTablesArgs* a, void* stream) {
  const char* who = "aspire_step_tables";
  if (!a) return invalid(who, "null argument");
  if (a->rows < 0 || a->tokens < 0 || a->tokens > INT32_MAX) return invalid(who, "rows or tokens out of range");
  if (a->page_size < 1) return invalid(who, "page_size must be > 0");
  if (a->free_capacity < 0 || a->free_capacity > INT32_MAX || a->block_table_cols < 0)
    return invalid(who, "free_capacity or block_table_cols out of range");
  if (!a->qo_indptr || !a->kv_indptr || !a->free_count || (a->free_capacity > 0 && !a->free_pages))
    return invalid(who, "null pointer");
  if (a->rows > 0 && (!a->lengths || !a->held || !a->kv_len || !a->last_page_len ||
                      (a->block_table_cols > 0 && !a->block_table)))
    return invalid(who, "null pointer");
  if (a->tokens > 0 && (!a->positions || !a->slots)) return invalid(who, "positions and slots are required");
  if (a->parents && (a->tree_mask_words < 1 || (a->tokens > 0 && !a->tree_mask)))
    return invalid(who, "parents need a tree mask");
  if (!a->parents && a->tree_mask_words != 0) return invalid(who, "a tree mask needs parents");
  StepTablesParams p;
  p.lengths = a->lengths;
  p.new_tokens = a->new_tokens;
  p.rows = a->rows;
  p.page_size = a->page_size;
  p.table = a->block_table;
  p.table_stride = a->block_table_stride;
  p.table_cols = a->block_table_cols;
  p.held = a->held;
  p.free_pages = a->free_pages;
  p.free_count = a->free_count;
  p.free_capacity = a->free_capacity;
  p.parents = a->parents;
  p.mask_words = a->parents ? a->tree_mask_words : 0;
  p.tokens = a->tokens;
  p.qo_indptr = a->qo_indptr;
  p.kv_indptr = a->kv_indptr;
  p.kv_len = a->kv_len;
  p.last_page_len = a->last_page_len;
  p.positions = a->positions;
  p.slots = a->slots;
  p.tree_mask = a->tree_mask;
  p.status = a->status;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  int rc = launch(aspire_step_tables_kernel, dim3(1), dim3(kTablesThreads), 0, st, "aspire_step_tables_kernel launch",
                  p);
  if (rc || a->tokens == 0 || a->rows == 0) return rc;
  const int64_t blocks = (a->tokens + kStepTokensThreads - 1) / kStepTokensThreads;
  return launch(aspire_step_tokens_kernel, dim3(unsigned(std::min<int64_t>(blocks, 4096))), dim3(kStepTokensThreads), 0,
                st, "aspire_step_tokens_kernel launch", p);
}

size_t logits_workspace(int64_t tokens, int32_t rows, int32_t vocab, bool bias, int sms) {
  return size_t(tokens) * size_t(slicing(rows, vocab, bias, sms).slices) * 8;
}

int adjust_logits(const AspireLogitsArgs* a, void* stream) {
  const char* who = "aspire_adjust_logits";
  if (!a) return invalid(who, "null argument");
  if (a->type < ASPIRE_T_F32 || a->type > ASPIRE_T_F16) return invalid(who, "type must be ASPIRE_T_F32, _BF16 or _F16");
  if (a->tokens < 0 || a->tokens > INT32_MAX || a->rows < 0 || a->rows > 65534 || a->vocab < 1)
    return invalid(who, "tokens, rows (at most 65534) or vocab out of range");
  if (!a->out && !a->ids) return invalid(who, "neither out nor ids is given");
  if (a->tokens == 0) return ASPIRE_OK;
  if (!a->logits) return invalid(who, "null logits");
  if (a->logits_stride < a->vocab || (a->out && a->out_stride < a->vocab))
    return invalid(who, "rows must be at least vocab apart");
  if (!a->indptr && a->rows != a->tokens) return invalid(who, "without indptr each token is a row of its own");
  if (a->history && (!a->history_len || a->history_cols < 0)) return invalid(who, "history needs history_len");
  if (a->tree_mask && (!a->step_tokens || a->tree_mask_words < 1))
    return invalid(who, "a tree mask needs step_tokens and mask words");
  if (a->bias_indptr && (a->bias_entries < 0 || a->bias_entries >= INT32_MAX ||
                         (a->bias_entries > 0 && (!a->bias_ids || !a->bias_values))))
    return invalid(who, "biases need their ids and values");
  if (a->allowed && a->allowed_stride < (int64_t(a->vocab) + 31) / 32) return invalid(who, "allowed needs a bit per entry");
  int sms = 0;
  int rc = current_sm_count(&sms);
  if (rc) return rc;
  const Slicing cut = slicing(a->rows, a->vocab, a->bias_indptr != nullptr, sms);
  if (a->ids && (!a->workspace || a->workspace_bytes < size_t(a->tokens) * size_t(cut.slices) * 8))
    return set_error(ASPIRE_ERR_CAPACITY, std::string(who) + ": workspace too small");
  LogitsParams p;
  p.logits = a->logits;
  p.logits_stride = a->logits_stride;
  p.out = a->out;
  p.out_stride = a->out_stride;
  p.tokens = a->tokens;
  p.vocab = a->vocab;
  p.rows = a->rows;
  p.indptr = a->indptr;
  p.history = a->history;
  p.history_stride = a->history_stride;
  p.history_cols = a->history_cols;
  p.history_len = a->history_len;
  p.prompt_len = a->prompt_len;
  p.step_tokens = a->step_tokens;
  p.tree_mask = a->tree_mask;
  p.mask_words = a->tree_mask ? a->tree_mask_words : 0;
  p.repetition = a->repetition;
  p.frequency = a->frequency;
  p.presence = a->presence;
  p.bias_indptr = a->bias_indptr;
  p.bias_ids = a->bias_ids;
  p.bias_values = a->bias_values;
  p.bias_entries = a->bias_entries;
  p.allowed = a->allowed;
  p.allowed_stride = a->allowed_stride;
  p.slice = cut.slice;
  p.slices = cut.slices;
  p.best_value = a->ids ? static_cast<float*>(a->workspace) : nullptr;
  p.best_id = a->ids ? static_cast<int32_t*>(a->workspace) + a->tokens * cut.slices : nullptr;
  p.ids = a->ids;
  p.status = a->status;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const bool tail = a->indptr && a->out && a->out != a->logits;
  if (a->rows > 0 || tail) {
    const LogitsKernel kernel = logits_kernel(a->type);
    const size_t smem = slice_bytes(p.slice, p.bias_indptr != nullptr);
    rc = ensure_smem(reinterpret_cast<const void*>(kernel), smem, g_logits_smem[a->type]);
    if (rc) return rc;
    rc = launch(kernel, dim3(unsigned(p.slices), unsigned(p.rows + (tail ? 1 : 0))), dim3(kLogitsThreads), smem, st,
                "aspire_logits_kernel launch", p);
    if (rc) return rc;
  }
  if (!a->ids) return ASPIRE_OK;
  const int64_t per = kPickThreads / 32;
  return launch(aspire_pick_kernel, dim3(unsigned((a->tokens + per - 1) / per)), dim3(kPickThreads), 0, st,
                "aspire_pick_kernel launch", p);
}

int tree_accept(const AspireTreeAcceptArgs* a, void* stream) {
  const char* who = "aspire_tree_accept";
  if (!a) return invalid(who, "null argument");
  if (a->rows < 0 || a->total < 0 || a->total > INT32_MAX) return invalid(who, "rows or total out of range");
  if (a->max_path < 1 || a->max_path > ASPIRE_MAX_PATH) return invalid(who, "max_path must be between 1 and 64");
  if (a->num_caches < 0 || a->num_caches > ASPIRE_MAX_CACHES) return invalid(who, "at most 128 caches a call");
  if (a->rows == 0) return ASPIRE_OK;
  if (!a->indptr || !a->lengths || !a->count || !a->path || !a->out_tokens || !a->new_lengths ||
      (a->total > 0 && (!a->tokens || !a->parents || !a->targets)))
    return invalid(who, "null pointer");
  if (a->new_lengths == a->lengths) return invalid(who, "new_lengths must not be lengths");
  AcceptParams p;
  if (a->num_caches > 0) {
    if (!a->caches || !a->block_table) return invalid(who, "caches need a block table");
    if (a->page_size < 1 || a->block_table_cols < 0 || a->pages < 0) return invalid(who, "bad cache geometry");
    if (a->token_bytes < 16 || a->token_bytes % 16) return invalid(who, "token_bytes must be a positive multiple of 16");
    for (int i = 0; i < a->num_caches; ++i) {
      if (!a->caches[i] || (reinterpret_cast<uintptr_t>(a->caches[i]) & 15))
        return invalid(who, "caches must be 16-byte aligned");
      p.caches[i] = static_cast<char*>(a->caches[i]);
    }
  }
  p.tokens = a->tokens;
  p.parents = a->parents;
  p.targets = a->targets;
  p.indptr = a->indptr;
  p.lengths = a->lengths;
  p.total = a->total;
  p.rows = a->rows;
  p.max_path = a->max_path;
  p.count = a->count;
  p.path = a->path;
  p.out_tokens = a->out_tokens;
  p.new_lengths = a->new_lengths;
  p.table = a->block_table;
  p.table_stride = a->block_table_stride;
  p.table_cols = a->block_table_cols;
  p.page_size = a->page_size;
  p.pages = a->pages;
  p.token_bytes = a->token_bytes;
  p.num_caches = a->num_caches;
  p.status = a->status;
  return launch(aspire_tree_accept_kernel, dim3(unsigned(a->rows), unsigned(std::max(a->num_caches, 1))),
                dim3(kAcceptThreads), 0, static_cast<cudaStream_t>(stream), "aspire_tree_accept_kernel launch", p);
}

}  // namespace
}  // namespace aspire

extern "C" {

int aspire_step_tables(const AspireStepTablesArgs* args, void* stream) {
  return aspire::guarded([&] { return aspire::step_tables(args, stream); });
}

size_t aspire_logits_workspace(int64_t tokens, int32_t rows, int32_t vocab, int32_t with_bias) {
  int sms = 0;
  if (tokens <= 0 || rows < 0 || vocab < 1 || aspire::current_sm_count(&sms)) return 0;
  return aspire::logits_workspace(tokens, rows, vocab, with_bias != 0, sms);
}

int aspire_adjust_logits(const AspireLogitsArgs* args, void* stream) {
  return aspire::guarded([&] { return aspire::adjust_logits(args, stream); });
}

int aspire_tree_accept(const AspireTreeAcceptArgs* args, void* stream) {
  return aspire::guarded([&] { return aspire::tree_accept(args, stream); });
}

}  // extern "C"
