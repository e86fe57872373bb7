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

SmemOptIn g_mark_smem[2], g_logits_smem[3][2];

int step_tables(const AspireStepTablesArgs* a, void* stream) {
  const char* who = "aspire_step_tables";
  if (!a) return invalid(who, "null argument");
  if (a->rows < 0 || a->tokens < 0 || a->tokens > INT32_MAX) return invalid(who, "rows or tokens out of range");
  if (a->page_size < 1) return invalid(who, "page_size must be > 0");
  if (a->free_capacity < 0 || a->free_capacity > INT32_MAX || a->block_table_cols < 0 || a->block_table_cols >= 1 << 22)
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
  const bool few = a->tokens > 0 && a->tokens <= kFewTokens && a->rows <= kTablesThreads && a->rows > 0;
  int rc = launch(step_tables_kernel(few), dim3(1), dim3(kTablesThreads), 0, st, "aspire_step_tables_kernel launch", p);
  if (rc || few || a->tokens == 0 || a->rows == 0) return rc;
  const int64_t per = int64_t(kStepTokensThreads) * 4;
  return launch(aspire_step_tokens_kernel, dim3(unsigned(std::min<int64_t>((a->tokens + per - 1) / per, 4096))),
                dim3(kStepTokensThreads), 0, st, "aspire_step_tokens_kernel launch", p);
}

// Whether anything touches single entries of the logits.
bool has_marks(const AspireLogitsArgs* a) {
  const bool penalties = a->repetition || a->frequency || a->presence;
  return a->rows > 0 && (a->bias_indptr || (penalties && (a->history || a->step_tokens)));
}

int32_t blocks_of(int32_t vocab) { return int32_t((int64_t(vocab) + kLogitsBlock - 1) / kLogitsBlock); }

// Entries of the marking CTAs' lists.  One lists no more than its row's history,
// tokens and biases, and no more than its own part of the vocabulary: the lists
// lie as the former or, `list_stride` apart, as the latter, whichever is less.
size_t list_entries(const AspireLogitsArgs* a, LogitsParams* p) {
  const size_t ranks = size_t(p->mark_ranks);
  const size_t given = ranks * (size_t(a->rows) * size_t(a->history ? a->history_cols : 0) + size_t(a->tokens) +
                                size_t(a->bias_indptr ? a->bias_entries : 0));
  const size_t share = size_t(p->mark_blocks) * kLogitsBlock, parts = ranks * size_t(a->rows) * share;
  p->list_stride = parts < given ? int32_t(share) : 0;
  return std::min(given, parts);
}

// The workspace's parts, from `base` on; returns their bytes.
size_t lay_out(const AspireLogitsArgs* a, char* base, int sms, LogitsParams* p) {
  // As many marking CTAs a row as the counts need, more for few rows.
  const int cols = a->history ? a->history_cols : 0;
  const int most = cols > kMarkNarrow ? kMarkMaxWide : kMarkMaxBlocks;
  const int all = blocks_of(a->vocab), need = (all + most - 1) / most;
  const int ranks = std::max(need, std::min({8, all, sms / std::max(a->rows, 1)}));
  p->mark_blocks = (all + ranks - 1) / ranks;
  p->mark_ranks = (all + p->mark_blocks - 1) / p->mark_blocks;
  size_t at = 0;
  const auto part = [&](size_t bytes) {
    char* here = base + at;
    at += (bytes + 15) / 16 * 16;
    return here;
  };
  if (a->ids) {
    p->keys = reinterpret_cast<unsigned long long*>(part(size_t(a->tokens) * 8));
    p->arrived = reinterpret_cast<uint32_t*>(part(size_t(a->tokens) * 4));
  }
  if (has_marks(a)) {
    const size_t blocks = size_t(a->rows) * size_t(all);
    const size_t entries = list_entries(a, p);
    p->table = reinterpret_cast<int2*>(part(blocks * (kLogitsBlock / kLogitsUnit) * 8));
    p->touched = reinterpret_cast<uint32_t*>(part(blocks * kLogitsBlock / 8));
    p->list = reinterpret_cast<int2*>(part(entries * 8));
    if (a->bias_indptr) p->list_bias = reinterpret_cast<uint2*>(part(entries * 8));
  }
  return at;
}

int launch_marks(const LogitsParams& p, cudaStream_t st) {
  const bool wide = p.history_cols > kMarkNarrow;
  const size_t smem = p.list ? mark_smem_bytes(p.mark_blocks, wide) : 0;
  const LogitsKernel mark = mark_kernel(wide);
  int rc = ensure_smem(reinterpret_cast<const void*>(mark), smem, g_mark_smem[wide]);
  if (rc) return rc;
  return launch(mark, dim3(unsigned(p.mark_ranks), unsigned(std::max(p.rows, 1))), dim3(kMarkThreads), smem, st,
                "aspire_logits_mark_kernel launch", p);
}

int adjust_logits(const AspireLogitsArgs* a, void* stream) {
  const char* who = "aspire_adjust_logits";
  if (!a) return invalid(who, "null argument");
  if (a->type < ASPIRE_T_F32 || a->type > ASPIRE_T_F16) return invalid(who, "type must be ASPIRE_T_F32, _BF16 or _F16");
  if (a->tokens < 0 || a->tokens > INT32_MAX || a->rows < 0 || a->rows > 65534 || a->vocab < 1)
    return invalid(who, "tokens, rows (at most 65534) or vocab out of range");
  if (!a->out == !a->ids) return invalid(who, "give either out or ids");
  if (a->vocab > 1 << 30) return invalid(who, "vocab must be at most 2^30");
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
  LogitsParams p = {};
  const size_t wanted = lay_out(a, static_cast<char*>(a->workspace), sms, &p);
  if (p.list && list_entries(a, &p) > size_t(INT32_MAX))
    return invalid(who, "histories, tokens and biases past 2^31 entries together");
  if (wanted > 0 && (!a->workspace || a->workspace_bytes < wanted || (reinterpret_cast<uintptr_t>(a->workspace) & 15)))
    return set_error(ASPIRE_ERR_CAPACITY, std::string(who) + ": workspace missing, too small or not 16-byte aligned");
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
  p.history_cols = a->history ? a->history_cols : 0;
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
  p.ids = a->ids;
  p.status = a->status;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (p.list || p.keys) {
    rc = launch_marks(p, st);
    if (rc) return rc;
  }
  // As many CTAs a token as are resident at once.
  const int slice = logits_slice(a->type);
  const int64_t slices = (int64_t(a->vocab) + slice - 1) / slice;
  const int64_t parts = std::max<int64_t>(1, std::min<int64_t>(slices, int64_t(kLogitsCtas) * sms / a->tokens));
  const LogitsKernel kernel = logits_kernel(a->type, a->ids != nullptr);
  rc = ensure_smem(reinterpret_cast<const void*>(kernel), logits_smem_bytes(), g_logits_smem[a->type][a->ids ? 1 : 0]);
  if (rc) return rc;
  return launch(kernel, dim3(unsigned(a->tokens), unsigned(parts)), dim3(kLogitsThreads), logits_smem_bytes(), st,
                "aspire_logits_kernel launch", p);
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
  p.kv_len = a->kv_len;
  // About four CTAs an SM: fewer walk a row's tree more seldom, more have more reads under way.
  int sms = 0;
  const int rc = current_sm_count(&sms);
  if (rc) return rc;
  const int shares = std::max(1, std::min(a->num_caches, (4 * sms + a->rows - 1) / a->rows));
  return launch(aspire_tree_accept_kernel, dim3(unsigned(a->rows), unsigned(shares)), dim3(kAcceptThreads), 0, static_cast<cudaStream_t>(stream), "aspire_tree_accept_kernel launch", p);
}

}  // namespace
}  // namespace aspire

extern "C" {

int aspire_step_tables(const AspireStepTablesArgs* args, void* stream) {
  return aspire::guarded([&] { return aspire::step_tables(args, stream); });
}

size_t aspire_logits_workspace(const AspireLogitsArgs* args) {
  if (!args || args->tokens <= 0 || args->rows < 0 || args->vocab < 1 || args->history_cols < 0 || args->bias_entries < 0)
    return 0;
  aspire::LogitsParams p = {};
  int sms = 0;
  return aspire::current_sm_count(&sms) ? 0 : aspire::lay_out(args, nullptr, sms, &p);
}

int aspire_adjust_logits(const AspireLogitsArgs* args, void* stream) {
  return aspire::guarded([&] { return aspire::adjust_logits(args, stream); });
}

int aspire_tree_accept(const AspireTreeAcceptArgs* args, void* stream) {
  return aspire::guarded([&] { return aspire::tree_accept(args, stream); });
}

}  // extern "C"
