// Block tables and slot maps of a step, from the rows' lengths, with no value
// read back by the host:
//
//   want_b = ceil((len_b + new_b) / page_size)       pages row b needs
//   pages held past want_b go back on the stack of free pages, in row order;
//   missing pages come from the top of the stack: the block of all served
//   rows' missing pages is handed out from its bottom, in row order, so that
//   giving the same pages back leaves the stack as it was;
//   qo_indptr, kv_indptr: prefix sums of new_b and of the pages;
//   token i of row b:  position = len_b + depth_i (i without a tree),
//                      slot = table[b, (len_b + i) / page] * page + (len_b + i) % page,
//                      mask = bit i | mask of its parent.
//
// A row that wants more columns than its table has, more nodes than the mask
// holds, or pages that the stack cannot give (rows are served in order; the
// first that cannot be served ends it) keeps the pages it holds, gets
// kv_len 0 and slots of -1, and the status word says so.
//
// aspire_step_tables_kernel: one CTA, 1024 rows at a time; scans in registers,
// then the rows' pages, a warp for four rows at a time (256 rows of 16 to 64
// pages: 31 us both ways against 36 with one row at a time).  Pages are pushed
// for all rows before any is popped, with a CTA barrier between.  It does the
// tokens too where they are few, one a thread (64 rows of 16 nodes, both ways:
// 20.6 us; four a thread, 22.7), and many are left to aspire_step_tokens_kernel
// on the whole grid.  Both are bound by latency up to some ten thousand tokens,
// by the bytes written beyond.
#include "tree.cuh"

namespace aspire {

namespace {

// Exclusive scan of one value per thread over the CTA; *total gets the sum.
// Consecutive calls use different `warp_sums`.
__device__ uint64_t scan_exclusive(uint64_t v, uint64_t* warp_sums, uint64_t* total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  uint64_t x = v;
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const uint64_t y = __shfl_up_sync(0xffffffffu, x, off);
    if (lane >= off) x += y;
  }
  if (lane == 31) warp_sums[warp] = x;
  __syncthreads();
  uint64_t w = warp_sums[lane];  // every warp sums the warps' sums for itself
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const uint64_t y = __shfl_up_sync(0xffffffffu, w, off);
    if (lane >= off) w += y;
  }
  *total = __shfl_sync(0xffffffffu, w, 31);
  const uint64_t before = __shfl_sync(0xffffffffu, w, max(warp - 1, 0));
  return (warp > 0 ? before : 0) + x - v;
}

// Two counts in one scan (pages: a table has less than 2^22 columns).
__device__ __forceinline__ uint64_t pair(uint32_t lo, uint32_t hi) { return uint64_t(lo) | (uint64_t(hi) << 32); }

struct RowNeed {
  int32_t len, fresh, want, have;
  bool fits, odd;  // odd: an entry out of range, taken as the nearest in it
};

__device__ __forceinline__ RowNeed row_need(const StepTablesParams& p, int64_t b) {
  RowNeed r;
  const int32_t len = p.lengths[b], fresh = p.new_tokens ? p.new_tokens[b] : 0, held = p.held[b];
  r.len = max(len, 0);
  r.fresh = max(fresh, 0);
  const int64_t end = int64_t(r.len) + r.fresh;
  const uint32_t size = uint32_t(p.page_size);
  const int64_t want = uint32_t(end) / size + (uint32_t(end) % size ? 1 : 0);  // (end has 32 bits)
  r.have = min(max(held, 0), p.table_cols);
  r.odd = len < 0 || fresh < 0 || held != r.have;
  r.fits = want <= p.table_cols && end <= INT32_MAX && (!p.parents || r.fresh <= 32 * p.mask_words);
  r.want = r.fits ? int32_t(want) : r.have;
  return r;
}

// Row of token t among `rows` prefix sums.
__device__ __forceinline__ int32_t row_of(const int32_t* indptr, int32_t rows, int32_t t) {
  int32_t lo = 0, hi = rows - 1;
  while (lo < hi) {
    const int32_t mid = (lo + hi) >> 1;
    if (t < indptr[mid + 1])
      hi = mid;
    else
      lo = mid + 1;
  }
  return lo;
}

// The ancestor mask of node i of the tree at `parents`; returns its depth.
__device__ __forceinline__ int32_t ancestors(const StepTablesParams& p, const int32_t* parents, int32_t i, int32_t* mask) {
  // Ancestors have falling indices, so their words fall too: one word at a time, zeros between.
  int32_t depth = -1, word = p.mask_words - 1;
  uint32_t bits = 0;
  for (int32_t j = i; j >= 0;) {
    for (; word > (j >> 5); --word) {
      mask[word] = int32_t(bits);
      bits = 0;
    }
    if (word == (j >> 5)) bits |= 1u << (j & 31);  // (nodes past the mask belong to a row that did not fit)
    ++depth;
    const int32_t up = parents[j];
    if (up >= j || up < -1) {
      record_status(p.status, ASPIRE_STATUS_BAD_ROW);  // not an earlier node: taken as none
      break;
    }
    j = up;
  }
  for (; word >= 0; --word) {
    mask[word] = int32_t(bits);
    bits = 0;
  }
  return depth;
}

// Tokens [t0, t0 + kPer) of the step: positions, slots, masks.  `indptr` are
// the rows' prefix sums, `lens` and `limits` their lengths and keys, `parents`
// the step's, wherever they lie.
template <int kPer>
__device__ __forceinline__ void tokens_of(const StepTablesParams& p, int64_t t0, const int32_t* indptr,
                                          const int32_t* lens, const int32_t* limits, const int32_t* parents, bool wide) {
  const int32_t total = indptr[p.rows];
  int32_t position[kPer];
  int64_t slot[kPer];
  int32_t b = -1, start = 0, end = 0, len = 0, limit = 0;
  int32_t col = -1, page = -1;
#pragma unroll
  for (int k = 0; k < kPer; ++k) {
    const int64_t t = t0 + k;
    position[k] = 0;
    slot[k] = -1;
    if (t >= p.tokens) continue;
    int32_t* mask = p.tree_mask + t * p.mask_words;
    if (t >= total) {
      for (int w = 0; w < p.mask_words; ++w) mask[w] = 0;
      continue;
    }
    if (b < 0 || t >= end) {
      b = row_of(indptr, p.rows, int32_t(t));
      start = indptr[b];
      end = indptr[b + 1];
      len = max(lens[b], 0);
      limit = limits[b];
      col = -1;
    }
    const int32_t i = int32_t(t) - start;
    const int32_t depth = parents ? ancestors(p, parents + start, i, mask) : i;
    position[k] = int32_t(min(int64_t(len) + depth, int64_t(INT32_MAX)));
    const uint32_t place = uint32_t(len) + uint32_t(i);  // (sums past 31 bits have no room: limit is 0)
    if (place < uint32_t(limit)) {
      const uint32_t size = uint32_t(p.page_size), c = place / size;
      if (int32_t(c) != col) {
        col = int32_t(c);
        page = __ldcg(p.table + b * p.table_stride + col);
      }
      if (page >= 0) slot[k] = int64_t(page) * size + (place - c * size);
    }
  }
  if constexpr (kPer == 4) {
    if (wide && t0 + kPer <= p.tokens) {
      *reinterpret_cast<int4*>(p.positions + t0) = make_int4(position[0], position[1], position[2], position[3]);
      *reinterpret_cast<longlong2*>(p.slots + t0) = make_longlong2(slot[0], slot[1]);
      *reinterpret_cast<longlong2*>(p.slots + t0 + 2) = make_longlong2(slot[2], slot[3]);
      return;
    }
  }
#pragma unroll
  for (int k = 0; k < kPer; ++k) {
    if (t0 + k >= p.tokens) break;
    p.positions[t0 + k] = position[k];
    p.slots[t0 + k] = slot[k];
  }
}

// Whether the tokens' tables can be written four at a time.
__device__ __forceinline__ bool wide_tables(const StepTablesParams& p) {
  return ((reinterpret_cast<uintptr_t>(p.positions) | reinterpret_cast<uintptr_t>(p.slots)) & 15) == 0;
}

}  // namespace

namespace {

// Pages of a tile's rows, `many` of each, a warp for kRows rows at a time with
// their loads under way together: f(row, i) is the value of a row's page i,
// g(row, i, value) stores it.
template <int kRows, typename F, typename G>
__device__ __forceinline__ void each_page(const int32_t* many, int rows, F&& f, G&& g) {
  constexpr int kWarps = kTablesThreads / 32, kPages = kRows > 1 ? 2 : 1;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  for (int r0 = warp; r0 < rows; r0 += kRows * kWarps) {
    int more = 0;
    int32_t v[kRows][kPages];
#pragma unroll
    for (int k = 0; k < kRows; ++k) {
      const int r = r0 + k * kWarps, n = r < rows ? many[r] : 0;
      more |= n > 32 * kPages;
#pragma unroll
      for (int u = 0; u < kPages; ++u)
        if (lane + 32 * u < n) v[k][u] = f(r, lane + 32 * u);
    }
#pragma unroll
    for (int k = 0; k < kRows; ++k) {
      const int r = r0 + k * kWarps, n = r < rows ? many[r] : 0;
#pragma unroll
      for (int u = 0; u < kPages; ++u)
        if (lane + 32 * u < n) g(r, lane + 32 * u, v[k][u]);
    }
    if (!more) continue;
    for (int k = 0; k < kRows && r0 + k * kWarps < rows; ++k) {
      const int r = r0 + k * kWarps, n = many[r];
#pragma unroll 4
      for (int i = lane + 32 * kPages; i < n; i += 32) g(r, i, f(r, i));
    }
  }
}

}  // namespace

// kFew: the tokens are done here, one a thread and round.
template <bool kFew>
__global__ void __launch_bounds__(kTablesThreads) aspire_step_tables_kernel(StepTablesParams p) {
  pdl_begin();
  __shared__ uint64_t sums[4][32];
  __shared__ int32_t at[kTablesThreads];     // first stack place of a row's pages, from the phase's base
  __shared__ int32_t first[kTablesThreads];  // first table column of those
  __shared__ int32_t many[kTablesThreads];   // and how many
  __shared__ int32_t taken_s;                // pages of the served rows
  __shared__ int32_t indptr_s[kFew ? kTablesThreads + 1 : 1];
  __shared__ int32_t len_s[kFew ? kTablesThreads : 1], limit_s[kFew ? kTablesThreads : 1];
  __shared__ int32_t parents_s[kFew ? kFewTokens : 1];
  constexpr int kRows = kFew ? 1 : 4;
  const int tid = threadIdx.x;
  const int64_t capacity = min(p.free_capacity, int64_t(INT32_MAX));  // (the count has 32 bits)
  uint32_t bad = 0;
  int32_t parent[kFew ? kFewTokens / kTablesThreads : 1];
  if constexpr (kFew) {  // on their way while the rows are done
#pragma unroll
    for (int k = 0; k < kFewTokens / kTablesThreads; ++k)
      if (p.parents && tid + k * kTablesThreads < p.tokens) parent[k] = p.parents[tid + k * kTablesThreads];
  }
  const int64_t count = min(max(int64_t(p.free_count[0]), int64_t(0)), capacity);
  if (tid == 0) taken_s = 0;
  const bool one_tile = p.rows <= kTablesThreads;
  RowNeed mine = {};  // of the only tile

  // Pages past what the rows need go on the stack; what they miss is summed up.
  int64_t given = 0, missing = 0;
  int64_t need_before = 0;  // of the thread's row (one tile)
  for (int64_t r0 = 0; r0 < p.rows; r0 += kTablesThreads) {
    const int64_t b = r0 + tid;
    int32_t n = 0, need = 0;
    if (b < p.rows) {
      const RowNeed r = row_need(p, b);
      n = max(r.have - r.want, 0);
      need = max(r.want - r.have, 0);
      first[tid] = r.want;
      if (r.odd || !r.fits) bad |= ASPIRE_STATUS_BAD_ROW;
      mine = r;
    }
    uint64_t total;
    const uint64_t before = scan_exclusive(pair(n, need), sums[0], &total);
    at[tid] = int32_t(min(given + int64_t(before & 0xffffffffu), int64_t(INT32_MAX)));
    many[tid] = n;
    need_before = int64_t(before >> 32);
    __syncthreads();
    const int rows = int(min(int64_t(kTablesThreads), p.rows - r0));
    if (total & 0xffffffffu)
      each_page<kRows>(
          many, rows, [&](int r, int i) { return p.table[(r0 + r) * p.table_stride + first[r] + i]; },
          [&](int r, int i, int32_t page) {
            const int64_t place = count + at[r] + i;
            if (place < capacity)
              p.free_pages[place] = page;
            else
              bad |= ASPIRE_STATUS_BAD_ROW;  // more pages given back than the pool has
            p.table[(r0 + r) * p.table_stride + first[r] + i] = -1;
          });
    given += int64_t(total & 0xffffffffu);
    missing += int64_t(total >> 32);
    if (!one_tile) __syncthreads();
  }
  const int64_t avail = min(count + given, capacity);

  // The rows' prefix sums; whose missing pages there are.
  int64_t need = 0, new_at = 0, page_at = 0;
  if (missing > 0 && missing > avail) {  // not all are served: how many pages are
    for (int64_t r0 = 0; r0 < p.rows; r0 += kTablesThreads) {
      const int64_t b = r0 + tid;
      const RowNeed r = b < p.rows ? row_need(p, b) : RowNeed{};
      const int32_t n = max(r.want - r.have, 0);
      uint64_t total;
      const int64_t upto = need + int64_t(scan_exclusive(uint64_t(n), sums[1], &total)) + n;
      if (n > 0 && upto <= avail) atomicMax(&taken_s, int32_t(upto));
      need += int64_t(total);
      __syncthreads();
    }
    need = 0;
  } else if (tid == 0) {
    taken_s = int32_t(missing);
  }
  for (int64_t r0 = 0; r0 < p.rows; r0 += kTablesThreads) {
    const int64_t b = r0 + tid;
    RowNeed r = mine;
    int64_t before = need_before;
    if (!one_tile) {
      r = b < p.rows ? row_need(p, b) : RowNeed{};
      uint64_t total;
      before = need + int64_t(scan_exclusive(uint64_t(max(r.want - r.have, 0)), sums[2], &total));
      need += int64_t(total);
    }
    const int32_t n = max(r.want - r.have, 0);
    const bool served = b < p.rows && r.fits && (n == 0 || before + n <= avail);
    const int32_t pages = served ? r.want : 0;
    uint64_t new_total, page_total;
    const int64_t qo = new_at + int64_t(scan_exclusive(uint64_t(r.fresh), sums[3], &new_total));
    const int64_t kv = page_at + int64_t(scan_exclusive(uint64_t(pages), sums[1], &page_total));
    // (Every thread is past the pages' pushes here, and taken_s is set.)
    if (b < p.rows) {
      if (!served && r.fits) bad |= ASPIRE_STATUS_NO_PAGES;
      const int32_t end = served ? r.len + r.fresh : 0;
      const int32_t start = int32_t(min(qo, int64_t(INT32_MAX)));  // (past the step's buffers in any case)
      p.qo_indptr[b] = start;
      if (kFew) {
        indptr_s[tid] = start;
        len_s[tid] = r.len;
        limit_s[tid] = end;
      }
      p.kv_indptr[b] = int32_t(min(kv, int64_t(INT32_MAX)));
      p.kv_len[b] = end;
      p.last_page_len[b] = end > 0 ? (end - 1) % p.page_size + 1 : 0;
      p.held[b] = served ? r.want : r.have;
    }
    at[tid] = int32_t(before);
    first[tid] = r.have;
    many[tid] = served ? n : 0;
    __syncthreads();
    const int rows = int(min(int64_t(kTablesThreads), p.rows - r0));
    const int32_t* src = p.free_pages + (avail - taken_s);
    if (missing > 0)
      each_page<kRows>(
          many, rows, [&](int r, int i) { return src[at[r] + i]; },
          [&](int r, int i, int32_t page) { p.table[(r0 + r) * p.table_stride + first[r] + i] = page; });
    new_at += int64_t(new_total);
    page_at += int64_t(page_total);
    if (!one_tile) __syncthreads();
  }
  if (tid == 0) {
    p.qo_indptr[p.rows] = int32_t(min(new_at, int64_t(INT32_MAX)));
    if (kFew) indptr_s[p.rows] = int32_t(min(new_at, int64_t(INT32_MAX)));
    p.kv_indptr[p.rows] = int32_t(min(page_at, int64_t(INT32_MAX)));
    p.free_count[0] = int32_t(avail - taken_s);
    if (new_at > p.tokens && p.tokens > 0) bad |= ASPIRE_STATUS_BAD_ROW;  // the step's buffers are too short
  }
  if (bad) record_status(p.status, bad);
  if constexpr (kFew) {
#pragma unroll
    for (int k = 0; k < kFewTokens / kTablesThreads; ++k)
      if (p.parents && tid + k * kTablesThreads < p.tokens) parents_s[tid + k * kTablesThreads] = parent[k];
    __syncthreads();  // (the tables' new pages are written)
    for (int64_t t = tid; t < p.tokens; t += kTablesThreads)
      tokens_of<1>(p, t, indptr_s, len_s, limit_s, p.parents ? parents_s : nullptr, false);
  }
}

TablesKernel step_tables_kernel(bool few) { return few ? &aspire_step_tables_kernel<true> : &aspire_step_tables_kernel<false>; }

// Positions, slots and ancestor masks of many tokens.
__global__ void __launch_bounds__(kStepTokensThreads) aspire_step_tokens_kernel(StepTablesParams p) {
  pdl_begin();
  __shared__ int32_t indptr_s[kTablesThreads + 1];
  const int32_t* indptr = p.qo_indptr;
  if (p.rows <= kTablesThreads) {
    for (int i = threadIdx.x; i <= p.rows; i += kStepTokensThreads) indptr_s[i] = p.qo_indptr[i];
    indptr = indptr_s;
  }
  __syncthreads();
  constexpr int kPer = 4;
  const bool wide = wide_tables(p);
  const int64_t step = int64_t(gridDim.x) * kStepTokensThreads * kPer;
  for (int64_t t = (int64_t(blockIdx.x) * kStepTokensThreads + threadIdx.x) * kPer; t < p.tokens; t += step)
    tokens_of<kPer>(p, t, indptr, p.lengths, p.kv_len, p.parents, wide);
}

}  // namespace aspire
