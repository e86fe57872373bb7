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
// aspire_step_tables_kernel: one CTA, 1024 rows at a time; scans in
// registers, then a warp per row for its pages.  Pages are pushed for all
// rows before any is popped, with a CTA barrier between.  The tokens follow
// in aspire_step_tokens_kernel, on the whole grid.
#include "tree.cuh"

namespace aspire {

namespace {

// Exclusive scan of one value per thread over the CTA; *total gets the sum.
__device__ int64_t scan_exclusive(int64_t v, int64_t* warp_sums, int64_t* total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int64_t x = v;
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const int64_t y = __shfl_up_sync(0xffffffffu, x, off);
    if (lane >= off) x += y;
  }
  if (lane == 31) warp_sums[warp] = x;
  __syncthreads();
  if (warp == 0) {
    int64_t w = warp_sums[lane];
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const int64_t y = __shfl_up_sync(0xffffffffu, w, off);
      if (lane >= off) w += y;
    }
    warp_sums[lane] = w;
  }
  __syncthreads();
  const int64_t before = (warp > 0 ? warp_sums[warp - 1] : 0) + x - v;
  *total = warp_sums[31];
  __syncthreads();
  return before;
}

struct RowNeed {
  int32_t len, fresh, want, have;
  bool fits;
};

__device__ __forceinline__ RowNeed row_need(const StepTablesParams& p, int64_t b) {
  RowNeed r;
  r.len = max(p.lengths[b], 0);
  r.fresh = p.new_tokens ? max(p.new_tokens[b], 0) : 0;
  const int64_t end = int64_t(r.len) + r.fresh;
  const int64_t want = (end + p.page_size - 1) / p.page_size;
  r.have = min(max(p.held[b], 0), p.table_cols);
  r.fits = want <= p.table_cols && end <= INT32_MAX && (!p.parents || r.fresh <= 32 * p.mask_words);
  r.want = r.fits ? int32_t(want) : r.have;
  return r;
}

// Row of token t: the last row that starts at or before it and is not empty.
__device__ __forceinline__ int32_t row_of(const int32_t* indptr, int32_t rows, int64_t t) {
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

}  // namespace

__global__ void __launch_bounds__(kTablesThreads) aspire_step_tables_kernel(StepTablesParams p) {
  pdl_begin();
  __shared__ int64_t warp_sums[32];
  __shared__ int32_t at[kTablesThreads];     // first stack place of a row's pages, from the phase's base
  __shared__ int32_t first[kTablesThreads];  // first table column of those
  __shared__ int32_t many[kTablesThreads];   // and how many
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int64_t capacity = p.free_capacity;
  const int64_t count = min(max(int64_t(p.free_count[0]), int64_t(0)), capacity);
  uint32_t bad = 0;

  // Pages past what a row needs.
  int64_t given = 0;
  for (int64_t r0 = 0; r0 < p.rows; r0 += kTablesThreads) {
    const int64_t b = r0 + tid;
    int32_t n = 0;
    if (b < p.rows) {
      const RowNeed r = row_need(p, b);
      n = max(r.have - r.want, 0);
      first[tid] = r.want;
      if (p.lengths[b] < 0 || (p.new_tokens && p.new_tokens[b] < 0) || r.have != p.held[b] || !r.fits)
        bad |= ASPIRE_STATUS_BAD_ROW;
    }
    int64_t total;
    const int64_t before = scan_exclusive(n, warp_sums, &total);
    at[tid] = int32_t(given + before);
    many[tid] = n;
    __syncthreads();
    const int rows = int(min(int64_t(kTablesThreads), p.rows - r0));
    for (int r = warp; total > 0 && r < rows; r += kTablesThreads / 32) {
      int32_t* row = p.table + (r0 + r) * p.table_stride + first[r];
      for (int i = lane; i < many[r]; i += 32) {
        const int64_t place = count + at[r] + i;
        if (place < capacity)
          p.free_pages[place] = row[i];
        else
          bad |= ASPIRE_STATUS_BAD_ROW;  // more pages given back than the pool has
        row[i] = -1;
      }
    }
    given += total;
    __syncthreads();
  }
  const int64_t avail = min(count + given, capacity);

  // How many pages the served rows miss: a running sum that stops at the first row past `avail`.
  int64_t missing = 0, taken = 0;
  for (int64_t r0 = 0; r0 < p.rows; r0 += kTablesThreads) {
    const int64_t b = r0 + tid;
    int32_t n = 0;
    if (b < p.rows) {
      const RowNeed r = row_need(p, b);
      n = max(r.want - r.have, 0);
    }
    int64_t total, served;
    const int64_t upto = missing + scan_exclusive(n, warp_sums, &total) + n;
    scan_exclusive(upto <= avail ? n : 0, warp_sums, &served);
    missing += total;
    taken += served;
  }

  int64_t need = 0, new_at = 0, page_at = 0;
  for (int64_t r0 = 0; r0 < p.rows; r0 += kTablesThreads) {
    const int64_t b = r0 + tid;
    RowNeed r = {};
    int32_t n = 0;
    if (b < p.rows) {
      r = row_need(p, b);
      n = max(r.want - r.have, 0);
    }
    int64_t total;
    const int64_t before = need + scan_exclusive(n, warp_sums, &total);
    need += total;
    const bool served = b < p.rows && r.fits && (n == 0 || before + n <= avail);
    const int32_t pages = served ? r.want : 0;
    int64_t new_total, page_total;
    const int64_t qo = new_at + scan_exclusive(r.fresh, warp_sums, &new_total);
    const int64_t kv = page_at + scan_exclusive(pages, warp_sums, &page_total);
    at[tid] = int32_t(before);
    first[tid] = r.have;
    many[tid] = served ? n : 0;
    if (b < p.rows) {
      if (!served && r.fits) bad |= ASPIRE_STATUS_NO_PAGES;
      const int32_t end = served ? r.len + r.fresh : 0;
      p.qo_indptr[b] = int32_t(qo);
      p.kv_indptr[b] = int32_t(kv);
      p.kv_len[b] = end;
      p.last_page_len[b] = end > 0 ? (end - 1) % p.page_size + 1 : 0;
      p.held[b] = served ? r.want : r.have;
    }
    __syncthreads();
    const int rows = int(min(int64_t(kTablesThreads), p.rows - r0));
    for (int w = warp; total > 0 && w < rows; w += kTablesThreads / 32) {
      int32_t* row = p.table + (r0 + w) * p.table_stride + first[w];
      const int32_t* src = p.free_pages + (avail - taken) + at[w];
      for (int i = lane; i < many[w]; i += 32) row[i] = src[i];
    }
    new_at += new_total;
    page_at += page_total;
    __syncthreads();
  }
  if (tid == 0) {
    p.qo_indptr[p.rows] = int32_t(new_at);
    p.kv_indptr[p.rows] = int32_t(page_at);
    p.free_count[0] = int32_t(avail - taken);
    if (new_at > p.tokens && p.tokens > 0) bad |= ASPIRE_STATUS_BAD_ROW;  // the step's buffers are too short
  }
  if (bad) record_status(p.status, bad);
}

// Positions, slots and ancestor masks, a thread per token.
__global__ void __launch_bounds__(kStepTokensThreads) aspire_step_tokens_kernel(StepTablesParams p) {
  pdl_begin();
  const int64_t total = p.qo_indptr[p.rows];
  const int64_t step = int64_t(gridDim.x) * blockDim.x;
  for (int64_t t = int64_t(blockIdx.x) * blockDim.x + threadIdx.x; t < p.tokens; t += step) {
    int32_t position = 0;
    int64_t slot = -1;
    int32_t* mask = p.tree_mask + t * p.mask_words;
    if (t >= total) {
      for (int w = 0; w < p.mask_words; ++w) mask[w] = 0;
    } else {
      const int32_t b = row_of(p.qo_indptr, p.rows, t);
      const int32_t start = p.qo_indptr[b];
      const int32_t i = int32_t(t - start);
      const int32_t len = max(p.lengths[b], 0);
      int32_t depth = i;
      if (p.parents) {
        // Ancestors have falling indices, so their words fall too: one word at a time, zeros between.
        depth = -1;
        int32_t word = p.mask_words - 1;
        uint32_t bits = 0;
        for (int32_t j = i; j >= 0;) {
          for (; word > (j >> 5); --word) {
            mask[word] = int32_t(bits);
            bits = 0;
          }
          if (word == (j >> 5)) bits |= 1u << (j & 31);  // (nodes past the mask belong to a row that did not fit)
          ++depth;
          const int32_t up = p.parents[start + j];
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
      }
      position = int32_t(min(int64_t(len) + depth, int64_t(INT32_MAX)));
      const int64_t place = int64_t(len) + i;
      if (place < p.kv_len[b]) {
        const int32_t page = p.table[b * p.table_stride + place / p.page_size];
        if (page >= 0) slot = int64_t(page) * p.page_size + place % p.page_size;
      }
    }
    p.positions[t] = position;
    p.slots[t] = slot;
  }
}

}  // namespace aspire
