// Penalties for repeated tokens, biases and grammar masks on the logits of a
// step's tokens, and the best token of the result:
//
//   c = occurrences of v in the row's history behind its prompt
//       + on the token's path (the step's tokens that its mask bits name)
//   x = x / r (x > 0) or x r        when v is in the history or on the path
//   x = x - f c - p [c > 0];  x = x + bias;  x = -inf where not allowed
//   id = the largest x, the lowest v on ties, -1 without any above -inf
//
// in fp32, one rounding per operation (no fused multiply-add, so the values
// are those of the formula step by step), rounded to the logits' type once.
//
// Two kernels.  aspire_logits_mark_kernel finds what each row's history, step
// tokens and biases touch: a few CTAs a row, each for its part of the
// vocabulary, count in shared memory (integer atomics: the order does not
// matter) and write a bitmap and the list of the touched entries in order.
// aspire_logits_kernel or aspire_logits_pick_kernel then streams the logits,
// which bound the call: listed entries are adjusted, all others go by the
// bitmap and the grammar's bits as they came.  Its first loads are on their way
// before the marks are done, but on SMs without a marking CTA only: the 1024
// threads of one have a whole register file, so none of the streaming CTAs fits
// beside it (64 rows of 151936 entries: 128 of 148 SMs).
#include "tree.cuh"

namespace aspire {

namespace {

constexpr uint32_t kInPrompt = 1u << 31;
constexpr uint32_t kInStep = 0x40000000u;  // one of the row's tokens of this step
constexpr uint32_t kBiased = 0x20000000u;  // the row has a bias for it
constexpr uint32_t kCount = 0x1fffffffu;
constexpr int kWarps = kLogitsThreads / 32;

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
template <typename T>
__device__ __forceinline__ T from_float(float v);
template <>
__device__ __forceinline__ float from_float<float>(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }

// Unsigned order of floats that are no NaN (-0 as 0).
__device__ __forceinline__ uint32_t ordered(float f) {
  const uint32_t b = __float_as_uint(f + 0.f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
constexpr uint32_t kOrderedNone = 0x007fffffu;  // ordered(-inf): not chosen
__device__ __forceinline__ float from_ordered(uint32_t o) {
  return __uint_as_float(o & 0x80000000u ? o & 0x7fffffffu : ~o);
}

// Tokens [lo, hi) and biases [from, to) of a row, bounded by the operands'
// sizes whatever the prefix sums say.
struct RowSpan {
  int64_t lo, hi, from, to;
  bool bad;
};
__device__ __forceinline__ RowSpan row_span(const LogitsParams& p, int b) {
  RowSpan s = {b, b + 1, 0, 0, false};
  if (p.indptr) {
    s.lo = p.indptr[b];
    s.hi = p.indptr[b + 1];
    s.bad = s.lo < 0 || s.hi < s.lo || s.hi > p.tokens;
    s.lo = min(max(s.lo, int64_t(0)), p.tokens);
    s.hi = min(max(s.hi, s.lo), p.tokens);
  }
  if (p.bias_indptr) {
    s.from = p.bias_indptr[b];
    s.to = p.bias_indptr[b + 1];
    if (s.from < 0 || s.to < s.from || s.to > p.bias_entries) {
      s.bad = true;
      s.from = min(max(s.from, int64_t(0)), p.bias_entries);
      s.to = s.from;
    }
  }
  return s;
}
// Where a marking CTA's list starts: each has room for the row's whole history,
// tokens and biases, or for its part of the vocabulary.
__device__ __forceinline__ int64_t list_base(const LogitsParams& p, int b, int rank, int ranks, const RowSpan& s) {
  if (p.list_stride) return (int64_t(b) * ranks + rank) * p.list_stride;
  return ranks * (int64_t(b) * p.history_cols + s.lo + s.from) +
         rank * (p.history_cols + (s.hi - s.lo) + (s.to - s.from));
}

// Inclusive sum over the warp's lanes.
__device__ __forceinline__ int warp_scan(int v, int lane) {
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, v, off);
    if (lane >= off) v += y;
  }
  return v;
}

}  // namespace

// What a row touches.  CTA `rank` of the row's takes blocks [rank *
// mark_blocks, ...) of kLogitsBlock entries: it counts the history's tokens
// that are its, flags the prompt's, the step's and the biased ones, sums the
// flags up, a warp 1024 entries at a time, and writes the list.  Counts have
// 16 bits where the history allows (kWide: 32): two CTAs then hold 152000
// entries.  An SM has one of these CTAs at a time, so rows times CTAs past the
// SMs are another wave (with two a row, from 75 rows on).  Bound by the latency of its few steps
// and by its instructions, so what it reads is requested before anything
// waits.  64 rows with histories of up to 16384 over 151936 entries: 19.6 us
// with cold caches; one row with 900 over eight CTAs: 8.7.
template <bool kWide>
__global__ void __launch_bounds__(kMarkThreads, 1) aspire_logits_mark_kernel(LogitsParams p) {
  // (The next kernel reads the logits before it waits for this one, so it may
  // start only when what came before is complete.)
  pdl_wait();
  pdl_launch_dependents();
  constexpr int kGroup = 1024;  // entries of a warp at a time, a word of bits a lane
  constexpr int kGroups = kLogitsBlock / kGroup;
  constexpr int kUnits = kLogitsBlock / kLogitsUnit;
  static_assert(kGroup == 2 * kLogitsUnit, "two units a group");
  constexpr int kWords = kWide ? kGroup : kGroup / 2;  // words of a group's counts
  constexpr int kMarkAhead = 4;                        // of a thread's history tokens, requested at a time
  extern __shared__ __align__(16) uint32_t mark_smem[];
  __shared__ int32_t upto[kMarkMaxBlocks * kGroups];  // touched entries up to the group's end
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int b = blockIdx.y, rank = blockIdx.x, ranks = gridDim.x;
  if (p.keys)
    for (int64_t t = (int64_t(b) * ranks + rank) * kMarkThreads + tid; t < p.tokens;
         t += int64_t(gridDim.y) * ranks * kMarkThreads) {
      p.keys[t] = 0;
      p.arrived[t] = 0;
    }
  if (!p.list) return;  // (nothing to mark)

  const int32_t* h = p.history ? p.history + b * p.history_stride : nullptr;
  int len = 0, prompt = 0;
  if (h) {
    len = p.history_len[b];
    prompt = p.prompt_len ? p.prompt_len[b] : 0;
  }
  const RowSpan span = row_span(p, b);
  len = min(max(len, 0), p.history_cols);
  int32_t ahead[kMarkAhead];
#pragma unroll
  for (int k = 0; k < kMarkAhead; ++k) ahead[k] = tid + k * kMarkThreads < len ? h[tid + k * kMarkThreads] : -1;
  const int32_t step_id = p.step_tokens && span.lo + tid < span.hi ? p.step_tokens[span.lo + tid] : -1;
  const bool has_bias = span.from + tid < span.to;
  const int32_t bias_id = has_bias ? p.bias_ids[span.from + tid] : -1;
  const float bias_value = has_bias ? p.bias_values[span.from + tid] : 0.f;

  const int blocks = (p.vocab + kLogitsBlock - 1) / kLogitsBlock;
  const int32_t v0 = rank * p.mark_blocks * kLogitsBlock;
  const int mine = max(0, min(p.mark_blocks, blocks - rank * p.mark_blocks));
  const int groups = mine * kGroups;
  const int limit = min(mine * kLogitsBlock, p.vocab - v0);
  // Shared memory: counts | prompt | step | biased | all of them | their sums.
  uint32_t* count = mark_smem;
  const int flag_words = p.mark_blocks * (kLogitsBlock / 32);
  uint32_t* in_prompt = count + p.mark_blocks * kGroups * kWords;
  uint32_t* in_step = in_prompt + flag_words;
  uint32_t* biased = in_step + flag_words;
  uint32_t* bits = biased + flag_words;
  uint16_t* start = reinterpret_cast<uint16_t*>(bits + flag_words);  // touched entries of a group before the word
  {
    const int words = p.mark_blocks * kGroups * kWords + 4 * flag_words;
    for (int i = tid; i < words / 4; i += kMarkThreads) reinterpret_cast<uint4*>(count)[i] = make_uint4(0, 0, 0, 0);
  }
  __syncthreads();
  // (16 bits: an entry shares its word with the one 512 places on or back.)
  const auto word_of = [](int e) { return kWide ? e : (e / kGroup) * kWords + (e & (kWords - 1)); };
  const auto shift_of = [](int e) { return !kWide && (e & kWords) ? 16 : 0; };
  const auto flag = [](uint32_t* a, int e) { atomicOr(&a[e >> 5], 1u << (e & 31)); };
  const auto inside = [&](int32_t v) { return uint32_t(v) - uint32_t(v0) < uint32_t(max(limit, 0)); };
  // Tokens behind the prompt are counted and flagged among all, the prompt's are flagged.
  const auto note = [&](int i, int32_t v) {
    if (!inside(v)) return;
    const int e = v - v0;
    flag(i < prompt ? in_prompt : bits, e);
    if (i >= prompt) atomicAdd(&count[word_of(e)], 1u << shift_of(e));
  };
#pragma unroll 1
  for (int i = tid; i < len; i += kMarkAhead * kMarkThreads) {
    int32_t now[kMarkAhead];
#pragma unroll
    for (int k = 0; k < kMarkAhead; ++k) {
      now[k] = ahead[k];
      const int at = i + (kMarkAhead + k) * kMarkThreads;
      ahead[k] = at < len ? h[at] : -1;
    }
#pragma unroll
    for (int k = 0; k < kMarkAhead; ++k) note(i + k * kMarkThreads, now[k]);
  }
  if (inside(step_id)) flag(in_step, step_id - v0);
  if (p.step_tokens)
    for (int64_t t = span.lo + tid + kMarkThreads; t < span.hi; t += kMarkThreads)
      if (inside(p.step_tokens[t])) flag(in_step, p.step_tokens[t] - v0);
  if (inside(bias_id)) flag(biased, bias_id - v0);
  for (int64_t i = span.from + tid + kMarkThreads; i < span.to; i += kMarkThreads)
    if (inside(p.bias_ids[i])) flag(biased, p.bias_ids[i] - v0);
  __syncthreads();

  uint32_t* touched = p.touched + (int64_t(b) * blocks + int64_t(rank) * p.mark_blocks) * (kLogitsBlock / 32);
  for (int g = warp; g < groups; g += kMarkThreads / 32) {
    const int at = g * 32 + lane;
    const uint32_t word = bits[at] | in_prompt[at] | in_step[at] | biased[at];
    bits[at] = word;
    touched[at] = word;
    const int end = warp_scan(__popc(word), lane);
    start[at] = uint16_t(end - __popc(word));
    if (lane == 31) upto[g] = end;
  }
  __syncthreads();
  if (warp == 0) {
    int carry = 0;
    for (int g0 = 0; g0 < groups; g0 += 32) {
      const int sum = carry + warp_scan(g0 + lane < groups ? upto[g0 + lane] : 0, lane);
      if (g0 + lane < groups) upto[g0 + lane] = sum;
      carry = __shfl_sync(0xffffffffu, sum, 31);
    }
  }
  __syncthreads();
  const int64_t base = list_base(p, b, rank, ranks, span);
  int2* table = p.table + (int64_t(b) * blocks + rank * p.mark_blocks) * kUnits;
  for (int u = tid; u < mine * kUnits; u += kMarkThreads) {
    const int before = int(base) + (u >= 2 ? upto[u / 2 - 1] : 0);  // (the list has less than 2^31 entries)
    const int middle = int(base) + (u / 2 > 0 ? upto[u / 2 - 1] : 0) + start[(u | 1) * (kLogitsUnit / 32)];
    table[u] = u & 1 ? make_int2(middle, int(base) + upto[u / 2]) : make_int2(before, middle);
  }
  // The list: a lane writes the entries of half a word, 512 entries a warp at a
  // time (the most frequent tokens crowd in a few words).
  for (int u = warp; u < 2 * groups; u += kMarkThreads / 32) {
    const int w = u * 16 + (lane & 15), g = u >> 1;
    const uint32_t word = bits[w], prompts = in_prompt[w], steps = in_step[w], biases = biased[w];
    const int64_t at = base + (g > 0 ? upto[g - 1] : 0) + start[w];
    int2* list = p.list + at;
    uint2* list_bias = p.list_bias + at;
    const uint32_t rare = steps | biases;
#pragma unroll 1
    for (uint32_t left = word & (lane < 16 ? 0xffffu : 0xffff0000u); left; left &= left - 1) {
      const int bit = __ffs(int(left)) - 1, e = w * 32 + bit;
      uint32_t c = count[word_of(e)];
      if constexpr (!kWide) c = (c >> shift_of(e)) & 0xffffu;
      c |= (prompts >> bit) << 31;
      const int to = __popc(word & ((1u << bit) - 1));
      if ((rare >> bit) & 1) {
        c |= ((steps >> bit) & 1 ? kInStep : 0u) | ((biases >> bit) & 1 ? kBiased : 0u);
        if (c & kBiased) list_bias[to].x = 0;
      }
      list[to] = make_int2(v0 + e, int32_t(c));
    }
  }
  if (span.to > span.from) {
    const auto place = [&](int e) {  // in the CTA's list
      const int g = e / kGroup, w = e / 32;
      return (g > 0 ? upto[g - 1] : 0) + start[w] + __popc(bits[w] & ((1u << (e & 31)) - 1));
    };
    const auto each = [&](const auto& f) {  // f(entry, its id, its bias) of the CTA's
      if (inside(bias_id)) f(span.from + tid, bias_id, bias_value);
      for (int64_t i = span.from + tid + kMarkThreads; i < span.to; i += kMarkThreads)
        if (inside(p.bias_ids[i])) f(i, p.bias_ids[i], p.bias_values[i]);
    };
    __syncthreads();
    each([&](int64_t i, int32_t v, float) {  // of a token listed twice, the later entry
      atomicMax(&p.list_bias[base + place(v - v0)].x, uint32_t(i) + 1);
    });
    __syncthreads();
    each([&](int64_t i, int32_t v, float value) {
      uint2* to = p.list_bias + base + place(v - v0);
      if (__ldcg(&to->x) == uint32_t(i) + 1) to->y = __float_as_uint(value);
    });
  }
  if (span.bad && tid == 0 && rank == 0) record_status(p.status, ASPIRE_STATUS_BAD_ROW);
}

LogitsKernel mark_kernel(bool wide) { return wide ? &aspire_logits_mark_kernel<true> : &aspire_logits_mark_kernel<false>; }

namespace {

// The row of token t, -1 for none; the same in all lanes of the warp.
__device__ __forceinline__ int row_of_token(const LogitsParams& p, int64_t t, int lane) {
  if (!p.indptr) return t < p.rows ? int(t) : -1;
  if (p.rows == 0 || t < p.indptr[0] || t >= p.indptr[p.rows]) return -1;
  int lo = 0, n = p.rows;
  while (n > 1) {
    const int step = (n + 31) / 32;
    const int last = min((lane + 1) * step, n);  // the first `last` rows end after t?
    const uint32_t after = __ballot_sync(0xffffffffu, t < p.indptr[lo + last]);
    const int k = after ? __ffs(int(after)) - 1 : 31;
    lo += k * step;
    n = max(1, min(step, n - k * step));
  }
  return min(lo, p.rows - 1);
}

// How often id v of each lane that asks is among the tokens on t's path.
__device__ __forceinline__ int on_path(const LogitsParams& p, const RowSpan& s, int64_t t, bool ask, int32_t v,
                                       int lane) {
  const int64_t end = p.tree_mask ? min(s.hi, s.lo + 32 * int64_t(p.mask_words)) : t + 1;
  int made = 0;
  for (uint32_t left = __ballot_sync(0xffffffffu, ask); left; left &= left - 1) {
    const int who = __ffs(int(left)) - 1;
    const int32_t want = __shfl_sync(0xffffffffu, v, who);
    int sum = 0;
    for (int64_t j0 = s.lo; j0 < end; j0 += 32) {
      const int64_t j = j0 + lane;
      bool hit = j < end && p.step_tokens[j] == want;
      if (p.tree_mask)
        hit = hit && ((uint32_t(p.tree_mask[t * p.mask_words + ((j0 - s.lo) >> 5)]) >> lane) & 1);
      sum += __popc(__ballot_sync(0xffffffffu, hit));
    }
    if (lane == who) made = sum;
  }
  return made;
}

// The largest of a lane's first `many` vectors' entries, whatever their bits; a NaN is never the largest.
constexpr int kMany = 4;  // vectors of a lane
__device__ __forceinline__ float largest(const uint4* raw, int many, float) {
  float f = -INFINITY;
#pragma unroll
  for (int j = 0; j < kMany; ++j)
    if (j < many)
      f = fmaxf(fmaxf(fmaxf(f, __uint_as_float(raw[j].x)), fmaxf(__uint_as_float(raw[j].y), __uint_as_float(raw[j].z))),
                __uint_as_float(raw[j].w));
  return f;
}
template <typename T2, typename T>
__device__ __forceinline__ float largest2(const uint4* raw, int many, T2 none) {
  T2 m = none;
#pragma unroll
  for (int j = 0; j < kMany; ++j)
    if (j < many) {
      const T2* x = reinterpret_cast<const T2*>(&raw[j]);
      m = __hmax2(m, __hmax2(__hmax2(x[0], x[1]), __hmax2(x[2], x[3])));
    }
  return fmaxf(fmaxf(to_float(m.x), to_float(m.y)), -INFINITY);
}
__device__ __forceinline__ float largest(const uint4* raw, int many, __nv_bfloat16 none) {
  return largest2<__nv_bfloat162, __nv_bfloat16>(raw, many, __nv_bfloat162(none, none));
}
__device__ __forceinline__ float largest(const uint4* raw, int many, __half none) {
  return largest2<__half2, __half>(raw, many, __half2(none, none));
}

// Bits of a warp's words (word `lane` each) from bit `at` on, as many as a
// vector has entries.
template <int kVec>
__device__ __forceinline__ uint32_t vector_bits(uint32_t words, int at) {
  const uint32_t lo = __shfl_sync(0xffffffffu, words, at >> 5);
  const uint32_t hi = __shfl_sync(0xffffffffu, words, (at >> 5) + 1);
  return __funnelshift_r(lo, hi, at & 31) & ((1u << kVec) - 1);
}

__device__ __forceinline__ void copy_async(void* to, const void* from) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(static_cast<uint32_t>(__cvta_generic_to_shared(to))),
               "l"(from)
               : "memory");
}

// A warp's way through a token's logits: chunks of kMany 16-byte vectors a
// lane, whole vectors of the logits' memory, copied to shared memory kAhead
// chunks ahead, and up to 16 / sizeof(T) entries before and behind them, one a
// lane.  Warp w of CTA y takes chunks 8 y + w, + 8 gridDim.y, ...
constexpr int kAhead = 3;
template <typename T>
struct Walk {
  static constexpr int kVec = 16 / int(sizeof(T));
  static constexpr int kChunk = kMany * 32 * kVec;
  static constexpr int kStage = kChunk * int(sizeof(T)) + 16;  // entry e at pad + e: vectors stay aligned
  static constexpr int kUnits = kChunk / kLogitsUnit;
  static_assert(kChunk % kLogitsUnit == 0, "a chunk is whole units of the marks");
  using Stages = uint8_t[kWarps][kAhead + 1][kStage];

  const T* logits;
  int vocab, pad, lane;  // pad: entries of the logits' first 16 bytes that are not theirs
  int chunk, step, chunks;
  uint8_t (*stages)[kStage];
  int slot;
  T next_edge;

  // The chunk's entries: n, of them `head` before the vectors, `edges` outside them.
  struct Part {
    int n, head, vectors, edges, edge_at;
  };
  __device__ __forceinline__ Part part(int c) const {
    Part a = {kChunk, 0, kChunk / kVec, 0, 0};
    if (pad == 0 && vocab - c * kChunk >= kChunk) return a;
    a.n = min(kChunk, vocab - c * kChunk);
    a.head = min(a.n, (kVec - pad) & (kVec - 1));
    a.vectors = (a.n - a.head) / kVec;
    a.edges = a.n - a.vectors * kVec;
    a.edge_at = lane < a.edges ? (lane < a.head ? lane : lane + a.vectors * kVec) : 0;
    return a;
  }
  __device__ __forceinline__ T* stage() const { return reinterpret_cast<T*>(stages[slot]) + pad; }
  // Requests chunk c for the slot that comes `ahead` after the current one.
  __device__ __forceinline__ void request(int c, int ahead) {
    if (c < chunks) {
      const Part a = part(c);
      uint8_t* to = stages[(slot + ahead) & kAhead] + (pad + a.head) * int(sizeof(T));
      const T* from = logits + c * kChunk + a.head;
#pragma unroll
      for (int j = 0; j < kMany; ++j)
        if (lane + 32 * j < a.vectors) copy_async(to + (lane + 32 * j) * 16, from + (lane + 32 * j) * kVec);
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  }
  __device__ __forceinline__ void request_edge(int c) {
    if (c >= chunks) return;
    const Part a = part(c);
    if (lane < a.edges) next_edge = logits[c * kChunk + a.edge_at];
  }
  __device__ __forceinline__ Walk(const LogitsParams& p, int64_t t, Stages& all)
      : logits(static_cast<const T*>(p.logits) + t * p.logits_stride), vocab(p.vocab),
        pad(int(reinterpret_cast<uintptr_t>(logits) & 15) / int(sizeof(T))), lane(threadIdx.x & 31),
        chunk(blockIdx.y * kWarps + (threadIdx.x >> 5)), step(gridDim.y * kWarps),
        chunks((p.vocab + kChunk - 1) / kChunk), stages(all[threadIdx.x >> 5]), slot(0) {
#pragma unroll
    for (int k = 0; k < kAhead; ++k) request(chunk + k * step, k);
    request_edge(chunk);
  }
  // The current chunk is staged, its edges too if it has any.
  __device__ __forceinline__ Part arrive() {
    asm volatile("cp.async.wait_group %0;" ::"n"(kAhead - 1) : "memory");
    const Part a = part(chunk);
    if (lane < a.edges) stage()[a.edge_at] = next_edge;
    __syncwarp();
    request(chunk + kAhead * step, kAhead);
    request_edge(chunk + step);
    return a;
  }
  __device__ __forceinline__ void advance() {
    __syncwarp();  // (what is staged there has been read)
    slot = (slot + 1) & kAhead;
    chunk += step;
  }
};
static_assert(((kAhead + 1) & kAhead) == 0, "the slots are counted modulo a power of two");

// A token's row: its terms and its list, of which a warp takes a chunk's part
// at a time.  The parts of 32 chunks are read at once, a lane each.
struct Listed {
  RowSpan span = {};
  const int2* list = nullptr;
  const uint2* bias = nullptr;
  const uint32_t* touched = nullptr;
  const int2* table = nullptr;
  float repetition = 1.f, frequency = 0.f, presence = 0.f;
  bool repeat = false;
  int from = 0, to = 0;  // lane i: the list's part of the warp's chunk i of 32

  // (Reads inputs only, nothing that the marks write.)
  __device__ __forceinline__ void open(const LogitsParams& p, int row) {
    const int64_t blocks = (p.vocab + kLogitsBlock - 1) / kLogitsBlock;
    table = p.table + row * blocks * (kLogitsBlock / kLogitsUnit);
    span = row_span(p, row);
    list = p.list;
    bias = p.list_bias;
    touched = p.touched + row * blocks * (kLogitsBlock / 32);
    repeat = p.repetition != nullptr;
    repetition = repeat ? p.repetition[row] : 1.f;
    frequency = p.frequency ? p.frequency[row] : 0.f;
    presence = p.presence ? p.presence[row] : 0.f;
  }
  template <typename T>
  __device__ __forceinline__ void look_ahead(const Walk<T>& w) {
    const int c = w.chunk + w.lane * w.step;
    if (c < w.chunks) {
      from = table[c * Walk<T>::kUnits].x;
      to = table[(c + 1) * Walk<T>::kUnits - 1].y;
    }
  }
  // The adjusted logit of an entry with these flags that is on the path `path` times.
  __device__ __forceinline__ float adjusted(float x, uint32_t flags, int path, float own_bias) const {
    const int made = int(flags & kCount) + path;
    if (repeat && (made > 0 || (flags & kInPrompt)))
      x = x > 0.f ? __fdiv_rn(x, repetition) : __fmul_rn(x, repetition);
    if (made > 0) {
      x = __fsub_rn(x, __fmul_rn(frequency, float(made)));
      x = __fsub_rn(x, presence);
    }
    return flags & kBiased ? __fadd_rn(x, own_bias) : x;
  }
};

}  // namespace

// The adjusted logits of token blockIdx.x.  The warps work on their own: no
// barrier, three chunks of each on their way while it adjusts the listed
// entries of one where they lie, in shared memory.  64 rows of 151936 fp32
// logits with some 4 to 16 thousand entries listed each: 23.6 us for 78 MB; both
// kernels in a graph 37.
template <typename T>
__global__ void __launch_bounds__(kLogitsThreads, kLogitsCtas) aspire_logits_kernel(LogitsParams p) {
  using W = Walk<T>;
  extern __shared__ __align__(16) uint8_t logits_stages[];
  const int lane = threadIdx.x & 31;
  const int64_t t = blockIdx.x;
  if (!p.list) pdl_begin();  // (nothing is marked: the logits may come from the kernel before)
  W w(p, t, *reinterpret_cast<typename W::Stages*>(logits_stages));
  const int row = row_of_token(p, t, lane);
  const uint32_t* allowed =
      p.allowed && row >= 0 ? reinterpret_cast<const uint32_t*>(p.allowed) + t * p.allowed_stride : nullptr;
  const auto grammar = [&](int c) {
    return allowed && c < w.chunks && 32 * lane < min(W::kChunk, p.vocab - c * W::kChunk)
               ? __ldcs(allowed + c * (W::kChunk / 32) + lane)
               : 0xffffffffu;
  };
  uint32_t next_ok = grammar(w.chunk);
  if (!p.list && blockIdx.y == 0 && threadIdx.x == 0 && row >= 0 && row_span(p, row).bad)
    record_status(p.status, ASPIRE_STATUS_BAD_ROW);  // (else the marks say so)
  Listed r;
  const bool listed = p.list && row >= 0;
  if (listed) r.open(p, row);
  if (p.list) {
    pdl_wait();
    pdl_launch_dependents();
  }
  if (listed) r.look_ahead(w);
  constexpr int kBatch = 4;  // listed entries of a lane on their way: a chunk of frequent tokens has hundreds
  int2 entry[kBatch];
  float bias[kBatch];
  const auto fetch = [&](int i, int end) {
#pragma unroll
    for (int k = 0; k < kBatch; ++k) {
      entry[k] = i + 32 * k < end ? r.list[i + 32 * k] : make_int2(0, 0);
      bias[k] = r.bias && i + 32 * k < end ? __uint_as_float(r.bias[i + 32 * k].y) : 0.f;
    }
  };
  if (listed) fetch(__shfl_sync(0xffffffffu, r.from, 0) + lane, __shfl_sync(0xffffffffu, r.to, 0));

  for (int it = 0; w.chunk < w.chunks; ++it) {
    const typename W::Part a = w.arrive();
    const uint32_t ok = next_ok;
    next_ok = grammar(w.chunk + w.step);
    T* stage = w.stage();
    if (listed) {
      const int begin = __shfl_sync(0xffffffffu, r.from, it & 31), end = __shfl_sync(0xffffffffu, r.to, it & 31);
      for (int i0 = begin; i0 < end; i0 += 32 * kBatch) {
        int2 now[kBatch];
        float own[kBatch];
#pragma unroll
        for (int k = 0; k < kBatch; ++k) {
          now[k] = entry[k];
          own[k] = bias[k];
        }
        if (i0 + 32 * kBatch < end) fetch(i0 + 32 * kBatch + lane, end);
#pragma unroll
        for (int k = 0; k < kBatch; ++k) {
          if (i0 + 32 * k >= end) break;
          const uint32_t flags = uint32_t(now[k].y);
          int path = 0;
          if (__any_sync(0xffffffffu, (flags & kInStep) != 0))
            path = on_path(p, r.span, t, (flags & kInStep) != 0, now[k].x, lane);
          // (Rows that overlap share their lists' memory: an entry may be another row's.)
          const int32_t e = now[k].x - w.chunk * W::kChunk;
          if (i0 + 32 * k + lane < end && uint32_t(e) < uint32_t(a.n)) {
            T* x = stage + e;
            *x = from_float<T>(r.adjusted(to_float(*x), flags, path, own[k]));
          }
        }
      }
      __syncwarp();
      if ((it & 31) == 31) {
        W ahead = w;
        ahead.chunk += w.step;
        r.look_ahead(ahead);
      }
      const int next = (it + 1) & 31;
      if (w.chunk + w.step < w.chunks)
        fetch(__shfl_sync(0xffffffffu, r.from, next) + lane, __shfl_sync(0xffffffffu, r.to, next));
    }

    T* dst = static_cast<T*>(p.out) + t * p.out_stride + w.chunk * W::kChunk;
    const bool wide_out = ((reinterpret_cast<uintptr_t>(dst + a.head) & 15) == 0);
#pragma unroll
    for (int j = 0; j < kMany; ++j) {
      const int at = a.head + (lane + 32 * j) * W::kVec;
      uint4 raw = make_uint4(0, 0, 0, 0);
      if (lane + 32 * j < a.vectors) raw = *reinterpret_cast<const uint4*>(stage + at);
      T* x = reinterpret_cast<T*>(&raw);
      if (allowed) {
        const uint32_t bits = vector_bits<W::kVec>(ok, at);
#pragma unroll
        for (int k = 0; k < W::kVec; ++k)
          if (!((bits >> k) & 1)) x[k] = from_float<T>(-INFINITY);
      }
      if (lane + 32 * j < a.vectors) {
        if (wide_out) {
          __stcs(reinterpret_cast<uint4*>(dst + at), raw);
        } else {
#pragma unroll
          for (int k = 0; k < W::kVec; ++k) dst[at + k] = x[k];
        }
      }
    }
    if (a.edges > 0) {
      const bool pass = (__shfl_sync(0xffffffffu, ok, a.edge_at >> 5) >> (a.edge_at & 31)) & 1;
      if (lane < a.edges) dst[a.edge_at] = pass ? stage[a.edge_at] : from_float<T>(-INFINITY);
    }
    w.advance();
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
}

// The best token of blockIdx.x's, by the same walk.  A chunk is looked into,
// with its grammar and mark bits, only where an entry reaches the bar, the
// best that the CTA has found; its listed entries, if a listed one does, or if
// a bias or the row's penalties can raise one.  The CTAs of a token meet as
// 64-bit keys (value, then lowest id), and the last one writes the id.
template <typename T>
__global__ void __launch_bounds__(kLogitsThreads, kLogitsCtas) aspire_logits_pick_kernel(LogitsParams p) {
  using W = Walk<T>;
  extern __shared__ __align__(16) uint8_t logits_stages[];
  __shared__ unsigned long long key;
  __shared__ uint32_t shared_bar;  // ordered()
  const int lane = threadIdx.x & 31;
  const int64_t t = blockIdx.x;
  if (!p.list) pdl_begin();  // (nothing is marked: the logits may come from the kernel before)
  W w(p, t, *reinterpret_cast<typename W::Stages*>(logits_stages));
  const int row = row_of_token(p, t, lane);
  const uint32_t* allowed =
      p.allowed && row >= 0 ? reinterpret_cast<const uint32_t*>(p.allowed) + t * p.allowed_stride : nullptr;
  // (The first chunk is looked into for sure.)
  const uint32_t first_ok =
      allowed && w.chunk < w.chunks && 32 * lane < min(W::kChunk, p.vocab - w.chunk * W::kChunk)
          ? allowed[w.chunk * (W::kChunk / 32) + lane]
          : 0xffffffffu;
  if (threadIdx.x == 0) {
    key = 0;
    shared_bar = kOrderedNone;
  }
  if (!p.list && blockIdx.y == 0 && threadIdx.x == 0 && row >= 0 && row_span(p, row).bad)
    record_status(p.status, ASPIRE_STATUS_BAD_ROW);  // (else the marks say so)
  Listed r;
  const bool listed = p.list && row >= 0;
  if (listed) r.open(p, row);
  if (p.list) {
    pdl_wait();
    pdl_launch_dependents();
  }
  if (listed) r.look_ahead(w);
  // Whether a listed entry may end up above what it came with.
  const bool raises = listed && (!(r.repetition >= 1.f && r.frequency >= 0.f && r.presence >= 0.f) ||
                                 r.span.to > r.span.from);
  __syncthreads();

  float best = -INFINITY;  // the lane's best, and its id
  int32_t id = INT32_MAX;
  float bar = -INFINITY;
  const auto better = [&](float x, int32_t v) {
    if (x > best || (x == best && x > -INFINITY && v < id)) {
      best = x;
      id = v;
    }
  };
  const auto raise_bar = [&]() {
    const uint32_t top = __reduce_max_sync(0xffffffffu, ordered(best));
    if (lane == 0) atomicMax(&shared_bar, top);
    bar = fmaxf(bar, from_ordered(top));
  };
  for (int it = 0; row >= 0 && w.chunk < w.chunks; ++it) {
    const typename W::Part a = w.arrive();
    const T* stage = w.stage();
    const int v0 = w.chunk * W::kChunk;
    const int many = max(0, min(kMany, (a.vectors - lane + 31) / 32));
    uint4 raw[kMany];
#pragma unroll
    for (int j = 0; j < kMany; ++j)
      if (j < many) raw[j] = *reinterpret_cast<const uint4*>(stage + a.head + (lane + 32 * j) * W::kVec);
    const float edge = lane < a.edges ? to_float(stage[a.edge_at]) : -INFINITY;
    const float most = fmaxf(largest(raw, many, from_float<T>(-INFINITY)), edge);
    bar = fmaxf(bar, from_ordered(*reinterpret_cast<volatile uint32_t*>(&shared_bar)));
    const int begin = __shfl_sync(0xffffffffu, r.from, it & 31), end = __shfl_sync(0xffffffffu, r.to, it & 31);
    bool look = raises && end > begin;
    if (__any_sync(0xffffffffu, most >= bar && most > -INFINITY)) {
      uint32_t ok = 0xffffffffu, touched = 0;
      if (32 * lane < a.n) {
        if (allowed) ok = it == 0 ? first_ok : allowed[v0 / 32 + lane];
        if (end > begin) touched = r.touched[v0 / 32 + lane];
      }
      const float old = bar;
      float listed_most = -INFINITY;
#pragma unroll
      for (int j = 0; j < kMany; ++j) {
        const int at = a.head + (lane + 32 * j) * W::kVec;
        const uint32_t bits = vector_bits<W::kVec>(ok, at), marked = vector_bits<W::kVec>(touched, at);
        const T* x = reinterpret_cast<const T*>(&raw[j]);
        if (j < many && most >= old) {
#pragma unroll
          for (int k = 0; k < W::kVec; ++k) {
            const float f = to_float(x[k]);
            if (!((bits >> k) & 1) || !(f >= old)) continue;
            if ((marked >> k) & 1)
              listed_most = fmaxf(listed_most, f);
            else
              better(f, v0 + at + k);
          }
        }
      }
      const uint32_t edge_ok = __shfl_sync(0xffffffffu, ok, a.edge_at >> 5) >> (a.edge_at & 31) & 1;
      const uint32_t edge_marked = __shfl_sync(0xffffffffu, touched, a.edge_at >> 5) >> (a.edge_at & 31) & 1;
      if (lane < a.edges && edge_ok) {
        if (edge_marked)
          listed_most = fmaxf(listed_most, edge);
        else
          better(edge, v0 + a.edge_at);
      }
      raise_bar();
      look |= __any_sync(0xffffffffu, listed_most >= bar && listed_most > -INFINITY) != 0;
    }
    if (look) {
      constexpr int kBatch = 4;  // entries of a lane requested together
      for (int i0 = begin; i0 < end; i0 += 32 * kBatch) {
        int2 entry[kBatch];
#pragma unroll
        for (int k = 0; k < kBatch; ++k) {
          const int i = i0 + 32 * k + lane;
          entry[k] = i < end ? r.list[i] : make_int2(0, 0);
        }
#pragma unroll
        for (int k = 0; k < kBatch; ++k) {
          const int i = i0 + 32 * k + lane;
          if (i0 + 32 * k >= end) break;
          const int32_t v = entry[k].x;
          const bool here = i < end && uint32_t(v - v0) < uint32_t(a.n);  // (rows that overlap share their lists' memory)
          const float x = here ? to_float(stage[v - v0]) : -INFINITY;
          const bool live = here && (raises || x >= bar) && (!allowed || ((allowed[v >> 5] >> (v & 31)) & 1));
          const uint32_t flags = live ? uint32_t(entry[k].y) : 0u;
          if (!__any_sync(0xffffffffu, live)) continue;
          int path = 0;
          if (__any_sync(0xffffffffu, (flags & kInStep) != 0))
            path = on_path(p, r.span, t, (flags & kInStep) != 0, v, lane);
          if (live) better(r.adjusted(x, flags, path, flags & kBiased ? __uint_as_float(r.bias[i].y) : 0.f), v);
        }
      }
      raise_bar();
    }
    if (listed && (it & 31) == 31) {
      W ahead = w;
      ahead.chunk += w.step;
      r.look_ahead(ahead);
    }
    w.advance();
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");

  const uint32_t top = __reduce_max_sync(0xffffffffu, ordered(best));
  if (top > kOrderedNone) {
    const uint32_t mine = __reduce_min_sync(0xffffffffu, ordered(best) == top ? uint32_t(id) : 0xffffffffu);
    if (lane == 0) atomicMax(&key, ((unsigned long long)top << 32) | (0xffffffffu - mine));
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    if (gridDim.y == 1) {
      p.ids[t] = key ? int32_t(0xffffffffu - uint32_t(key)) : -1;
      return;
    }
    if (key) atomicMax(&p.keys[t], key);
    __threadfence();
    if (atomicAdd(&p.arrived[t], 1u) == gridDim.y - 1) {
      __threadfence();
      const unsigned long long k = atomicMax(&p.keys[t], 0ull);
      p.ids[t] = k ? int32_t(0xffffffffu - uint32_t(k)) : -1;
    }
  }
}

LogitsKernel logits_kernel(int type, bool pick) {
  switch (type) {
    case ASPIRE_T_F32: return pick ? &aspire_logits_pick_kernel<float> : &aspire_logits_kernel<float>;
    case ASPIRE_T_BF16: return pick ? &aspire_logits_pick_kernel<__nv_bfloat16> : &aspire_logits_kernel<__nv_bfloat16>;
    default: return pick ? &aspire_logits_pick_kernel<__half> : &aspire_logits_kernel<__half>;
  }
}

int logits_slice(int type) { return kWarps * (type == ASPIRE_T_F32 ? Walk<float>::kChunk : Walk<__half>::kChunk); }
size_t logits_smem_bytes() { return sizeof(Walk<float>::Stages); }
static_assert(sizeof(Walk<float>::Stages) == sizeof(Walk<__half>::Stages), "stages are as long for each type");

// A count and four bits an entry, a sum a word of bits.
size_t mark_smem_bytes(int blocks, bool wide) { return size_t(blocks) * kLogitsBlock / 16 * (wide ? 73 : 41); }

}  // namespace aspire
