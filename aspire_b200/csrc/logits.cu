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
// A CTA owns a slice of one row's vocabulary: it counts the history's tokens
// in its slice in shared memory (integer atomics: the order does not matter)
// and marks them in a bitmap, then goes over the slices of all the row's
// tokens, which share the history.  Eight (or four) logits at a time whose
// bits are clear pass as they are.  The slices' best tokens are joined by
// aspire_pick_kernel.
#include "tree.cuh"

namespace aspire {

namespace {

constexpr uint32_t kInPrompt = 0x80000000u;

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

// Bits [at, at + 8) of a bit array of `words` words.
__device__ __forceinline__ uint32_t bits8(const uint32_t* a, int64_t at, int64_t words) {
  const int64_t w = at >> 5;
  const int s = int(at & 31);
  uint32_t v = a[w] >> s;
  if (s > 24 && w + 1 < words) v |= a[w + 1] << (32 - s);
  return v & 0xff;
}

struct RowTerms {
  float repetition, frequency, presence;
  bool repeat;
};

struct Slice {
  uint32_t* count;   // [slice] occurrences, kInPrompt for tokens of the prompt
  uint32_t* biased;  // [slice] 1 + the entry of the token's bias, NULL without biases
  uint32_t* touched; // bitmap: count or bias set
};

// The adjusted logit of slice entry e.
__device__ __forceinline__ float adjusted(const LogitsParams& p, const Slice& s, const RowTerms& r, int e, float x) {
  const uint32_t c = s.count[e];
  if (c) {
    const uint32_t made = c & ~kInPrompt;
    if (r.repeat) x = x > 0.f ? __fdiv_rn(x, r.repetition) : __fmul_rn(x, r.repetition);
    if (made) {
      x = __fsub_rn(x, __fmul_rn(r.frequency, float(made)));
      x = __fsub_rn(x, r.presence);
    }
  }
  if (s.biased) {
    const uint32_t b = s.biased[e];
    if (b) x = __fadd_rn(x, p.bias_values[b - 1]);
  }
  return x;
}

struct Best {
  float value;
  int32_t id;
};
__device__ __forceinline__ void better(Best& a, float value, int32_t id) {
  if (value > a.value || (value == a.value && id < a.id && value > -INFINITY)) {
    a.value = value;
    a.id = id;
  }
}

}  // namespace

template <typename T>
__global__ void __launch_bounds__(kLogitsThreads) aspire_logits_kernel(LogitsParams p) {
  pdl_begin();
  extern __shared__ uint32_t logits_smem[];
  __shared__ Best warp_best[kLogitsThreads / 32];
  constexpr int kVec = 16 / int(sizeof(T));
  const int tid = threadIdx.x;
  const int b = blockIdx.y;
  const int64_t v0 = int64_t(blockIdx.x) * p.slice;
  const int n = int(min(int64_t(p.slice), p.vocab - v0));
  const T* logits = static_cast<const T*>(p.logits);
  T* out = static_cast<T*>(p.out);

  int64_t lo = b, hi = b + 1;
  if (b >= p.rows) {  // tokens behind the last row's: as they are
    lo = p.indptr ? min(max(int64_t(p.indptr[p.rows]), int64_t(0)), p.tokens) : min(int64_t(p.rows), p.tokens);
    if (out == nullptr || static_cast<const void*>(out) == p.logits) return;
    for (int64_t t = lo; t < p.tokens; ++t)
      for (int e = tid; e < n; e += kLogitsThreads) out[t * p.out_stride + v0 + e] = logits[t * p.logits_stride + v0 + e];
    return;
  }
  if (p.indptr) {
    lo = p.indptr[b];
    hi = p.indptr[b + 1];
    if (lo < 0 || hi < lo || hi > p.tokens) {
      if (tid == 0) record_status(p.status, ASPIRE_STATUS_BAD_ROW);
      lo = min(max(lo, int64_t(0)), p.tokens);
      hi = min(max(hi, lo), p.tokens);
    }
  }
  if (lo >= hi) return;

  const int bit_words = (p.slice + 31) / 32;
  Slice s;
  s.touched = logits_smem;
  s.count = logits_smem + bit_words;
  s.biased = p.bias_indptr ? s.count + p.slice : nullptr;
  for (int i = tid; i < bit_words + p.slice * (p.bias_indptr ? 2 : 1); i += kLogitsThreads) logits_smem[i] = 0;
  __syncthreads();

  RowTerms r;
  r.repeat = p.repetition != nullptr;
  r.repetition = p.repetition ? p.repetition[b] : 1.f;
  r.frequency = p.frequency ? p.frequency[b] : 0.f;
  r.presence = p.presence ? p.presence[b] : 0.f;
  const auto mark = [&](int e) { atomicOr(&s.touched[e >> 5], 1u << (e & 31)); };
  if (p.history) {
    const int len = min(max(p.history_len[b], 0), p.history_cols);
    const int prompt = p.prompt_len ? p.prompt_len[b] : 0;
    const int32_t* h = p.history + b * p.history_stride;
    for (int i = tid; i < len; i += kLogitsThreads) {
      const int64_t e = h[i] - v0;
      if (e >= 0 && e < n) {
        if (i < prompt)
          atomicOr(&s.count[e], kInPrompt);
        else
          atomicAdd(&s.count[e], 1u);
        mark(int(e));
      }
    }
  }
  if (p.step_tokens) {
    for (int64_t t = lo + tid; t < hi; t += kLogitsThreads) {
      const int64_t e = p.step_tokens[t] - v0;
      if (e >= 0 && e < n) mark(int(e));
    }
  }
  if (p.bias_indptr) {
    int64_t from = p.bias_indptr[b], to = p.bias_indptr[b + 1];
    if (from < 0 || to < from || to > p.bias_entries) {
      if (tid == 0) record_status(p.status, ASPIRE_STATUS_BAD_ROW);
      from = to = 0;
    }
    for (int64_t i = from + tid; i < to; i += kLogitsThreads) {
      const int64_t e = p.bias_ids[i] - v0;
      if (e >= 0 && e < n) {
        atomicMax(&s.biased[e], uint32_t(i) + 1);  // of a token listed twice, the later entry
        mark(int(e));
      }
    }
  }

  for (int64_t t = lo; t < hi; ++t) {
    // The path's tokens count for this token alone.
    const auto path = [&](uint32_t change) {
      if (!p.step_tokens) return;
      // (Without masks the earlier tokens' counts are still there.)
      for (int64_t j = (p.tree_mask ? lo : t) + tid; j < (p.tree_mask ? hi : t + 1); j += kLogitsThreads) {
        const int64_t i = j - lo;
        if (p.tree_mask && (i >= 32 * int64_t(p.mask_words) ||
                            !((uint32_t(p.tree_mask[t * p.mask_words + (i >> 5)]) >> (i & 31)) & 1)))
          continue;
        const int64_t e = p.step_tokens[j] - v0;
        if (e >= 0 && e < n) atomicAdd(&s.count[e], change);
      }
    };
    path(1u);
    __syncthreads();

    const T* src = logits + t * p.logits_stride + v0;
    T* dst = out ? out + t * p.out_stride + v0 : nullptr;
    const uint32_t* allowed =
        p.allowed ? reinterpret_cast<const uint32_t*>(p.allowed) + t * p.allowed_stride : nullptr;
    const int64_t allowed_words = (int64_t(p.vocab) + 31) / 32;
    Best best = {-INFINITY, -1};
    const auto one = [&](int e) {
      float x = to_float(src[e]);
      if ((s.touched[e >> 5] >> (e & 31)) & 1) x = adjusted(p, s, r, e, x);
      const int64_t v = v0 + e;
      if (allowed && !((allowed[v >> 5] >> (v & 31)) & 1)) x = -INFINITY;
      if (dst) dst[e] = from_float<T>(x);
      better(best, x, int32_t(v));
    };
    // Entries up to the first 16-byte boundary, whole vectors, the rest.
    const int head = min(n, int((16 - (reinterpret_cast<uintptr_t>(src) & 15)) & 15) / int(sizeof(T)));
    const int vectors = (n - head) / kVec;
    const bool wide_out = dst && ((reinterpret_cast<uintptr_t>(dst + head) & 15) == 0);
    for (int e = tid; e < head; e += kLogitsThreads) one(e);
    for (int i = tid; i < vectors; i += kLogitsThreads) {
      const int e0 = head + i * kVec;
      uint4 raw = *reinterpret_cast<const uint4*>(src + e0);
      T* x = reinterpret_cast<T*>(&raw);
      uint32_t hit = bits8(s.touched, e0, bit_words);
      uint32_t ok = allowed ? bits8(allowed, v0 + e0, allowed_words) : 0xffu;
      hit &= (1u << kVec) - 1;
      ok |= ~((1u << kVec) - 1);
      float f[kVec];
#pragma unroll
      for (int k = 0; k < kVec; ++k) f[k] = to_float(x[k]);
      if (hit || ok != 0xffffffffu) {
#pragma unroll
        for (int k = 0; k < kVec; ++k) {
          if ((hit >> k) & 1) f[k] = adjusted(p, s, r, e0 + k, f[k]);
          if (!((ok >> k) & 1)) f[k] = -INFINITY;
          x[k] = from_float<T>(f[k]);
        }
      }
      if (dst) {
        if (wide_out) {
          *reinterpret_cast<uint4*>(dst + e0) = raw;
        } else {
#pragma unroll
          for (int k = 0; k < kVec; ++k) dst[e0 + k] = x[k];
        }
      }
      if (p.best_value) {
#pragma unroll
        for (int k = 0; k < kVec; ++k) better(best, f[k], int32_t(v0 + e0 + k));
      }
    }
    for (int e = head + vectors * kVec + tid; e < n; e += kLogitsThreads) one(e);

    if (p.best_value) {
#pragma unroll
      for (int off = 16; off >= 1; off >>= 1) {
        const float v = __shfl_xor_sync(0xffffffffu, best.value, off);
        const int32_t id = __shfl_xor_sync(0xffffffffu, best.id, off);
        if (id >= 0 && (best.id < 0 || v > best.value || (v == best.value && id < best.id))) best = {v, id};
      }
      if ((tid & 31) == 0) warp_best[tid >> 5] = best;
    }
    __syncthreads();
    if (p.best_value && tid == 0) {
      for (int w = 1; w < kLogitsThreads / 32; ++w) {
        const Best o = warp_best[w];
        if (o.id >= 0 && (best.id < 0 || o.value > best.value || (o.value == best.value && o.id < best.id))) best = o;
      }
      p.best_value[t * p.slices + blockIdx.x] = best.value;
      p.best_id[t * p.slices + blockIdx.x] = best.id;
    }
    if (p.tree_mask) path(0xffffffffu);
    __syncthreads();
  }
}

LogitsKernel logits_kernel(int type) {
  return type == ASPIRE_T_F32    ? &aspire_logits_kernel<float>
         : type == ASPIRE_T_BF16 ? &aspire_logits_kernel<__nv_bfloat16>
                                 : &aspire_logits_kernel<__half>;
}

// The best of the slices' best tokens, a warp per token; -1 for tokens of no row.
__global__ void __launch_bounds__(kPickThreads) aspire_pick_kernel(LogitsParams p) {
  pdl_begin();
  const int lane = threadIdx.x & 31;
  const int64_t t = int64_t(blockIdx.x) * (kPickThreads / 32) + (threadIdx.x >> 5);
  if (t >= p.tokens) return;
  const int64_t first = p.indptr ? p.indptr[0] : 0, end = p.indptr ? int64_t(p.indptr[p.rows]) : int64_t(p.rows);
  Best best = {-INFINITY, -1};
  if (t >= first && t < end) {
    for (int i = lane; i < p.slices; i += 32) {
      const float v = p.best_value[t * p.slices + i];
      const int32_t id = p.best_id[t * p.slices + i];
      if (id >= 0 && id < p.vocab && (best.id < 0 || v > best.value)) best = {v, id};
    }
  }
#pragma unroll
  for (int off = 16; off >= 1; off >>= 1) {
    const float v = __shfl_xor_sync(0xffffffffu, best.value, off);
    const int32_t id = __shfl_xor_sync(0xffffffffu, best.id, off);
    if (id >= 0 && (best.id < 0 || v > best.value || (v == best.value && id < best.id))) best = {v, id};
  }
  if (lane == 0) p.ids[t] = best.id;
}

}  // namespace aspire
