// Products with 4-bit weights and group scales: parameters, tile lookup and
// the unpacking shared by the two kernels (w4_small.cu for few tokens,
// w4_tc.cu for many).
//
//   y[t, n] = sum_k x[t, k] (q[n, k] - z[n, k / G]) s[n, k / G]  (+ r[t, n])
//
// or, with the activation, rows [0, n) of the matrix are the gate's and rows
// [n, 2n) the up product's: y = silu(gate) * up.  Sums are in fp32 and each
// output is rounded once.  A matrix is uint32 words [rows, k / 8]: word j of a
// row holds weights 8j..8j+7, weight 8j+2i in bits 4i and weight 8j+2i+1 in
// bits 16+4i, so (word >> 4i) & 0x000F000F is a pair of neighbouring weights
// in the two halves of a register.
#pragma once

#include <cooperative_groups.h>

#include "kernels.cuh"

namespace aspire {

struct W4Params {
  const uint16_t* x;        // [rows, k] bf16 or fp16
  int64_t x_stride;
  int32_t rows;
  const uint32_t* codes;    // [experts,] [matrix rows, k / 8]
  int64_t codes_stride, codes_stride_e;    // words
  const uint16_t* scales;   // [experts,] [matrix rows, k / group], x's type
  int64_t scales_stride, scales_stride_e;
  const uint8_t* zeros;     // the same shape, or NULL: 8
  int64_t zeros_stride, zeros_stride_e;
  const uint16_t* residual; // [rows, n] or NULL
  int64_t residual_stride;
  uint16_t* out;            // [rows, n]
  int64_t out_stride;
  int32_t out_quads;        // every four neighbouring outputs of a token are 8-byte aligned, and n a multiple of 4
  int32_t n, k;
  int32_t group_blocks;     // groups of 128 m weights: m; else 1
  uint32_t group_recip;     // floor(2^32 / m) + 1, or 0 when m is 1
  // Whether rows are aligned such that the groups of 256 weights load at once
  // (with one group per 128 weights: that group is 128, and a word holds them).
  int32_t scales_vec, zeros_vec;
  const int32_t* offsets;   // rows of expert e: [offsets[e], offsets[e + 1]); NULL: one matrix for all rows
  int32_t num_experts;
  uint32_t* status;
  uint64_t wait_ns;         // bound of one pipeline wait (tcgen05 kernel)
};

constexpr int kW4MaxExperts = 1024;

namespace w4 {

constexpr int kRows = 128;  // matrix rows of a tile (of each half of one in the tcgen05 kernel)

// A CTA's share of the output: `count` rows of x from `row0`, with the matrix
// of `expert`.  expert -1: the rows belong to none and their outputs are zero.
// count 0: nothing to do.
struct Tile {
  int32_t expert, row0, count;
};

// A row range [lo, hi) cut to [0, rows); one that leaves it or runs backwards is
// reported.
__device__ __forceinline__ void cut_range(const W4Params& p, int lo, int hi, int& begin, int& count) {
  begin = min(max(lo, 0), p.rows);
  const int end = min(max(hi, begin), p.rows);
  if (lo != begin || hi != end) record_status(p.status, ASPIRE_STATUS_BAD_ROW);
  count = end - begin;
}

// For every expert its rows and its first token tile (tiles of `width` rows,
// numbered in expert order); the last entries are the end of the last expert's
// rows and the number of tiles.  The tiles of the rows of no expert, before the
// first's and past the last's, follow.
struct ExpertTiles {
  int32_t begin[kW4MaxExperts + 1];
  int32_t end[kW4MaxExperts + 1];
  int32_t tile[kW4MaxExperts + 1];
};

// Fills them; run by one whole warp, whose loads for 128 experts are in flight
// together.
__device__ __forceinline__ void expert_tiles(const W4Params& p, int width, int lane, ExpertTiles& t) {
  int base = 0;
  const int last = p.offsets[p.num_experts];
  for (int e0 = 0; e0 < p.num_experts; e0 += 128) {
    int lo[4], hi[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int e = e0 + i * 32 + lane;
      lo[i] = hi[i] = 0;
      if (e < p.num_experts) {
        lo[i] = p.offsets[e];
        hi[i] = p.offsets[e + 1];
      }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int e = e0 + i * 32 + lane;
      int begin, count;
      cut_range(p, lo[i], hi[i], begin, count);
      const int mine = (count + width - 1) / width;
      int incl = mine;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, incl, d);
        if (lane >= d) incl += v;
      }
      if (e < p.num_experts) {
        t.begin[e] = begin;
        t.end[e] = begin + count;
        t.tile[e] = base + incl - mine;
      }
      base += __shfl_sync(0xffffffffu, incl, 31);
    }
  }
  if (lane == 0) {
    t.begin[p.num_experts] = min(max(last, 0), p.rows);
    t.tile[p.num_experts] = base;
  }
}

// Number of token tiles, those of the rows of no expert included.
__device__ __forceinline__ int token_tile_count(const W4Params& p, int width, const ExpertTiles& t) {
  if (p.offsets == nullptr) return (p.rows + width - 1) / width;
  return t.tile[p.num_experts] + (t.begin[0] + width - 1) / width +
         (p.rows - t.begin[p.num_experts] + width - 1) / width;
}

// Token tile `index`.
__device__ __forceinline__ Tile find_tile(const W4Params& p, int index, int width, const ExpertTiles& t) {
  if (p.offsets == nullptr) return Tile{0, index * width, min(width, p.rows - index * width)};
  const int E = p.num_experts;
  if (index >= t.tile[E]) {
    const int first = t.begin[0], i = index - t.tile[E], before = (first + width - 1) / width;
    if (i < before) return Tile{-1, i * width, min(width, first - i * width)};
    const int row0 = t.begin[E] + (i - before) * width;
    return Tile{-1, row0, min(width, p.rows - row0)};
  }
  int lo = 0, hi = E;  // the last expert whose first tile is at or before the index
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (t.tile[mid] <= index) lo = mid; else hi = mid;
  }
  const int row0 = t.begin[lo] + (index - t.tile[lo]) * width;
  return Tile{lo, row0, min(width, t.end[lo] - row0)};
}

// ------------------------------------------------------------------ numbers
// The two activation types and how a word of codes becomes numbers: unpack()
// gives (q - z) / kUnit of its eight weights as four pairs of neighbours, each
// exactly.  c0 and c1 hold the zero point as that takes it (zero_consts).
// Pairs whose nibbles sit in the low four bits are OR-ed into the mantissa of
// 128 (bf16, 7 bits) or 1024 (fp16, 10 bits): the number plus q.  The nibbles
// above them would need a shift each, but are numbers as they stand: in fp16
// OR-ed into 1024 they are 1024 + 16 q, and in bf16 the bare bits are q 2^-129
// (below 8 a subnormal, above it the first binade, which continues it), which
// one fused operation scales by 2^127.  So a word takes one shift.
template <bool BF16>
struct Num;

__device__ __forceinline__ uint32_t and_or(uint32_t a, uint32_t mask, uint32_t or_) {
  // One three-input operation, written out: the compiler keeps it as two when
  // both constants are immediates.
  uint32_t r;
  asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(r) : "r"(a), "r"(mask), "r"(or_));
  return r;
}

template <>
struct Num<true> {
  static constexpr float kUnit = 4.0f;
  __device__ static __forceinline__ float to_float(uint16_t v) { return __uint_as_float(uint32_t(v) << 16); }
  __device__ static __forceinline__ uint16_t from_float(float v) {
    return __bfloat16_as_ushort(__float2bfloat16_rn(v));
  }
  __device__ static __forceinline__ uint32_t pack2(float lo, float hi) {
    const __nv_bfloat162 r = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&r);
  }
  __device__ static __forceinline__ uint32_t fma2(uint32_t a, uint32_t b, uint32_t c) {
    uint32_t d;
    asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(d) : "r"(a), "r"(b), "r"(c));
    return d;
  }
  __device__ static __forceinline__ uint32_t mul2(uint32_t a, uint32_t b) {
    const __nv_bfloat162 r = __hmul2(*reinterpret_cast<__nv_bfloat162*>(&a), *reinterpret_cast<__nv_bfloat162*>(&b));
    return *reinterpret_cast<const uint32_t*>(&r);
  }
  // c0 = -(128 + z) / 4 and c1 = -z / 4, as pairs.
  __device__ static __forceinline__ void zero_consts(uint32_t z, uint32_t& c0, uint32_t& c1) {
    c0 = 0xC200C200u + z * 0x00010001u;
    c1 = fma2(c0, 0x3F803F80u, 0x42004200u);  // + 32
  }
  __device__ static __forceinline__ void unpack(uint32_t word, uint32_t c0, uint32_t c1, uint32_t* v) {
    const uint32_t high = word >> 8;
    v[0] = fma2(and_or(word, 0x000F000Fu, 0x43004300u), 0x3E803E80u, c0);
    v[1] = fma2(word & 0x00F000F0u, 0x7F007F00u, c1);
    v[2] = fma2(and_or(high, 0x000F000Fu, 0x43004300u), 0x3E803E80u, c0);
    v[3] = fma2(high & 0x00F000F0u, 0x7F007F00u, c1);
  }
};
template <>
struct Num<false> {
  static constexpr float kUnit = 1.0f;
  __device__ static __forceinline__ float to_float(uint16_t v) { return __half2float(__ushort_as_half(v)); }
  __device__ static __forceinline__ uint16_t from_float(float v) { return __half_as_ushort(__float2half_rn(v)); }
  __device__ static __forceinline__ uint32_t pack2(float lo, float hi) {
    const __half2 r = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&r);
  }
  __device__ static __forceinline__ uint32_t fma2(uint32_t a, uint32_t b, uint32_t c) {
    uint32_t d;
    asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(d) : "r"(a), "r"(b), "r"(c));
    return d;
  }
  __device__ static __forceinline__ uint32_t mul2(uint32_t a, uint32_t b) {
    const __half2 r = __hmul2(*reinterpret_cast<__half2*>(&a), *reinterpret_cast<__half2*>(&b));
    return *reinterpret_cast<const uint32_t*>(&r);
  }
  // c0 = -(1024 + z) and c1 = -(64 + z), as pairs.
  __device__ static __forceinline__ void zero_consts(uint32_t z, uint32_t& c0, uint32_t& c1) {
    c0 = 0xE400E400u + z * 0x00010001u;
    c1 = fma2(c0, 0x3C003C00u, 0x63806380u);  // + 960
  }
  __device__ static __forceinline__ void unpack(uint32_t word, uint32_t c0, uint32_t c1, uint32_t* v) {
    const uint32_t high = word >> 8;
    v[0] = fma2(and_or(word, 0x000F000Fu, 0x64006400u), 0x3C003C00u, c0);
    v[1] = fma2(and_or(word, 0x00F000F0u, 0x64006400u), 0x2C002C00u, c1);
    v[2] = fma2(and_or(high, 0x000F000Fu, 0x64006400u), 0x3C003C00u, c0);
    v[3] = fma2(and_or(high, 0x00F000F0u, 0x64006400u), 0x2C002C00u, c1);
  }
};

// A group's scale (bits 16-31) and zero point (4 bits: larger ones are cut).
__device__ __forceinline__ uint32_t pack_scale(uint16_t scale, uint32_t zero) {
  return (uint32_t(scale) << 16) | (zero & 15u);
}
__device__ __forceinline__ uint32_t scale_pair(uint32_t packed) { return __byte_perm(packed, 0, 0x3232); }

// One matrix row's packed scales, GROUPS (1, 2, 4) for every block of 128
// weights; a group of 128 m weights has one for m blocks.
template <bool BF16, int GROUPS>
struct ScaleRow {
  const uint16_t* scale;
  const uint8_t* zero;  // NULL: 8
  bool live;

  __device__ __forceinline__ ScaleRow(const uint16_t* scale_, const uint8_t* zero_, bool live_)
      : scale(scale_), zero(zero_), live(live_) {}
  __device__ __forceinline__ ScaleRow(const W4Params& p, int expert, int64_t row, bool live_)
      : scale(p.scales + int64_t(expert) * p.scales_stride_e + row * p.scales_stride),
        zero(p.zeros ? p.zeros + int64_t(expert) * p.zeros_stride_e + row * p.zeros_stride : nullptr),
        live(live_) {}

  __device__ __forceinline__ static int first_group(const W4Params& p, int block) {
    if (GROUPS > 1) return block * GROUPS;
    return p.group_recip ? int(__umulhi(uint32_t(block), p.group_recip)) : block;
  }
  // What load() reads: the groups' scales and zero points as they lie in
  // memory.  Nothing is computed from them before packed() asks, so that the
  // loads stay in flight.
  struct Raw {
    uint32_t scale[(GROUPS + 1) / 2];
    uint32_t zero;
  };
  // Blocks past the row's end give scale 0.
  __device__ __forceinline__ Raw load(const W4Params& p, int block) const {
    Raw v;
#pragma unroll
    for (int e = 0; e < (GROUPS + 1) / 2; ++e) v.scale[e] = 0;
    v.zero = 0x08080808u;
    if (!live || block * 128 >= p.k) return v;
    const int gi = first_group(p, block);
    if constexpr (GROUPS == 1) {
      v.scale[0] = __ldg(scale + gi);
      if (zero) v.zero = __ldg(zero + gi);
    } else {
      // A whole block's groups in one load each, where rows are aligned for it.
      const bool whole = block * 128 + 128 <= p.k;
      if (whole && p.scales_vec) {
        if constexpr (GROUPS == 4) {
          const uint2 u = __ldg(reinterpret_cast<const uint2*>(scale + gi));
          v.scale[0] = u.x;
          v.scale[1] = u.y;
        } else {
          v.scale[0] = __ldg(reinterpret_cast<const uint32_t*>(scale + gi));
        }
      } else {
#pragma unroll
        for (int e = 0; e < GROUPS; ++e)
          if (block * 128 + e * (128 / GROUPS) < p.k) v.scale[e / 2] |= uint32_t(__ldg(scale + gi + e)) << (16 * (e & 1));
      }
      if (zero) {
        if (whole && p.zeros_vec) {
          if constexpr (GROUPS == 4)
            v.zero = __ldg(reinterpret_cast<const uint32_t*>(zero + gi));
          else
            v.zero = __ldg(reinterpret_cast<const uint16_t*>(zero + gi));
        } else {
          v.zero = 0;
#pragma unroll
          for (int e = 0; e < GROUPS; ++e)
            if (block * 128 + e * (128 / GROUPS) < p.k) v.zero |= uint32_t(__ldg(zero + gi + e)) << (8 * e);
        }
      }
    }
    return v;
  }
  // Group e's scale and zero point in one word (pack_scale).
  __device__ __forceinline__ static uint32_t packed(const Raw& v, int e) {
    return pack_scale(uint16_t(v.scale[e / 2] >> (16 * (e & 1))), v.zero >> (8 * e));
  }
};

__device__ __forceinline__ float silu(float v) { return v / (1.0f + __expf(-v)); }

// The outputs of a tile of ROWS matrix rows from the ranks' fp32 partials `red`
// [tokens][pitch] (matrix rows along a line), added in rank order: rank r
// finishes its part of the features.  Threads go along the features, so a
// token's outputs leave as consecutive elements.
template <bool BF16, bool SWIGLU, int ROWS>
__device__ __forceinline__ void finish_tile(const W4Params& p, const Tile& tile, int f0, int rank, int ranks,
                                            float* red, int pitch, int tid, int threads) {
  constexpr int FEATURES = SWIGLU ? ROWS / 2 : ROWS;
  const int share = FEATURES / ranks;  // a power of two
  const int shift = 31 - __clz(share);
  for (int i = tid; i < tile.count * share; i += threads) {
    const int t = i >> shift, fl = rank * share + (i & (share - 1)), f = f0 + fl;
    if (f >= p.n) continue;
    const int at = t * pitch + fl;
    float a = 0.f, b = 0.f;
    if (ranks == 1) {
      a = red[at];
      if (SWIGLU) b = red[at + FEATURES];
    } else {
      float va[8], vb[8];  // all in flight at once
#pragma unroll
      for (int q = 0; q < 8; ++q) {
        va[q] = vb[q] = 0.f;
        if (q < ranks) {
          const float* rq = cooperative_groups::this_cluster().map_shared_rank(red, q);
          va[q] = rq[at];
          if (SWIGLU) vb[q] = rq[at + FEATURES];
        }
      }
#pragma unroll
      for (int q = 0; q < 8; ++q) {
        a += va[q];
        if (SWIGLU) b += vb[q];
      }
    }
    const int64_t row = tile.row0 + t;
    if (SWIGLU) a = silu(a) * b;
    if (p.residual) a += Num<BF16>::to_float(p.residual[row * p.residual_stride + f]);
    p.out[row * p.out_stride + f] = Num<BF16>::from_float(a);
  }
}

}  // namespace w4

constexpr int kW4SmallThreads = 256;
// The small kernel's dynamic shared memory, by tokens per tile (8, 16)
// and groups per 128 weights of a row (1, 2, 4).
size_t w4_small_smem(int tokens, int groups);
// The kernel for an activation type, tokens per tile (8, 16), groups per
// 128 weights (1, 2, 4) and output form.
using W4Kernel = void (*)(W4Params);
W4Kernel w4_small_kernel(bool bf16, int tokens, int groups, bool swiglu);

// The tcgen05 kernel, by tokens per tile (32, 64, 128).  Its tensor maps:
// the codes as int32 [experts, rows, k / 8] with boxes of 32 words x 128 rows,
// the tokens as [rows, k] with boxes of 64 x tokens, both with the 128-byte
// swizzle.
constexpr int kW4TcThreads = 640;
size_t w4_tc_smem(int tokens);
using W4TcKernel = void (*)(W4Params, CUtensorMap, CUtensorMap);
W4TcKernel w4_tc_kernel(bool bf16, int tokens, int groups, bool swiglu);

}  // namespace aspire
