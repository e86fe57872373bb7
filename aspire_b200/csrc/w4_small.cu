// 4-bit products of few tokens (a drafting or verifying row, a decode batch).
//
// The weights' bytes are its floor: 0.5 byte feeds 2 x tokens operations.  What
// it spends beyond them is waiting where stages are handed over (one row 4096 ->
// 151936: 57 % of the issue slots used, no pipe above 46 %).  A CTA
// owns 128 matrix rows (64 gate and 64 up rows with the activation), 8 or 16
// tokens and a range of K, and streams the rows' codes through a ring of
// 256-weight stages in shared memory (asynchronous 16-byte copies, 128
// contiguous bytes of a row at a time).  The loop is unrolled over the ring,
// so that its addresses are constants: unpacking a weight takes about 1.2
// instructions, and every one around it counts.
//
// The products run on warp-level matrix instructions with the weights as A
// (16 rows x 16 k) unpacked in registers and the tokens as B (8 columns): at
// 16 tokens and fewer the tensor rate does not limit the stream (26 % of that
// pipe), and unpacked fragments go straight from registers into the
// instruction.  The sum over k may run in any order, so the instruction's k
// slots are assigned to the codes as they lie: of each group's part of a stage
// lane (g, c) of a warp (g = lane / 4) loads the c-th quarter of row g's codes
// with one load, and a word's first two pairs of weights feed one instruction,
// its last two the next.  The tokens' matching 8-element pieces are permuted
// on their way into shared memory such that a fragment is one conflict-free
// 16-byte load; the codes' 16-byte chunks are placed at slot chunk ^ reversed
// bits of (row & 7), which keeps 4-, 8- and 16-byte fragment loads free of
// conflicts.
//
// Codes minus zero points are exact in 16 bits; a group's sum is scaled in
// fp32 and added to the running sum, so nothing is rounded before the output.
//
// Two warpgroups take the two 128-weight halves of each stage.  When there
// are fewer tiles than SMs, a cluster of 2, 4 or 8 CTAs splits K; the
// partials meet in distributed shared memory in rank order (no atomics, no
// workspace, the same bits every time).  One row 4096 -> 151936, groups of 128:
// 74 us (4.4 TB/s); 64 tokens over 128 experts 2048 -> 2 x 768: 55 us.
#include <cooperative_groups.h>

#include "w4.cuh"

namespace aspire {

namespace {

namespace cg = cooperative_groups;
using namespace w4;

constexpr int kStageK = 256;                      // weights of a row per stage
constexpr int kCodeBytes = kRows * kStageK / 2;   // 16 KiB
constexpr int kXPitch = kStageK * 2 + 64;         // bytes; 64 mod 128: conflict-free 16-byte fragment loads
constexpr int kRedPitch = kRows + 4;              // floats
constexpr int kSmemBudget = 113 * 1024;           // two CTAs per SM

// A stage: codes, tokens, and 128 rows' scales (2 x groups of 2 bytes) and
// zero points (a byte each; 4 bytes at least, the smallest copy).
__host__ __device__ constexpr int scale_row_bytes(int groups) { return 4 * groups; }
__host__ __device__ constexpr int zero_row_bytes(int groups) { return groups == 4 ? 8 : 4; }
__host__ __device__ constexpr int scale_at(int tokens) { return kCodeBytes + tokens * kXPitch; }
__host__ __device__ constexpr int zero_at(int tokens, int groups) {
  return scale_at(tokens) + kRows * scale_row_bytes(groups);
}
__host__ __device__ constexpr int stage_bytes(int tokens, int groups) {
  return zero_at(tokens, groups) + kRows * zero_row_bytes(groups);
}
__host__ __device__ constexpr int stages_for(int tokens, int groups) {
  const int s = kSmemBudget / stage_bytes(tokens, groups);
  return s > 4 ? 4 : s;
}
__host__ __device__ constexpr int ring_bytes(int tokens, int groups) {
  const int ring = stages_for(tokens, groups) * stage_bytes(tokens, groups);
  const int red = tokens * kRedPitch * 4;  // the partials reuse the ring
  return ring > red ? ring : red;
}
static_assert(sizeof(ExpertTiles) <= ring_bytes(8, 1), "the experts' tiles use the ring before it starts");

// Slot of a row's 16-byte chunk: chunk ^ this (f of row 0..7: 0 4 2 6 1 5 3 7).
__device__ __forceinline__ int slot_mask(int row) { return ((row & 1) << 2) | (row & 2) | ((row >> 2) & 1); }

// 16 bytes, of which `size` (16 or 0) come from src and the rest are zero.
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, uint32_t size) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(size) : "memory");
}
// SIZE bytes (4, 8 or 16), the first `size` of them from src, the rest zero.
template <int SIZE>
__device__ __forceinline__ void cp_async_small(uint32_t dst, const void* src, uint32_t size) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(dst), "l"(src), "n"(SIZE), "r"(size) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

template <bool BF16>
__device__ __forceinline__ void mma16816(float* d, const uint32_t* a, uint32_t b0, uint32_t b1) {
  if (BF16)
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, "
        "%2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, "
        "%2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// TOKENS: tokens of a tile (8, 16).  GROUPS: scale groups per 128 weights of a row (a
// group of more than 128 counts as one).  Grid: (cluster ranks, row tiles,
// token tiles).
template <bool BF16, int TOKENS, int GROUPS, bool SWIGLU>
__global__ void __launch_bounds__(kW4SmallThreads, 2) aspire_w4_small_kernel(const __grid_constant__ W4Params p) {
  // The next launch may start, and this one's addresses are worked out while the
  // last one ends; nothing is read before pdl_wait.
  pdl_launch_dependents();
  constexpr int NT = TOKENS / 8;
  constexpr int STAGES = stages_for(TOKENS, GROUPS);
  constexpr int WORDS = 4 / GROUPS;  // words of a group's part a lane loads
  // One barrier for two stages: with 8 tokens, whose stages are used up fastest,
  // 75 -> 73 us (one row 4096 -> 151936); with 16 tokens 121 -> 123.
  constexpr bool PAIRS = TOKENS == 8;
  static_assert(!PAIRS || STAGES == 4, "two pairs of stages");
  constexpr int STAGE = stage_bytes(TOKENS, GROUPS);
  constexpr int FEATURES = SWIGLU ? kRows / 2 : kRows;
  extern __shared__ __align__(128) uint8_t smem[];
  float* red = reinterpret_cast<float*>(smem);
  __shared__ Tile tile_s;

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int g = lane >> 2, c = lane & 3;
  const int rank = blockIdx.x, ranks = gridDim.x;
  const int f0 = blockIdx.y * FEATURES;
  if (warp == 0) {
    // (The ring's memory is free until the first copies.)
    ExpertTiles& tiles = *reinterpret_cast<ExpertTiles*>(smem);
    if (p.offsets != nullptr) {
      pdl_wait();
      expert_tiles(p, TOKENS, lane, tiles);
      __syncwarp();
    }
    if (lane == 0) {
      tile_s = Tile{0, 0, 0};
      if (int(blockIdx.z) < token_tile_count(p, TOKENS, tiles)) tile_s = find_tile(p, blockIdx.z, TOKENS, tiles);
    }
  }
  __syncthreads();
  const Tile tile = tile_s;
  if (tile.count <= 0) return;  // the whole cluster: its CTAs share the tile
  if (tile.expert < 0) {
    pdl_wait();
    if (rank == 0)
      for (int i = tid; i < tile.count * FEATURES; i += kW4SmallThreads) {
        const int t = i / FEATURES, f = f0 + i % FEATURES;
        if (f < p.n) p.out[int64_t(tile.row0 + t) * p.out_stride + f] = 0;
      }
    return;
  }
  const uint32_t* codes = p.codes + int64_t(tile.expert) * p.codes_stride_e;
  const uint16_t* x = p.x + int64_t(tile.row0) * p.x_stride;

  // Matrix row of tile row r (-1 past the matrix).
  auto matrix_row = [&](int r) -> int64_t {
    if (SWIGLU) {
      const int f = f0 + (r & (FEATURES - 1));
      return f < p.n ? int64_t(f) + (r >= FEATURES ? p.n : 0) : -1;
    }
    return f0 + r < p.n ? f0 + r : -1;
  };

  const int n_stages = (p.k + kStageK - 1) / kStageK;
  const int s_begin = int(int64_t(n_stages) * rank / ranks), s_end = int(int64_t(n_stages) * (rank + 1) / ranks);

  const void* const codes_any = p.codes;  // a readable address for copies of size 0
  // Copies of a stage: thread tid moves 16-byte chunk tid % 8 of rows tid / 8
  // + 32 i and 8-element piece lane of tokens warp + 8 i.  A size of 0 fills
  // with zeros and reads nothing.
  const int cc = tid & 7;
  const uint32_t* code_src[4];
  uint32_t code_size[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int64_t mr = matrix_row((tid >> 3) + 32 * i);
    code_size[i] = mr >= 0 ? 16 : 0;
    code_src[i] = codes + (mr >= 0 ? mr : 0) * p.codes_stride + int64_t(s_begin) * (kStageK / 8) + cc * 4;
  }
  constexpr int XN = TOKENS / 8;
  const uint16_t* x_src[XN];
  uint32_t x_size[XN];
#pragma unroll
  for (int i = 0; i < XN; ++i) {
    const int t = warp + i * 8;
    x_size[i] = t < tile.count ? 16 : 0;
    x_src[i] = x + (t < tile.count ? t : 0) * p.x_stride + int64_t(s_begin) * kStageK + lane * 8;
  }
  const uint32_t ring = static_cast<uint32_t>(__cvta_generic_to_shared(smem));
  const uint32_t code_dst = ring + (tid >> 3) * 128 + ((cc ^ slot_mask(tid >> 3)) << 4);
  // Piece u = WORDS c + i of a group's part goes to place 4 i + c.
  const int u = lane & (4 * WORDS - 1);
  const int place = (lane & ~(4 * WORDS - 1)) + (u % WORDS) * 4 + u / WORDS;
  const uint32_t x_dst = ring + kCodeBytes + warp * kXPitch + place * 16;
  // Scales and zero points: threads 0-127 copy their row's scales of the
  // stage, threads 128-255 its zero points.  Rows that are not aligned for
  // those copies are read element by element when the stage is loaded.
  constexpr int SB = scale_row_bytes(GROUPS), ZB = zero_row_bytes(GROUPS), PER_STAGE = 2 * GROUPS;
  const int sr = tid & (kRows - 1);
  const bool is_zero = tid >= kRows;
  const int64_t srow = matrix_row(sr);
  const uint8_t* side_src = nullptr;  // the row's first scale or zero point; NULL: nothing to copy
  if (srow >= 0) {
    if (!is_zero)
      side_src = reinterpret_cast<const uint8_t*>(p.scales + int64_t(tile.expert) * p.scales_stride_e +
                                                  srow * p.scales_stride);
    else if (p.zeros)
      side_src = p.zeros + int64_t(tile.expert) * p.zeros_stride_e + srow * p.zeros_stride;
  }
  const bool side_fast = is_zero ? p.zeros_vec : p.scales_vec;
  const int n_groups = int(int64_t(p.k) * GROUPS / 128);  // of a row, where the copies are used
  const uint32_t side_dst = ring + (is_zero ? zero_at(TOKENS, GROUPS) + sr * ZB : scale_at(TOKENS) + sr * SB);
  auto load_side = [&](int s, int slot) {
    const uint32_t dst = side_dst + slot * STAGE;
    if (side_fast) {
      // A stage's zero points with one group per 128 weights are half a word:
      // the word is copied, the reader picks its half.
      const int first = s * PER_STAGE & (is_zero ? ~(ZB - 1) : ~0);
      const int left = max(n_groups - first, 0);
      if (!is_zero)
        cp_async_small<SB>(dst, side_src ? side_src + first * 2 : codes_any, side_src ? min(left * 2, SB) : 0);
      else
        cp_async_small<ZB>(dst, side_src ? side_src + first : codes_any, side_src ? min(left, ZB) : 0);
    } else {
#pragma unroll
      for (int e = 0; e < PER_STAGE; ++e) {
        const int block = s * 2 + e / GROUPS;
        const int gi = ScaleRow<BF16, GROUPS>::first_group(p, block) + e % GROUPS;
        const bool live = side_src && block * 128 + (e % GROUPS) * (128 / GROUPS) < p.k;
        if (!is_zero)
          *reinterpret_cast<uint16_t*>(smem + (dst - ring) + e * 2) =
              live ? __ldg(reinterpret_cast<const uint16_t*>(side_src) + gi) : 0;
        else
          smem[dst - ring + (ZB > PER_STAGE ? (s & 1) * PER_STAGE : 0) + e] = live ? __ldg(side_src + gi) : 8;
      }
    }
  };
  // Stage s_first + ahead into ring slot `slot`, from sources at stage s_first.
  auto load_stage = [&](int s_first, int ahead, int slot) {
    const int s = s_first + ahead;
    if (s < s_end) {
      const bool code_live = s * kStageK + cc * 32 < p.k, x_live = s * kStageK + lane * 8 < p.k;
#pragma unroll
      for (int i = 0; i < 4; ++i)
        cp_async16(code_dst + slot * STAGE + i * 32 * 128, code_src[i] + ahead * (kStageK / 8),
                   code_live ? code_size[i] : 0);
#pragma unroll
      for (int i = 0; i < XN; ++i)
        cp_async16(x_dst + slot * STAGE + i * 8 * kXPitch, x_src[i] + ahead * kStageK, x_live ? x_size[i] : 0);
      if (!is_zero || p.zeros) load_side(s, slot);
    }
    cp_commit();
  };

  float acc[2][NT][4];
#pragma unroll
  for (int m = 0; m < 2; ++m)
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[m][t][i] = 0.f;

  const int wg = warp >> 2;             // half of the stage
  const int row_w = (warp & 3) * 32;    // the warp's 32 tile rows
  pdl_wait();
#pragma unroll
  for (int s = 0; s < (PAIRS ? 2 : STAGES - 1); ++s) load_stage(s_begin, s, s);

  const uint8_t* const scale_src = smem + scale_at(TOKENS) + (row_w + g) * SB + wg * GROUPS * 2;
  const uint8_t* const zero_src = smem + zero_at(TOKENS, GROUPS) + (row_w + g) * ZB + wg * GROUPS;
  const bool has_zeros = p.zeros != nullptr;
  // The lane's codes of each group's part (16, 8 or 4 bytes of the row), and
  // its piece of the tokens.
  const uint8_t* code_at[GROUPS];
#pragma unroll
  for (int gr = 0; gr < GROUPS; ++gr) {
    const int byte = wg * 64 + gr * 16 * WORDS + c * 4 * WORDS;
    code_at[gr] = smem + (row_w + g) * 128 + (((byte >> 4) ^ slot_mask(g)) << 4) + (byte & 15);
  }
  const uint8_t* const x_at = smem + kCodeBytes + g * kXPitch + wg * 256 + c * 16;

  for (int s0 = s_begin; s0 < s_end; s0 += STAGES) {
#pragma unroll
    for (int u = 0; u < STAGES; ++u) {
      const int s = s0 + u;
      if (s >= s_end) break;
      if (!PAIRS) {
        cp_wait<STAGES - 2>();
        __syncthreads();
        load_stage(s0, u + STAGES - 1, (u + STAGES - 1) % STAGES);
      } else if (u % 2 == 0) {
        // Both stages of the pair have landed, and the pair before is used up:
        // its slots take the next one.
        cp_wait<0>();
        __syncthreads();
        load_stage(s0, u + 2, (u + 2) % STAGES);
        load_stage(s0, u + 3, (u + 3) % STAGES);
      }
      const uint8_t* const zero_s = zero_src + u * STAGE + (ZB > PER_STAGE ? (s & 1) * PER_STAGE : 0);
#pragma unroll
      for (int gr = 0; gr < GROUPS; ++gr) {
        uint32_t w[2][2][4];  // row g and g + 8 of both 16-row tiles
#pragma unroll
        for (int m = 0; m < 2; ++m)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const uint8_t* at = code_at[gr] + u * STAGE + (m * 16 + h * 8) * 128;
            if constexpr (WORDS == 4) *reinterpret_cast<uint4*>(w[m][h]) = *reinterpret_cast<const uint4*>(at);
            if constexpr (WORDS == 2) *reinterpret_cast<uint2*>(w[m][h]) = *reinterpret_cast<const uint2*>(at);
            if constexpr (WORDS == 1) w[m][h][0] = *reinterpret_cast<const uint32_t*>(at);
          }
        float ks[2][2];
        uint32_t z0[2][2], z1[2][2];
#pragma unroll
        for (int m = 0; m < 2; ++m)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int r = m * 16 + h * 8;
            ks[m][h] = Num<BF16>::to_float(
                *reinterpret_cast<const uint16_t*>(scale_src + u * STAGE + r * SB + gr * 2));
            uint32_t z = 8;
            if (has_zeros) z = zero_s[r * ZB + gr] & 15u;
            Num<BF16>::zero_consts(z, z0[m][h], z1[m][h]);
          }
        float blk[2][NT][4];
#pragma unroll
        for (int m = 0; m < 2; ++m)
#pragma unroll
          for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) blk[m][t][i] = 0.f;
#pragma unroll
        for (int q = 0; q < WORDS; ++q) {
          uint4 xf[NT];
#pragma unroll
          for (int t = 0; t < NT; ++t)
            xf[t] = *reinterpret_cast<const uint4*>(x_at + u * STAGE + t * 8 * kXPitch + (gr * WORDS + q) * 64);
#pragma unroll
          for (int m = 0; m < 2; ++m) {
            uint32_t lo[4], hi[4];  // rows g and g + 8
            Num<BF16>::unpack(w[m][0][q], z0[m][0], z1[m][0], lo);
            Num<BF16>::unpack(w[m][1][q], z0[m][1], z1[m][1], hi);
            const uint32_t a[2][4] = {{lo[0], hi[0], lo[1], hi[1]}, {lo[2], hi[2], lo[3], hi[3]}};
#pragma unroll
            for (int t = 0; t < NT; ++t) {
              mma16816<BF16>(blk[m][t], a[0], xf[t].x, xf[t].y);
              mma16816<BF16>(blk[m][t], a[1], xf[t].z, xf[t].w);
            }
          }
        }
#pragma unroll
        for (int m = 0; m < 2; ++m) {
          const float k0 = ks[m][0], k1 = ks[m][1];
#pragma unroll
          for (int t = 0; t < NT; ++t) {
            acc[m][t][0] = fmaf(blk[m][t][0], k0, acc[m][t][0]);
            acc[m][t][1] = fmaf(blk[m][t][1], k0, acc[m][t][1]);
            acc[m][t][2] = fmaf(blk[m][t][2], k1, acc[m][t][2]);
            acc[m][t][3] = fmaf(blk[m][t][3], k1, acc[m][t][3]);
          }
        }
      }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) code_src[i] += STAGES * (kStageK / 8);
#pragma unroll
    for (int i = 0; i < XN; ++i) x_src[i] += STAGES * kStageK;
  }

  // The second warpgroup's partials join the first's, then the ranks' meet.
  cp_wait<0>();
  __syncthreads();
  auto red_at = [&](int m, int t, int i) {
    return (t * 8 + 2 * c + (i & 1)) * kRedPitch + row_w + m * 16 + (i >> 1) * 8 + g;
  };
  if (wg == 1) {
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) red[red_at(m, t, i)] = acc[m][t][i] * Num<BF16>::kUnit;
  }
  __syncthreads();
  if (wg == 0) {
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) red[red_at(m, t, i)] += acc[m][t][i] * Num<BF16>::kUnit;
  }
  if (ranks > 1)
    cg::this_cluster().sync();
  else
    __syncthreads();
  finish_tile<BF16, SWIGLU, kRows>(p, tile, f0, rank, ranks, red, kRedPitch, tid, kW4SmallThreads);
  if (ranks > 1) cg::this_cluster().sync();  // peers read this CTA's partials until here
}

template <bool BF16, int TOKENS, bool SWIGLU>
W4Kernel by_groups(int groups) {
  if (groups == 1) return aspire_w4_small_kernel<BF16, TOKENS, 1, SWIGLU>;
  if (groups == 2) return aspire_w4_small_kernel<BF16, TOKENS, 2, SWIGLU>;
  return aspire_w4_small_kernel<BF16, TOKENS, 4, SWIGLU>;
}
template <bool BF16, bool SWIGLU>
W4Kernel by_tokens(int tokens, int groups) {
  return tokens == 8 ? by_groups<BF16, 8, SWIGLU>(groups) : by_groups<BF16, 16, SWIGLU>(groups);
}

}  // namespace

size_t w4_small_smem(int tokens, int groups) { return size_t(ring_bytes(tokens, groups)); }

W4Kernel w4_small_kernel(bool bf16, int tokens, int groups, bool swiglu) {
  if (bf16) return swiglu ? by_tokens<true, true>(tokens, groups) : by_tokens<true, false>(tokens, groups);
  return swiglu ? by_tokens<false, true>(tokens, groups) : by_tokens<false, false>(tokens, groups);
}

}  // namespace aspire
