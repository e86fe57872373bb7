// 4-bit products of few tokens (a drafting or verifying row, a decode batch).
//
// The weights' bytes bound it: 0.5 byte feeds 2 x tokens operations.  A CTA
// owns 128 matrix rows (64 gate and 64 up rows with the activation), 8, 16 or
// 32 tokens and a range of K, and streams the rows' codes through a ring of
// 256-weight stages in shared memory (asynchronous 16-byte copies, 128
// contiguous bytes of a row at a time; chunk c of row r sits at slot c ^ (r &
// 7), so the fragment loads below touch every bank once).
//
// The products run on warp-level matrix instructions with the weights as A
// (16 rows x 16 k) unpacked in registers and the tokens as B (8 columns): at
// 8 to 32 tokens the unpacking, not the tensor rate, is what could slow the
// stream, and unpacked fragments go straight from registers into the
// instruction.  Lane (g, c) of a warp (g = lane / 4) holds word c of a row's
// 32-weight chunk, and the sum over k may run in any order, so the
// instruction's k slots are assigned to the word's weights in place (its
// first two pairs feed one instruction, the last two the next) and the
// tokens' fragment is the 16 contiguous bytes x[token g][32 i + 8 c ...].
//
// Codes minus zero points are exact in 16 bits; a group's sum is scaled in
// fp32 and added to the running sum, so nothing is rounded before the output.
//
// Two warpgroups take the two 128-weight halves of each stage.  When there
// are fewer tiles than SMs, a cluster of 2, 4 or 8 CTAs splits K; the
// partials meet in distributed shared memory in rank order (no atomics, no
// workspace, the same bits every time).
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

__host__ __device__ constexpr int stage_bytes(int tokens) { return kCodeBytes + tokens * kXPitch; }
// Packed scales of a stage: 128 rows x groups of 256 weights, double buffered.
__host__ __device__ constexpr int scale_bytes(int groups) { return 2 * 2 * groups * kRows * 4; }
__host__ __device__ constexpr int stages_for(int tokens, int groups) {
  const int s = (kSmemBudget - scale_bytes(groups)) / stage_bytes(tokens);
  return s > 4 ? 4 : s;
}
__host__ __device__ constexpr int ring_bytes(int tokens, int groups) {
  const int ring = stages_for(tokens, groups) * stage_bytes(tokens);
  const int red = 2 * tokens * kRedPitch * 4;  // the partials reuse the ring
  return ring > red ? ring : red;
}

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool live) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(live ? 16 : 0) : "memory");
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

// TOKENS: tokens of a tile.  GROUPS: scale groups per 128 weights of a row (a
// group of more than 128 counts as one).  Grid: (cluster ranks, row tiles,
// token tiles).
template <bool BF16, int TOKENS, int GROUPS, bool SWIGLU>
__global__ void __launch_bounds__(kW4SmallThreads, 2) aspire_w4_small_kernel(const __grid_constant__ W4Params p) {
  pdl_begin();
  constexpr int NT = TOKENS / 8;
  constexpr int STAGES = stages_for(TOKENS, GROUPS);
  constexpr int ENTRIES = 2 * GROUPS * kRows / kW4SmallThreads;  // packed scales of a stage per thread
  constexpr int CHUNKS_PER_GROUP = 4 / GROUPS;
  constexpr int FEATURES = SWIGLU ? kRows / 2 : kRows;
  extern __shared__ __align__(128) uint8_t smem[];
  uint32_t* sc = reinterpret_cast<uint32_t*>(smem + ring_bytes(TOKENS, GROUPS));
  float* red = reinterpret_cast<float*>(smem);
  __shared__ Tile tile_s;

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int g = lane >> 2, c = lane & 3;
  const int rank = blockIdx.x, ranks = gridDim.x;
  const int f0 = blockIdx.y * FEATURES;
  if (p.offsets != nullptr) {
    if (warp == 0) {
      const Tile t = find_tile(p, blockIdx.z, TOKENS, lane);
      if (lane == 0) tile_s = t;
    }
    __syncthreads();
  } else if (tid == 0) {
    tile_s = find_tile(p, blockIdx.z, TOKENS, 0);
  }
  if (p.offsets == nullptr) __syncthreads();
  const Tile tile = tile_s;
  if (tile.count <= 0) return;  // the whole cluster: its CTAs share the tile
  if (tile.expert < 0) {
    if (rank == 0)
      for (int i = tid; i < tile.count * FEATURES; i += kW4SmallThreads) {
        const int t = i / FEATURES, f = f0 + i % FEATURES;
        if (f < p.n) p.out[int64_t(tile.row0 + t) * p.out_stride + f] = 0;
      }
    return;
  }
  const uint32_t* codes = p.codes + int64_t(tile.expert) * p.codes_stride_e;
  const uint16_t* scales = p.scales + int64_t(tile.expert) * p.scales_stride_e;
  const uint8_t* zeros = p.zeros ? p.zeros + int64_t(tile.expert) * p.zeros_stride_e : nullptr;
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

  // Copies of a stage: thread tid moves 16-byte chunk tid % 8 of rows tid / 8
  // + 32 i, and its share of the tokens' chunks.
  const int cc = tid & 7;
  const uint32_t* code_src[4];
  bool code_live[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int64_t mr = matrix_row((tid >> 3) + 32 * i);
    code_live[i] = mr >= 0;
    code_src[i] = codes + (mr >= 0 ? mr : 0) * p.codes_stride + cc * 4;
  }
  const uint32_t ring = static_cast<uint32_t>(__cvta_generic_to_shared(smem));
  auto load_stage = [&](int s) {
    if (s < s_end) {
      const uint32_t base = ring + uint32_t((s - s_begin) % STAGES) * stage_bytes(TOKENS);
      const int kc = s * kStageK + cc * 32;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int r = (tid >> 3) + 32 * i;
        const bool live = code_live[i] && kc < p.k;
        cp_async16(base + r * 128 + ((cc ^ (r & 7)) << 4), live ? code_src[i] + s * (kStageK / 8) : codes, live);
      }
#pragma unroll
      for (int i = 0; i < TOKENS * 32 / kW4SmallThreads; ++i) {
        const int e = tid + i * kW4SmallThreads, t = e >> 5, ch = e & 31;
        const int kx = s * kStageK + ch * 8;
        const bool live = t < tile.count && kx < p.k;
        cp_async16(base + kCodeBytes + t * kXPitch + ch * 16, live ? x + t * p.x_stride + kx : p.x, live);
      }
    }
    cp_commit();
  };
  // Packed scales of a stage: entry e of row r covers weights [e * 128 /
  // GROUPS, ...) of the stage; loaded one stage ahead into registers.
  auto load_scales = [&](int s, uint32_t* v) {
#pragma unroll
    for (int i = 0; i < ENTRIES; ++i) {
      const int r = tid & (kRows - 1), e = (tid >> 7) + 2 * i;
      const int k0 = s * kStageK + e * (128 / GROUPS);
      const int64_t mr = matrix_row(r);
      v[i] = pack_scale<BF16>(0, 8);
      if (s < s_end && mr >= 0 && k0 < p.k) {
        const int gi = k0 / p.group;
        const uint32_t z = zeros ? zeros[mr * p.zeros_stride + gi] : 8u;
        v[i] = pack_scale<BF16>(scales[mr * p.scales_stride + gi], z);
      }
    }
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
  uint32_t next_sc[ENTRIES];
  load_scales(s_begin, next_sc);
#pragma unroll
  for (int s = 0; s < STAGES - 1; ++s) load_stage(s_begin + s);

  for (int s = s_begin; s < s_end; ++s) {
    uint32_t* sb = sc + ((s - s_begin) & 1) * (2 * GROUPS * kRows);
#pragma unroll
    for (int i = 0; i < ENTRIES; ++i) sb[((tid >> 7) + 2 * i) * kRows + (tid & (kRows - 1))] = next_sc[i];
    cp_wait<STAGES - 2>();
    __syncthreads();
    load_stage(s + STAGES - 1);
    load_scales(s + 1, next_sc);
    const uint8_t* st = smem + ((s - s_begin) % STAGES) * stage_bytes(TOKENS);
    const uint8_t* xs = st + kCodeBytes + g * kXPitch + wg * 256 + c * 16;
#pragma unroll
    for (int gr = 0; gr < GROUPS; ++gr) {
      uint32_t ps[2][2];
#pragma unroll
      for (int m = 0; m < 2; ++m)
#pragma unroll
        for (int h = 0; h < 2; ++h) ps[m][h] = sb[(wg * GROUPS + gr) * kRows + row_w + m * 16 + h * 8 + g];
      float blk[2][NT][4];
#pragma unroll
      for (int m = 0; m < 2; ++m)
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int i = 0; i < 4; ++i) blk[m][t][i] = 0.f;
#pragma unroll
      for (int q = 0; q < CHUNKS_PER_GROUP; ++q) {
        const int ch = gr * CHUNKS_PER_GROUP + q;  // 32-weight chunk of the half stage
        uint4 xf[NT];
#pragma unroll
        for (int t = 0; t < NT; ++t) xf[t] = *reinterpret_cast<const uint4*>(xs + t * 8 * kXPitch + ch * 64);
#pragma unroll
        for (int m = 0; m < 2; ++m) {
          const int r = row_w + m * 16 + g;  // r & 7 == g for this row and the one 8 below
          const uint8_t* wr = st + r * 128 + (((wg * 4 + ch) ^ g) << 4) + c * 4;
          const uint32_t w0 = *reinterpret_cast<const uint32_t*>(wr);
          const uint32_t w1 = *reinterpret_cast<const uint32_t*>(wr + 8 * 128);
          const uint32_t z0 = zero_pair(ps[m][0]), z1 = zero_pair(ps[m][1]);
          uint32_t a[2][4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            a[i >> 1][(i & 1) * 2] = Num<BF16>::sub2(magic_pair<BF16>(w0, i), z0);
            a[i >> 1][(i & 1) * 2 + 1] = Num<BF16>::sub2(magic_pair<BF16>(w1, i), z1);
          }
#pragma unroll
          for (int t = 0; t < NT; ++t) {
            mma16816<BF16>(blk[m][t], a[0], xf[t].x, xf[t].y);
            mma16816<BF16>(blk[m][t], a[1], xf[t].z, xf[t].w);
          }
        }
      }
#pragma unroll
      for (int m = 0; m < 2; ++m) {
        const float s0 = scale_of<BF16>(ps[m][0]), s1 = scale_of<BF16>(ps[m][1]);
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          acc[m][t][0] = fmaf(blk[m][t][0], s0, acc[m][t][0]);
          acc[m][t][1] = fmaf(blk[m][t][1], s0, acc[m][t][1]);
          acc[m][t][2] = fmaf(blk[m][t][2], s1, acc[m][t][2]);
          acc[m][t][3] = fmaf(blk[m][t][3], s1, acc[m][t][3]);
        }
      }
    }
  }

  // The warpgroups' and ranks' partials meet in shared memory.
  cp_wait<0>();
  __syncthreads();
#pragma unroll
  for (int m = 0; m < 2; ++m)
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        red[(wg * TOKENS + t * 8 + 2 * c + (i & 1)) * kRedPitch + row_w + m * 16 + (i >> 1) * 8 + g] = acc[m][t][i];
  if (ranks > 1)
    cg::this_cluster().sync();
  else
    __syncthreads();
  // Rank r finishes features [r, r + 1) x FEATURES / ranks.
  const int share = FEATURES / ranks;
  for (int i = tid; i < tile.count * share; i += kW4SmallThreads) {
    const int t = i / share, fl = rank * share + i % share, f = f0 + fl;
    if (f >= p.n) continue;
    float a = 0.f, b = 0.f;
    for (int q = 0; q < ranks; ++q) {
      const float* rq = ranks > 1 ? cg::this_cluster().map_shared_rank(red, q) : red;
      a += rq[t * kRedPitch + fl];
      a += rq[(TOKENS + t) * kRedPitch + fl];
      if (SWIGLU) {
        b += rq[t * kRedPitch + FEATURES + fl];
        b += rq[(TOKENS + t) * kRedPitch + FEATURES + fl];
      }
    }
    const int64_t row = tile.row0 + t;
    if (SWIGLU) a = silu(a) * b;
    if (p.residual) a += Num<BF16>::to_float(p.residual[row * p.residual_stride + f]);
    p.out[row * p.out_stride + f] = Num<BF16>::from_float(a);
  }
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
  if (tokens == 8) return by_groups<BF16, 8, SWIGLU>(groups);
  if (tokens == 16) return by_groups<BF16, 16, SWIGLU>(groups);
  return by_groups<BF16, 32, SWIGLU>(groups);
}

}  // namespace

size_t w4_small_smem(int tokens, int groups) { return size_t(ring_bytes(tokens, groups)) + scale_bytes(groups); }

W4Kernel w4_small_kernel(bool bf16, int tokens, int groups, bool swiglu) {
  if (bf16) return swiglu ? by_tokens<true, true>(tokens, groups) : by_tokens<true, false>(tokens, groups);
  return swiglu ? by_tokens<false, true>(tokens, groups) : by_tokens<false, false>(tokens, groups);
}

}  // namespace aspire
