// 4-bit products of many tokens (a decode batch, a prefill chunk) on tcgen05.
//
// A CTA owns 128 matrix rows (64 gate and 64 up rows with the activation) as
// the MMA's M dimension, TOKENS tokens as its N, and a range of K.  The
// weights' way is HBM -> shared memory (TMA, 128 rows x 256 weights a stage)
// -> registers -> TMEM: thread r of a warpgroup unpacks row r's 64 weights of
// a step, (q - z) exactly and times the scale with one rounding to the
// activations' type, and stores them as the MMA's A operand in TMEM, lane r.
// The tokens come by TMA as the K-major B operand, 64 of K a stage, and the
// fp32 sums stay in TMEM until the epilogue.  So the unpacked weights never
// take shared-memory bandwidth, which the B operand needs, and every thread
// meets one row's scales only.
//
// Roles: warps 0-3 and 4-7 unpack (one warpgroup takes steps 0 and 1 of a
// 256-weight stage, the other steps 2 and 3; the sum's order is free, so the
// MMA takes them alternately) and run the epilogue, warp 8 loads the tokens,
// warp 10 the codes (each as far ahead as its own ring allows), warp 9 issues
// the MMAs.  Every wait is bounded; after a timeout the CTA
// reports it, lets its copies and MMAs land, frees TMEM and returns.
//
// Few tiles: a cluster splits K and adds the partials in distributed shared
// memory in rank order, as in the kernel for few tokens.
#include <cooperative_groups.h>

#include "tc_pipeline.cuh"
#include "tc_ptx.cuh"
#include "w4.cuh"

namespace aspire {

namespace {

namespace cg = cooperative_groups;
using namespace w4;
using pipe::drain_bar;
using pipe::wait_bar;

constexpr int kStageK = 256;                     // weights of a row per code stage
constexpr int kStepK = 64;                       // K of one A / B stage
constexpr int kSteps = kStageK / kStepK;
constexpr uint32_t kCodeBytes = kRows * kStageK / 2;
constexpr int kRedPitch = kRows + 4;             // floats
constexpr int kUnpackThreads = 256;
constexpr int kXWarp = 8, kMmaWarp = 9, kCodeWarp = 10;

template <int TOKENS>
struct Shape {
  static constexpr int kCodeStages = TOKENS == 128 ? 2 : 3;  // two CTAs per SM below 256 tokens
  static constexpr int kXStages = TOKENS == 64 ? 6 : 4;
  static constexpr uint32_t kXBytes = uint32_t(TOKENS) * kStepK * 2;
  static constexpr uint32_t kTmemCols = TOKENS == 256 ? 512 : 256;
  static constexpr int kAStages = (int(kTmemCols) - TOKENS) / 32 > 4 ? ((int(kTmemCols) - TOKENS) / 32 >= 8 ? 8 : 6) : 4;
  static constexpr size_t kRing = size_t(kCodeStages) * kCodeBytes + size_t(kXStages) * kXBytes;
  static constexpr size_t kRed = size_t(TOKENS) * kRedPitch * 4;
  static constexpr size_t kBytes = (kRing > kRed ? kRing : kRed) + 1024;  // 1 KiB to align the swizzled tiles
  static_assert(TOKENS + 32 * kAStages <= int(kTmemCols), "TMEM columns");
};

struct Control {
  uint64_t w_full[3], w_empty[3];
  uint64_t x_full[6], x_empty[6];
  uint64_t a_full[8], a_empty[8];
  uint64_t d_full;
  uint64_t wait_ns;
  uint32_t tmem_base;
  int abort_flag;
  Tile tile;
};

template <bool BF16, int TOKENS, int GROUPS, bool SWIGLU>
__global__ void __launch_bounds__(kW4TcThreads, TOKENS == 256 ? 1 : 2)
    aspire_w4_tc_kernel(const __grid_constant__ W4Params p, const __grid_constant__ CUtensorMap codes_map,
                        const __grid_constant__ CUtensorMap x_map) {
  pdl_begin();
  using S = Shape<TOKENS>;
  constexpr int FEATURES = SWIGLU ? kRows / 2 : kRows;
  constexpr int SW = S::kCodeStages, SX = S::kXStages, SA = S::kAStages;
  extern __shared__ uint8_t smem_raw[];
  __shared__ Control sm;
  uint8_t* smem = smem_raw + ((1024 - (ptx::smem_addr(smem_raw) & 1023)) & 1023);
  uint8_t* codes_s = smem;
  uint8_t* x_s = smem + SW * kCodeBytes;
  float* red = reinterpret_cast<float*>(smem);

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int rank = blockIdx.x, ranks = gridDim.x;
  const int f0 = blockIdx.y * FEATURES;
  if (warp == 0) {
    const Tile t = find_tile(p, blockIdx.z, TOKENS, lane);
    if (lane == 0) {
      sm.tile = t;
      sm.abort_flag = 0;
      sm.wait_ns = p.wait_ns;
      for (int i = 0; i < SW; ++i) {
        ptx::mbar_init(ptx::smem_addr(&sm.w_full[i]), 1);
        ptx::mbar_init(ptx::smem_addr(&sm.w_empty[i]), kUnpackThreads / 32);
      }
      for (int i = 0; i < SX; ++i) {
        ptx::mbar_init(ptx::smem_addr(&sm.x_full[i]), 1);
        ptx::mbar_init(ptx::smem_addr(&sm.x_empty[i]), 1);
      }
      for (int i = 0; i < SA; ++i) {
        ptx::mbar_init(ptx::smem_addr(&sm.a_full[i]), 4);
        ptx::mbar_init(ptx::smem_addr(&sm.a_empty[i]), 1);
      }
      ptx::mbar_init(ptx::smem_addr(&sm.d_full), 1);
      ptx::mbar_fence_init();
    }
  }
  __syncthreads();
  const Tile tile = sm.tile;
  if (tile.count <= 0) return;  // the whole cluster: its CTAs share the tile
  if (tile.expert < 0) {
    if (rank == 0)
      for (int i = tid; i < tile.count * FEATURES; i += kW4TcThreads) {
        const int t = i / FEATURES, f = f0 + i % FEATURES;
        if (f < p.n) p.out[int64_t(tile.row0 + t) * p.out_stride + f] = 0;
      }
    return;
  }
  if (warp == kMmaWarp) {
    ptx::tmem_alloc(ptx::smem_addr(&sm.tmem_base), S::kTmemCols);
    ptx::tmem_relinquish();
  }
  ptx::tc_fence_before();
  __syncthreads();
  ptx::tc_fence_after();
  const uint32_t tmem = sm.tmem_base;
  const uint32_t a_col = TOKENS;  // A stages follow the sums

  const int n_stages = (p.k + kStageK - 1) / kStageK;
  const int s_begin = int(int64_t(n_stages) * rank / ranks), s_end = int(int64_t(n_stages) * (rank + 1) / ranks);
  const int stages = s_end - s_begin;
  const int steps = stages * kSteps;
  // Step i of the MMA's order: stage i / 4, K sub-block (0, 2, 1, 3)[i % 4].
  auto sub_of = [](int i) { return ((i & 1) << 1) | ((i >> 1) & 1); };

  if (warp == kCodeWarp) {
    if (lane == 0) {
      ptx::prefetch_tmap(&codes_map);
      int s = 0;
      for (; s < stages; ++s) {
        const int ws = s % SW;
        if (!wait_bar(sm, sm.w_empty[ws], ((s / SW) & 1) ^ 1, p.status)) break;
        const uint32_t bar = ptx::smem_addr(&sm.w_full[ws]);
        const uint32_t dst = ptx::smem_addr(codes_s + ws * kCodeBytes);
        const int c0 = (s_begin + s) * (kStageK / 8);
        ptx::mbar_arrive_expect_tx(bar, kCodeBytes);
        ptx::tma_load_3d(dst, &codes_map, bar, c0, f0, tile.expert);
        if (SWIGLU) ptx::tma_load_3d(dst + kCodeBytes / 2, &codes_map, bar, c0, p.n + f0, tile.expert);
      }
      // After a timeout anywhere the copies in flight land before the CTA ends.
      if (s < stages || pipe::aborted(sm))
        for (int i = max(0, s - SW); i < s; ++i) drain_bar(sm.w_full[i % SW], (i / SW) & 1);
    }
  } else if (warp == kXWarp) {
    if (lane == 0) {
      ptx::prefetch_tmap(&x_map);
      int i = 0;
      for (; i < steps; ++i) {
        const int xs = i % SX;
        if (!wait_bar(sm, sm.x_empty[xs], ((i / SX) & 1) ^ 1, p.status)) break;
        const uint32_t bar = ptx::smem_addr(&sm.x_full[xs]);
        ptx::mbar_arrive_expect_tx(bar, S::kXBytes);
        ptx::tma_load_2d(ptx::smem_addr(x_s + xs * S::kXBytes), &x_map, bar,
                         (s_begin + i / kSteps) * kStageK + sub_of(i % kSteps) * kStepK, tile.row0);
      }
      if (i < steps || pipe::aborted(sm))
        for (int j = max(0, i - SX); j < i; ++j) drain_bar(sm.x_full[j % SX], (j / SX) & 1);
    }
  } else if (warp == kMmaWarp) {
    constexpr uint32_t idesc =
        BF16 ? ptx::idesc_bf16(kRows, TOKENS, false, false) : ptx::idesc_f16(kRows, TOKENS, false, false);
    bool ok = true;
    for (int i = 0; i < steps; ++i) {
      const int as = i % SA, xs = i % SX;
      if (!wait_bar(sm, sm.x_full[xs], (i / SX) & 1, p.status) || !wait_bar(sm, sm.a_full[as], (i / SA) & 1, p.status))
        ok = false;
      if (!__all_sync(0xffffffffu, ok)) break;
      ptx::tc_fence_after();
      if (lane == 0) {
        const uint64_t b = ptx::smem_desc(ptx::smem_addr(x_s + xs * S::kXBytes), 16, 1024, ptx::kLayoutSw128);
#pragma unroll
        for (int kk = 0; kk < kStepK / 16; ++kk)
          ptx::mma_bf16_ts(tmem, tmem + a_col + uint32_t(as) * 32 + uint32_t(kk) * 8, b + uint64_t(kk * 32 >> 4), idesc,
                           (i > 0 || kk > 0) ? 1u : 0u);
        ptx::mma_commit(ptx::smem_addr(&sm.a_empty[as]));
        ptx::mma_commit(ptx::smem_addr(&sm.x_empty[xs]));
      }
      __syncwarp();
    }
    // Fires once every MMA issued so far has completed, after a timeout too.
    if (lane == 0) ptx::mma_commit(ptx::smem_addr(&sm.d_full));
    __syncwarp();
    drain_bar(sm.d_full, 0);
  } else if (warp < 8) {
    // -------------------------------------------------------------- unpack
    const int wg = warp >> 2;              // half of a stage
    const int r = tid & (kRows - 1);       // tile row
    int64_t mr = SWIGLU ? f0 + (r & (FEATURES - 1)) : f0 + r;
    const bool live = mr < p.n;
    if (SWIGLU && r >= FEATURES) mr += p.n;
    if (!live) mr = 0;
    const ScaleRow<BF16, GROUPS> scales(p, tile.expert, mr, live);
    const uint32_t lanes = tmem + (uint32_t((warp & 3) * 32) << 16);
    uint32_t cur[GROUPS], nxt[GROUPS];
    scales.load(p, s_begin * 2 + wg, nxt);
    bool ok = true;
    for (int s = 0; s < stages && ok; ++s) {
#pragma unroll
      for (int e = 0; e < GROUPS; ++e) cur[e] = nxt[e];
      if (s + 1 < stages) scales.load(p, (s_begin + s + 1) * 2 + wg, nxt);
      const int ws = s % SW;
      if (!wait_bar(sm, sm.w_full[ws], (s / SW) & 1, p.status)) ok = false;
      if (!__all_sync(0xffffffffu, ok)) break;
      const uint8_t* row = codes_s + ws * kCodeBytes + r * 128;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int i = s * kSteps + h * 2 + wg, as = i % SA;
        uint32_t w[8];
        *reinterpret_cast<uint4*>(w) = *reinterpret_cast<const uint4*>(row + (((wg * 4 + h * 2) ^ (r & 7)) << 4));
        *reinterpret_cast<uint4*>(w + 4) = *reinterpret_cast<const uint4*>(row + (((wg * 4 + h * 2 + 1) ^ (r & 7)) << 4));
        uint32_t a[32];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const uint32_t ps = cur[(h * 64 + j * 8) * GROUPS / 128];
          const uint32_t m = scale_pair(ps);
          uint32_t z0, z1;
          Num<BF16>::zero_consts(ps & 15u, z0, z1);
          Num<BF16>::unpack(w[j], z0, z1, a + j * 4);
#pragma unroll
          for (int q = 0; q < 4; ++q) a[j * 4 + q] = Num<BF16>::mul2(a[j * 4 + q], m);
        }
        if (!wait_bar(sm, sm.a_empty[as], ((i / SA) & 1) ^ 1, p.status)) ok = false;
        if (!__all_sync(0xffffffffu, ok)) break;
        ptx::tc_fence_after();
        ptx::tmem_st32(lanes + a_col + uint32_t(as) * 32, a);
        ptx::tmem_wait_st();
        ptx::tc_fence_before();
        __syncwarp();
        if (lane == 0) ptx::mbar_arrive(ptx::smem_addr(&sm.a_full[as]));
      }
      __syncwarp();
      if (lane == 0) ptx::mbar_arrive(ptx::smem_addr(&sm.w_empty[ws]));
    }
    // The sums, once every MMA has completed (and with it every read of the
    // rings, whose memory the partials take).
    if (ok && !wait_bar(sm, sm.d_full, 0, p.status)) ok = false;
  }
  __syncthreads();
  ptx::tc_fence_after();
  const bool good = !pipe::aborted(sm);
  if (good && warp < 8) {
    const uint32_t lanes = tmem + (uint32_t((warp & 3) * 32) << 16);
    const int r = tid & (kRows - 1);
#pragma unroll 1
    for (int c = (warp >> 2) * (TOKENS / 2); c < ((warp >> 2) + 1) * (TOKENS / 2); c += 32) {
      float v[32];
      ptx::tmem_ld32(lanes + uint32_t(c), v);
      ptx::tmem_wait_ld();
#pragma unroll
      for (int j = 0; j < 32; ++j) red[(c + j) * kRedPitch + r] = v[j] * Num<BF16>::kUnit;
    }
  }
  ptx::tc_fence_before();
  if (ranks > 1)
    cg::this_cluster().sync();
  else
    __syncthreads();
  if (warp == kMmaWarp) {
    ptx::tc_fence_after();
    ptx::tmem_dealloc(tmem, S::kTmemCols);
  }
  if (good) {
    finish_tile<BF16, SWIGLU>(p, tile, f0, rank, ranks, red, kRedPitch, tid, kW4TcThreads);
  }
  if (ranks > 1) cg::this_cluster().sync();  // peers read this CTA's partials until here
}

template <bool BF16, int TOKENS, bool SWIGLU>
W4TcKernel by_groups(int groups) {
  if (groups == 1) return aspire_w4_tc_kernel<BF16, TOKENS, 1, SWIGLU>;
  if (groups == 2) return aspire_w4_tc_kernel<BF16, TOKENS, 2, SWIGLU>;
  return aspire_w4_tc_kernel<BF16, TOKENS, 4, SWIGLU>;
}
template <bool BF16, bool SWIGLU>
W4TcKernel by_tokens(int tokens, int groups) {
  if (tokens == 64) return by_groups<BF16, 64, SWIGLU>(groups);
  if (tokens == 128) return by_groups<BF16, 128, SWIGLU>(groups);
  return by_groups<BF16, 256, SWIGLU>(groups);
}

}  // namespace

size_t w4_tc_smem(int tokens) {
  return tokens == 64 ? Shape<64>::kBytes : (tokens == 128 ? Shape<128>::kBytes : Shape<256>::kBytes);
}

W4TcKernel w4_tc_kernel(bool bf16, int tokens, int groups, bool swiglu) {
  if (bf16) return swiglu ? by_tokens<true, true>(tokens, groups) : by_tokens<true, false>(tokens, groups);
  return swiglu ? by_tokens<false, true>(tokens, groups) : by_tokens<false, false>(tokens, groups);
}

}  // namespace aspire
