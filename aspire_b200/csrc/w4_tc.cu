// 4-bit products of many tokens (a decode batch, a prefill chunk) on tcgen05.
//
// One CTA per SM walks over tiles of 256 matrix rows x 32, 64 or 128 tokens.
// A tile's two halves of 128 rows (gate and up rows with the activation) are
// the M dimension of two MMAs that share every tile of tokens.  The weights'
// way is HBM -> shared memory (TMA, 256 rows x 256 weights a stage) ->
// registers -> TMEM: thread r of a warpgroup unpacks row r's 128 weights of a
// step, (q - z) exactly and times the scale with one rounding to the
// activations' type, and stores them as the MMA's A operand in TMEM, lane r.
// The tokens come by TMA as the K-major B operand, 128 of K a step, and the
// fp32 sums stay in TMEM until the epilogue.  So the unpacked weights never
// take shared-memory bandwidth, which the B operand needs, and every thread
// meets one row's scales only.
//
// An MMA of 128 rows x 16 k takes 64 cycles up to 128 tokens, and the thread
// that issues it spends 100 to 200 more on every wait and commit.  So each
// half has its own issuing warp, a step is 8 MMAs between one wait and one
// commit, and the rest is the unpacking warps' business: they see to it that
// the tokens are there before they report a step as unpacked, and release the
// tokens' stage when they find a step's operand free again.
//
// Roles: warps 0-15 unpack (warpgroup q takes half q & 1 of every other step)
// and run the epilogue, warp 16 loads the tokens, warp 17 the codes (each as
// far ahead as its own ring allows, into the next tiles too), warps 18 and 19
// issue the halves' MMAs.  Every wait is bounded; after a timeout the CTA
// reports it, lets its copies and MMAs land, frees TMEM and returns.
//
// The epilogue goes from TMEM by registers to global memory, while the MMAs of
// the next tile's first steps (unpacked before it) run: a lane holds one row, so a
// warp's stores are 32 neighbouring outputs of four tokens; gate and up sums of
// an output are in the same lane.  Few tiles: a cluster splits K and adds the
// partials in distributed shared memory in rank order, as in the kernel for
// few tokens.
//
// 4099 tokens 4096 -> 12288, bf16, groups of 128: 358 us (1.15 PFLOP/s), bound by
// the issue of the MMAs between waits; 64 tokens 4096 -> 2 x 12288: 31 us.  The
// 128-token forms spill 40 to 252 bytes a thread around the epilogue.
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

constexpr int kTileRows = 2 * kRows;
constexpr int kStageK = 256;                     // weights of a row per code stage
constexpr int kStepK = 128;                      // K of one A / B stage
constexpr int kSteps = kStageK / kStepK;
constexpr uint32_t kHalfCodes = kRows * kStageK / 2;
constexpr uint32_t kCodeBytes = 2 * kHalfCodes;
constexpr int kRedPitch = kTileRows + 4;         // floats
constexpr int kUnpackWarps = 16;
constexpr int kXWarp = 16, kCodeWarp = 17, kMmaWarp = 18;  // and 19: the second half's
constexpr uint32_t kTmemCols = 512;

template <int TOKENS>
struct Shape {
  static constexpr uint32_t kBox = uint32_t(TOKENS) * 128;   // 64 of K
  static constexpr uint32_t kXBytes = 2 * kBox;
  static constexpr int kXStages = 4;
  static constexpr int kCodeStages = TOKENS == 128 ? 2 : (TOKENS == 64 ? 4 : 5);
  // TMEM: the halves' sums, then the A stages (64 columns a half).
  static constexpr uint32_t kColA = 2 * TOKENS;
  static constexpr int kAStages = int(kTmemCols - kColA) / 128;
  static constexpr size_t kRing = size_t(kCodeStages) * kCodeBytes + size_t(kXStages) * kXBytes;
  static constexpr size_t kRed = size_t(TOKENS) * kRedPitch * 4;
  static_assert(kRed <= kRing, "the partials reuse the rings");
  static_assert(kAStages >= 2 && kAStages <= 3, "both parities of steps are in flight");
  static constexpr size_t kBytes = kRing + sizeof(ExpertTiles) + 1024;  // 1 KiB to align the swizzled tiles
};

struct Control {
  uint64_t w_full[5], w_empty[5];
  uint64_t x_full[4], x_empty[4];
  uint64_t a_full[3][2], a_empty[3][2];  // by half
  uint64_t d_full, d_empty, done;
  uint64_t wait_ns;
  uint32_t tmem_base;
  int abort_flag;
};

// TOKENS: tokens of a tile (32, 64, 128).  GROUPS: scale groups per 128
// weights of a row (a group of more than 128 counts as one).  Grid: (cluster
// ranks, CTAs or clusters); with more than one rank a cluster has one tile at
// most.
template <bool BF16, int TOKENS, int GROUPS, bool SWIGLU>
__global__ void __launch_bounds__(kW4TcThreads, 1)
    aspire_w4_tc_kernel(const __grid_constant__ W4Params p, const __grid_constant__ CUtensorMap codes_map,
                        const __grid_constant__ CUtensorMap x_map) {
  pdl_begin();
  using S = Shape<TOKENS>;
  constexpr int FEATURES = SWIGLU ? kRows : kTileRows;
  constexpr int SW = S::kCodeStages, SX = S::kXStages, SA = S::kAStages;
  extern __shared__ uint8_t smem_raw[];
  __shared__ Control sm;
  uint8_t* const codes_s = smem_raw + ((1024 - (ptx::smem_addr(smem_raw) & 1023)) & 1023);
  uint8_t* const x_s = codes_s + SW * kCodeBytes;
  float* const red = reinterpret_cast<float*>(codes_s);
  ExpertTiles& experts = *reinterpret_cast<ExpertTiles*>(codes_s + S::kRing);

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int rank = blockIdx.x, ranks = gridDim.x;
  if (warp == 0) {
    if (lane == 0) {
      sm.abort_flag = 0;
      sm.wait_ns = p.wait_ns;
      for (int i = 0; i < SW; ++i) {
        ptx::mbar_init(ptx::smem_addr(&sm.w_full[i]), 1);
        ptx::mbar_init(ptx::smem_addr(&sm.w_empty[i]), kUnpackWarps);
      }
      for (int i = 0; i < SX; ++i) {
        ptx::mbar_init(ptx::smem_addr(&sm.x_full[i]), 1);
        ptx::mbar_init(ptx::smem_addr(&sm.x_empty[i]), 2);
      }
      for (int i = 0; i < SA; ++i)
        for (int h = 0; h < 2; ++h) {
          ptx::mbar_init(ptx::smem_addr(&sm.a_full[i][h]), 4);
          ptx::mbar_init(ptx::smem_addr(&sm.a_empty[i][h]), 1);
        }
      ptx::mbar_init(ptx::smem_addr(&sm.d_full), 2);
      ptx::mbar_init(ptx::smem_addr(&sm.done), 2);
      ptx::mbar_init(ptx::smem_addr(&sm.d_empty), kUnpackWarps);
      ptx::mbar_fence_init();
    }
    if (p.offsets != nullptr) expert_tiles(p, TOKENS, lane, experts);
  }
  if (warp == kMmaWarp) {
    ptx::tmem_alloc(ptx::smem_addr(&sm.tmem_base), kTmemCols);
    ptx::tmem_relinquish();
  }
  ptx::tc_fence_before();
  __syncthreads();
  ptx::tc_fence_after();
  const uint32_t tmem = sm.tmem_base;
  const int row_tiles = (p.n + FEATURES - 1) / FEATURES;
  const int n_tiles = row_tiles * token_tile_count(p, TOKENS, experts);
  const int n_stages = (p.k + kStageK - 1) / kStageK;
  const int s_begin = int(int64_t(n_stages) * rank / ranks), s_end = int(int64_t(n_stages) * (rank + 1) / ranks);
  const int stages = s_end - s_begin, steps = stages * kSteps;
  const int first_tile = blockIdx.y, tile_step = gridDim.y;
  auto tile_of = [&](int i) { return find_tile(p, i / row_tiles, TOKENS, experts); };

  if (warp == kCodeWarp) {
    if (lane == 0) {
      ptx::prefetch_tmap(&codes_map);
      int n = 0;  // stages so far, over all tiles
      bool ok = true;
      for (int i = first_tile; i < n_tiles && ok; i += tile_step) {
        const Tile tile = tile_of(i);
        if (tile.expert < 0) continue;
        const int f0 = (i % row_tiles) * FEATURES;
        for (int s = s_begin; s < s_end; ++s, ++n) {
          const int ws = n % SW;
          if (!wait_bar(sm, sm.w_empty[ws], ((n / SW) & 1) ^ 1, p.status)) {
            ok = false;
            break;
          }
          const uint32_t bar = ptx::smem_addr(&sm.w_full[ws]);
          const uint32_t dst = ptx::smem_addr(codes_s + ws * kCodeBytes);
          ptx::mbar_arrive_expect_tx(bar, kCodeBytes);
          ptx::tma_load_3d(dst, &codes_map, bar, s * (kStageK / 8), f0, tile.expert);
          // (Past the matrix's last row the copy fills with zeros.)
          ptx::tma_load_3d(dst + kHalfCodes, &codes_map, bar, s * (kStageK / 8), SWIGLU ? p.n + f0 : f0 + kRows,
                           tile.expert);
        }
      }
      // The last copies land before the CTA ends, whatever stops the other roles:
      // a timeout may come after this warp has issued everything.
      for (int j = max(0, n - SW); j < n; ++j) drain_bar(sm.w_full[j % SW], (j / SW) & 1);
    }
  } else if (warp == kXWarp) {
    if (lane == 0) {
      ptx::prefetch_tmap(&x_map);
      int n = 0;  // steps so far
      bool ok = true;
      for (int i = first_tile; i < n_tiles && ok; i += tile_step) {
        const Tile tile = tile_of(i);
        if (tile.expert < 0) continue;
        for (int j = 0; j < steps; ++j, ++n) {
          const int xs = n % SX;
          if (!wait_bar(sm, sm.x_empty[xs], ((n / SX) & 1) ^ 1, p.status)) {
            ok = false;
            break;
          }
          const uint32_t bar = ptx::smem_addr(&sm.x_full[xs]);
          ptx::mbar_arrive_expect_tx(bar, S::kXBytes);
          const uint32_t dst = ptx::smem_addr(x_s + xs * S::kXBytes);
          const int k = s_begin * kStageK + j * kStepK;
          ptx::tma_load_2d(dst, &x_map, bar, k, tile.row0);
          ptx::tma_load_2d(dst + S::kBox, &x_map, bar, k + 64, tile.row0);
        }
      }
      for (int j = max(0, n - SX); j < n; ++j) drain_bar(sm.x_full[j % SX], (j / SX) & 1);
    }
  } else if (warp >= kMmaWarp) {
    constexpr uint32_t idesc =
        BF16 ? ptx::idesc_bf16(kRows, TOKENS, false, false) : ptx::idesc_f16(kRows, TOKENS, false, false);
    const int half = warp - kMmaWarp;
    const uint32_t d = tmem + half * TOKENS, a0 = tmem + S::kColA + half * 64;
    int n = 0, tiles = 0;
    bool ok = true;
    for (int i = first_tile; i < n_tiles && ok; i += tile_step) {
      if (tile_of(i).expert < 0) continue;
      // The previous tile's sums have been read.  (The warp decides as one: around
      // a timeout some lanes may find the phase complete and others the abort.)
      if (tiles > 0) ok = __all_sync(0xffffffffu, wait_bar(sm, sm.d_empty, (tiles - 1) & 1, p.status));
      for (int j = 0; j < steps && ok; ++j, ++n) {
        const int as = n % SA, xs = n % SX;
        // (Of a step whose tokens have arrived as well.)
        ok = wait_bar(sm, sm.a_full[as][half], (n / SA) & 1, p.status);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        ptx::tc_fence_after();
        if (lane == 0) {
          const uint64_t b = ptx::smem_desc(ptx::smem_addr(x_s + xs * S::kXBytes), 16, 1024, ptx::kLayoutSw128);
#pragma unroll
          for (int kk = 0; kk < kStepK / 16; ++kk)
            ptx::mma_bf16_ts(d, a0 + uint32_t(as) * 128 + kk * 8, b + (((kk / 4) * S::kBox + (kk % 4) * 32) >> 4), idesc,
                             (j > 0 || kk > 0) ? 1u : 0u);
          ptx::mma_commit(ptx::smem_addr(&sm.a_empty[as][half]));
          if (j == steps - 1) ptx::mma_commit(ptx::smem_addr(&sm.d_full));
        }
        __syncwarp();
      }
      ++tiles;
    }
    // Fires once every MMA issued so far has completed, after a timeout too.
    if (lane == 0) ptx::mma_commit(ptx::smem_addr(&sm.done));
    __syncwarp();
    drain_bar(sm.done, 0);
  } else {
    // -------------------------------------------------------------- unpack
    const int half = (warp >> 2) & 1, parity = warp >> 3;
    const int r = tid & (kRows - 1);       // row of the half
    const uint32_t lanes = tmem + (uint32_t((warp & 3) * 32) << 16);
    const uint32_t a_lanes = lanes + S::kColA + half * 64;
    uint32_t row_at[4];                    // the warp's 16-byte chunks of a stage: block `parity` of 128 weights
#pragma unroll
    for (int q = 0; q < 4; ++q) row_at[q] = half * kHalfCodes + r * 128 + (((parity * 4 + q) ^ (r & 7)) << 4);
    int n = 0, tiles = 0;                  // stages unpacked and tiles finished so far
    bool ok = true;
    // The tile being unpacked: its thread's output, and the block's scales,
    // loaded a stage ahead.
    int f = 0;
    bool live = false;
    ScaleRow<BF16, GROUPS> scales(nullptr, nullptr, false);
    typename ScaleRow<BF16, GROUPS>::Raw nxt;
    auto enter = [&](const Tile& tile, int i) {
      const int f0 = (i % row_tiles) * FEATURES;
      f = SWIGLU ? f0 + r : f0 + half * kRows + r;
      live = f < p.n;
      scales = ScaleRow<BF16, GROUPS>(p, tile.expert, live ? (SWIGLU && half ? int64_t(p.n) + f : f) : 0, live);
      nxt = scales.load(p, s_begin * 2 + parity);
    };
    auto unpack_stage = [&](int s) -> bool {
      uint32_t sc[GROUPS];
#pragma unroll
      for (int e = 0; e < GROUPS; ++e) sc[e] = ScaleRow<BF16, GROUPS>::packed(nxt, e);
      if (s + 1 < stages) nxt = scales.load(p, (s_begin + s + 1) * 2 + parity);
      const int ws = n % SW;
      if (!__all_sync(0xffffffffu, wait_bar(sm, sm.w_full[ws], (n / SW) & 1, p.status))) return false;
      const uint8_t* const st = codes_s + ws * kCodeBytes;
      const int j = n * kSteps + parity, as = j % SA;
      ++n;
      uint32_t w[16];
#pragma unroll
      for (int q = 0; q < 4; ++q) *reinterpret_cast<uint4*>(w + q * 4) = *reinterpret_cast<const uint4*>(st + row_at[q]);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        uint32_t a[32];
#pragma unroll
        for (int q = 0; q < 8; ++q) {
          const uint32_t ps = sc[(h * 8 + q) * GROUPS / 16], m = scale_pair(ps);
          uint32_t z0, z1;
          Num<BF16>::zero_consts(ps & 15u, z0, z1);
          Num<BF16>::unpack(w[h * 8 + q], z0, z1, a + q * 4);
#pragma unroll
          for (int e = 0; e < 4; ++e) a[q * 4 + e] = Num<BF16>::mul2(a[q * 4 + e], m);
        }
        if (h == 0) {
          // The A stage's previous step is through the tensor core, and with it
          // its tokens.
          if (!__all_sync(0xffffffffu, wait_bar(sm, sm.a_empty[as][half], ((j / SA) & 1) ^ 1, p.status))) return false;
          ptx::tc_fence_after();
          if (j >= SA && (warp & 3) == 0 && lane == 0) ptx::mbar_arrive(ptx::smem_addr(&sm.x_empty[(j - SA) % SX]));
        }
        ptx::tmem_st32(a_lanes + uint32_t(as) * 128 + h * 32, a);
      }
      // The stage is released only after the stores that take what was unpacked
      // from its last codes: an arrival does not wait for loads that are still on
      // their way, and only the stores (as volatile as the arrival) hold the order.
      __syncwarp();
      if (lane == 0) ptx::mbar_arrive(ptx::smem_addr(&sm.w_empty[ws]));
      ptx::tmem_wait_st();
      if ((warp & 3) == 0 &&
          !__all_sync(0xffffffffu, wait_bar(sm, sm.x_full[j % SX], (j / SX) & 1, p.status)))
        return false;
      ptx::tc_fence_before();
      __syncwarp();
      if (lane == 0) ptx::mbar_arrive(ptx::smem_addr(&sm.a_full[as][half]));
      return true;
    };

    int i = first_tile;
    Tile tile{-1, 0, 0};
    if (i < n_tiles) tile = tile_of(i);
    int ahead = 0;  // stages of the tile that were unpacked before its turn
    if (tile.expert >= 0) enter(tile, i);
    while (i < n_tiles && tile.expert >= 0) {
      for (int s = ahead; s < stages && ok; ++s) ok = unpack_stage(s);
      // The next tile's first stage is unpacked before this one's epilogue, so
      // that its MMAs start as soon as the sums have been read.
      const Tile done = tile;
      const int done_f = f;
      const bool done_live = live;
      i += tile_step;
      ahead = 0;
      if (i < n_tiles) {
        tile = tile_of(i);
        if (tile.expert >= 0 && ok) {
          enter(tile, i);
          ok = unpack_stage(0);
          ahead = 1;
        }
      }
      // ---------------------------------------------------------- epilogue
      if (ok) ok = __all_sync(0xffffffffu, wait_bar(sm, sm.d_full, tiles & 1, p.status));
      if (!ok) break;
      ++tiles;
      ptx::tc_fence_after();
      if (ranks > 1) {
        // (The rings are idle: their memory takes the partials.)
#pragma unroll 1
        for (int c = parity * (TOKENS / 2); c < (parity + 1) * (TOKENS / 2); c += 16) {
          float v[16];
          ptx::tmem_ld16(lanes + half * TOKENS + uint32_t(c), v);
          ptx::tmem_wait_ld();
#pragma unroll
          for (int e = 0; e < 16; ++e) red[(c + e) * kRedPitch + half * kRows + r] = v[e] * Num<BF16>::kUnit;
        }
        continue;
      }
      // Without the activation a warp writes its half's rows; with it, both
      // halves' warps share the tokens and read gate and up sums.  All sums go
      // to registers first: the next tile's MMAs run during the rest.
      constexpr int SHARE = SWIGLU ? TOKENS / 4 : TOKENS / 2;
      constexpr int AT_ONCE = SHARE < 16 ? SHARE : 16;
      const int c0 = SWIGLU ? (parity * 2 + half) * SHARE : parity * SHARE;
      float v[SHARE], u[SWIGLU ? SHARE : 1];
#pragma unroll
      for (int e = 0; e < SHARE; e += 8) {
        ptx::tmem_ld8(lanes + (SWIGLU ? 0 : half * TOKENS) + uint32_t(c0 + e), v + e);
        if constexpr (SWIGLU) ptx::tmem_ld8(lanes + TOKENS + uint32_t(c0 + e), u + e);
      }
      ptx::tmem_wait_ld();
      ptx::tc_fence_before();
      __syncwarp();
      if (lane == 0) ptx::mbar_arrive(ptx::smem_addr(&sm.d_empty));
      const int64_t out_stride = p.out_stride, res_stride = p.residual_stride;
#pragma unroll
      for (int c = 0; c < SHARE; c += AT_ONCE) {
        const int left = done.count - c0 - c;
        if (left <= 0) break;
        const int64_t row = done.row0 + c0 + c;
        uint16_t* const out = p.out + row * out_stride + done_f;
        if (p.residual) {
          const uint16_t* const res = p.residual + row * res_stride + done_f;
          uint16_t add[AT_ONCE];
#pragma unroll
          for (int e = 0; e < AT_ONCE; ++e) add[e] = done_live && e < left ? res[e * res_stride] : 0;
#pragma unroll
          for (int e = 0; e < AT_ONCE; ++e) v[c + e] = fmaf(v[c + e], Num<BF16>::kUnit, Num<BF16>::to_float(add[e]));
        } else {
#pragma unroll
          for (int e = 0; e < AT_ONCE; ++e) {
            v[c + e] *= Num<BF16>::kUnit;
            if constexpr (SWIGLU) v[c + e] = silu(v[c + e]) * (u[c + e] * Num<BF16>::kUnit);
          }
        }
        if (p.out_quads) {
          // Four lanes' rows of four tokens change places, so that a lane
          // stores four rows of one token (8 bytes, a quarter of the stores).
          const int quad = lane & 3;
          const bool odd = quad & 1, high = quad & 2;
          uint16_t* to = out - quad + quad * out_stride;
#pragma unroll
          for (int e = 0; e < AT_ONCE; e += 4, to += 4 * out_stride) {
            const uint32_t t01 = Num<BF16>::pack2(v[c + e], v[c + e + 1]);
            const uint32_t t23 = Num<BF16>::pack2(v[c + e + 2], v[c + e + 3]);
            const uint32_t got = __shfl_xor_sync(0xffffffffu, __byte_perm(t01, t23, odd ? 0x5410 : 0x7632), 1);
            const uint32_t ra = __byte_perm(t01, got, odd ? 0x3254 : 0x5410);  // token 0 or 1, two rows
            const uint32_t rb = __byte_perm(t23, got, odd ? 0x3276 : 0x7610);  // token 2 or 3
            const uint32_t other = __shfl_xor_sync(0xffffffffu, high ? ra : rb, 2);
            if (done_live && e + quad < left)
              *reinterpret_cast<uint2*>(to) = high ? make_uint2(other, rb) : make_uint2(ra, other);
          }
        } else {
#pragma unroll
          for (int e = 0; e < AT_ONCE; ++e)
            if (done_live && e < left) out[e * out_stride] = Num<BF16>::from_float(v[c + e]);
        }
      }
    }
    // Rows of no expert: the last tiles.
    for (; ok && i < n_tiles; i += tile_step) {
      const Tile rest = tile_of(i);
      const int f0 = (i % row_tiles) * FEATURES;
      if (rest.expert >= 0 || rank != 0) continue;
      for (int j = tid; j < rest.count * FEATURES; j += kUnpackWarps * 32) {
        const int t = j / FEATURES, at = f0 + j % FEATURES;
        if (at < p.n) p.out[int64_t(rest.row0 + t) * p.out_stride + at] = 0;
      }
    }
  }
  ptx::tc_fence_before();
  __syncthreads();
  if (warp == kMmaWarp) {
    ptx::tc_fence_after();
    ptx::tmem_dealloc(tmem, kTmemCols);
  }
  if (ranks > 1) {
    // One tile per cluster: its CTAs' partials meet, added in rank order.
    cg::this_cluster().sync();
    if (first_tile < n_tiles) {
      const Tile tile = tile_of(first_tile);
      if (tile.expert >= 0 && !pipe::aborted(sm))
        finish_tile<BF16, SWIGLU, kTileRows>(p, tile, (first_tile % row_tiles) * FEATURES, rank, ranks, red, kRedPitch,
                                             tid, kW4TcThreads);
    }
    cg::this_cluster().sync();  // peers read this CTA's partials until here
  }
}

template <bool BF16, int TOKENS, bool SWIGLU>
W4TcKernel by_groups(int groups) {
  if (groups == 1) return aspire_w4_tc_kernel<BF16, TOKENS, 1, SWIGLU>;
  if (groups == 2) return aspire_w4_tc_kernel<BF16, TOKENS, 2, SWIGLU>;
  return aspire_w4_tc_kernel<BF16, TOKENS, 4, SWIGLU>;
}
template <bool BF16, bool SWIGLU>
W4TcKernel by_tokens(int tokens, int groups) {
  if (tokens == 32) return by_groups<BF16, 32, SWIGLU>(groups);
  if (tokens == 64) return by_groups<BF16, 64, SWIGLU>(groups);
  return by_groups<BF16, 128, SWIGLU>(groups);
}

}  // namespace

size_t w4_tc_smem(int tokens) {
  return tokens == 32 ? Shape<32>::kBytes : (tokens == 64 ? Shape<64>::kBytes : Shape<128>::kBytes);
}

W4TcKernel w4_tc_kernel(bool bf16, int tokens, int groups, bool swiglu) {
  if (bf16) return swiglu ? by_tokens<true, true>(tokens, groups) : by_tokens<true, false>(tokens, groups);
  return swiglu ? by_tokens<false, true>(tokens, groups) : by_tokens<false, false>(tokens, groups);
}

}  // namespace aspire
