// The gated feed-forward product H = act(X Wg) * (X Wu) with W = [Wg | Wu] (IMEX_OP_GATED_FFN), by the number
// of tokens:
//
//   gated_pair_kernel    more than 128 tokens: the CTA-pair GEMM's arrangement (gemm_tcgen05_2cta.cu) with a
//                        256 x 256 accumulator whose left half is the gate and whose right half is the up
//                        projection of the same 128 columns of H: CTA 0 of the pair loads the gate's 128
//                        columns of W, CTA 1 the up projection's, and every thread of the epilogue has both
//                        values of its elements in its own TMEM lane.
//   gated_tile_kernel    more than 128 tokens, but few such tiles: 128 tokens x 64 columns of H, whose gate and up
//                        columns are one 128-column operand, two CTAs per SM.
//   gated_few_kernel     up to 128 tokens, where W's bytes are the time: W^T is the M operand (the gate's and
//                        the up projection's columns of 64 columns of H per tile, as they lie), the tokens
//                        are the N operand, so that no part of a tensor-core tile is wasted on rows that do
//                        not exist.
//
// In the last two k is shared out between the CTAs of a cluster where there are few tiles; they add their parts up
// through distributed shared memory, in order.
#include "gated_common.cuh"

namespace imex {
namespace {

using attn::from_f32;
using attn::to_f32;
using namespace tc;
using namespace tc_host;

// Eight consecutive results of a row, `count` of which exist; by one access when `wide`.
template <bool BF16> __device__ __forceinline__ void store8(uint16_t *to, const float (&v)[8], bool wide, int count) {
  if (!wide) {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (e < count) to[e] = from_f32<BF16>(v[e]);
    return;
  }
  uint32_t w[4];
#pragma unroll
  for (int e = 0; e < 4; ++e)
    w[e] = static_cast<uint32_t>(from_f32<BF16>(v[2 * e])) | (static_cast<uint32_t>(from_f32<BF16>(v[2 * e + 1])) << 16);
  *reinterpret_cast<uint4 *>(to) = make_uint4(w[0], w[1], w[2], w[3]);
}

__device__ __forceinline__ void tmem_alloc_one(uint32_t slot, uint32_t columns) {
  asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(slot), "r"(columns) : "memory");
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
}

// ------------------------------------------------------------------------------------------ many tokens
namespace pair {
constexpr int BM = 128;   // rows per CTA, 256 per pair
constexpr int BF = 128;   // columns of H per tile
constexpr int BK = 128;
constexpr int STAGES = 3;
constexpr int BOX = 128 * 128;        // 128 rows x 64 k of X, or 128 k x 64 columns of W
constexpr int STAGE_BYTES = 4 * BOX;  // two boxes of each
constexpr int THREADS = 192;
constexpr int SMEM_BYTES = STAGES * STAGE_BYTES + 256;
struct Params {
  uint16_t *h, *gu;
  unsigned *status;
  long long ldh;
  int tokens, d_ff, act, tiles_m, tiles_f, num_tiles, k_blocks;
  int up;    // first column of the up projection in W
  int wide;  // results may be stored 16 bytes at a time
  uint32_t idesc;
};
// Bands of eight row blocks: the tiles in flight share few columns of W and few rows of X.
__device__ __forceinline__ void coords(int tile, const Params &p, int &mb, int &fb) {
  const int band_tiles = 8 * p.tiles_f, band = tile / band_tiles, first = band * 8;
  const int rows = min(8, p.tiles_m - first), t = tile - band * band_tiles;
  fb = t / rows;
  mb = first + t % rows;
}
} // namespace pair

template <bool BF16>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(pair::THREADS, 1)
gated_pair_kernel(const __grid_constant__ CUtensorMap tmap_x, const __grid_constant__ CUtensorMap tmap_w, const pair::Params p) {
  using namespace pair;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  const uint32_t base = smem_u32(smem_raw), bars = base + STAGES * STAGE_BYTES;
  auto full_bar = [&](int s) { return bars + 8u * s; };
  auto empty_bar = [&](int s) { return bars + 8u * (STAGES + s); };
  auto acc_full = [&](int a) { return bars + 8u * (2 * STAGES + a); };
  auto acc_empty = [&](int a) { return bars + 8u * (2 * STAGES + 2 + a); };
  const uint32_t slot = bars + 8u * (2 * STAGES + 4);
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();
  const int cluster = blockIdx.x >> 1, clusters = gridDim.x >> 1;

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(full_bar(s), 1);   // used in CTA 0: its own expect-tx arrival
      mbar_init(empty_bar(s), 1);  // one multicast commit per round
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(acc_full(a), 1);
      mbar_init(acc_empty(a), 8);  // used in CTA 0: four epilogue warps of both CTAs
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(slot), "r"(512) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  tcgen05_fence_before();
  __syncthreads();
  cluster_sync_all();  // the peer's barriers exist before anything signals them
  tcgen05_fence_after();
  const uint32_t tmem = *reinterpret_cast<volatile uint32_t *>(smem_raw + (slot - base));

  if (warp == 0) {
    if (lane == 0) {
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int tile = cluster; tile < p.num_tiles && ok; tile += clusters) {
        int mb, fb;
        coords(tile, p, mb, fb);
        const int row0 = mb * 2 * BM + static_cast<int>(rank) * BM;
        const int col0 = fb * BF + (rank ? p.up : 0);  // CTA 0: the gate's columns, CTA 1: the up projection's
        for (int kb = 0; kb < p.k_blocks; ++kb) {
          if (!mbar_wait(empty_bar(stage), phase ^ 1u)) {
            report(p.status, kStatusTmaWaitTimeout);
            ok = false;
            break;
          }
          const uint32_t bar = map_to_cta(full_bar(stage), 0);
          if (rank == 0) mbar_expect_tx(full_bar(stage), 2 * STAGE_BYTES);
          const uint32_t x = base + stage * STAGE_BYTES, w = x + 2 * BOX;
          tma_load_2d_pair(x, &tmap_x, kb * BK, row0, bar);
          tma_load_2d_pair(x + BOX, &tmap_x, kb * BK + 64, row0, bar);
          tma_load_2d_pair(w, &tmap_w, col0, kb * BK, bar);
          tma_load_2d_pair(w + BOX, &tmap_w, col0 + 64, kb * BK, bar);
          if (++stage == STAGES) stage = 0, phase ^= 1u;
        }
      }
      // everything this CTA loaded has been used before it may go
      for (int s = 0; s < STAGES; ++s) {
        if (!mbar_wait(empty_bar(stage), phase ^ 1u)) break;
        if (++stage == STAGES) stage = 0, phase ^= 1u;
      }
    }
  } else if (warp == 1) {
    if (rank == 0) {
      // the whole warp walks the loop, one thread issues (see attention_tc.cuh)
      const uint32_t leader = attn::elect_one();
      int stage = 0, acc = 0;
      uint32_t phase = 0, acc_phase = 0;
      bool ok = true;
      auto wait = [&](uint32_t bar, uint32_t parity) {
        ok = __all_sync(0xffffffffu, mbar_wait(bar, parity));
        return ok;
      };
      for (int tile = cluster; tile < p.num_tiles && ok; tile += clusters) {
        if (!wait(acc_empty(acc), acc_phase ^ 1u)) break;
        tcgen05_fence_after();
        for (int kb = 0; kb < p.k_blocks; ++kb) {
          if (!wait(full_bar(stage), phase)) break;
          tcgen05_fence_after();
          const uint32_t x = base + stage * STAGE_BYTES;
          const uint64_t a = make_smem_desc(x, 16, 1024), w = make_smem_desc(x + 2 * BOX, BOX, 1024);
#pragma unroll
          for (int k = 0; k < BK / 16; ++k)
            attn::mma_pair(tmem + acc * 256, a + (((k >> 2) * BOX + (k & 3) * 32) >> 4), w + (k * 2048 >> 4), p.idesc,
                           (kb | k) ? 1u : 0u, leader);
          attn::commit_pair(empty_bar(stage), leader);
          if (++stage == STAGES) stage = 0, phase ^= 1u;
        }
        if (!ok) break;
        attn::commit_pair(acc_full(acc), leader);
        if (++acc == 2) acc = 0, acc_phase ^= 1u;
      }
      if (!ok && lane == 0) report(p.status, kStatusMmaWaitTimeout);
    }
  } else {
    const int lane_group = warp & 3;
    int acc = 0;
    uint32_t acc_phase = 0;
    for (int tile = cluster; tile < p.num_tiles; tile += clusters) {
      int mb, fb;
      coords(tile, p, mb, fb);
      if (!__all_sync(0xffffffffu, mbar_wait(acc_full(acc), acc_phase))) {
        if (lane == 0) report(p.status, kStatusEpiWaitTimeout);
        break;
      }
      tcgen05_fence_after();
      const int row = mb * 2 * BM + static_cast<int>(rank) * BM + lane_group * 32 + lane;
      const uint32_t t = tmem + (static_cast<uint32_t>(lane_group * 32) << 16) + acc * 256;
#pragma unroll 1
      for (int c0 = 0; c0 < BF; c0 += 32) {
        uint32_t g[32], u[32];
        tmem_ld_32x32(t + c0, g);
        tmem_ld_32x32(t + BF + c0, u);
        tmem_ld_wait();
        if (row < p.tokens) {
#pragma unroll
          for (int j = 0; j < 32; j += 8) {
            const int col = fb * BF + c0 + j;
            if (col < p.d_ff) {
              const int count = p.d_ff - col;
              float x[8], y[8], v[8];
#pragma unroll
              for (int e = 0; e < 8; ++e) {
                x[e] = __uint_as_float(g[j + e]);
                y[e] = __uint_as_float(u[j + e]);
                v[e] = apply_epilogue_fast(x[e], p.act) * y[e];
              }
              store8<BF16>(p.h + row * p.ldh + col, v, p.wide, count);
              if (p.gu) {
                uint16_t *gu = p.gu + static_cast<long long>(row) * 2 * p.d_ff + col;
                store8<BF16>(gu, x, p.wide, count);
                store8<BF16>(gu + p.d_ff, y, p.wide, count);
              }
            }
          }
        }
        __syncwarp();
      }
      tcgen05_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_cluster(map_to_cta(acc_empty(acc), 0));
      if (++acc == 2) acc = 0, acc_phase ^= 1u;
    }
  }

  __syncwarp();
  tcgen05_fence_before();
  __syncthreads();
  cluster_sync_all();  // neither CTA leaves while the other may still touch its memory
  if (warp == 1) {
    tcgen05_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
  }
}

// -------------------------------------------------------------------------------- some tokens, few tiles
namespace mid {
constexpr int BK = 64, STAGES = 3;
constexpr int BF = 64;                         // columns of H per tile
constexpr int TILE_BYTES = 128 * 128;          // 128 tokens x 64 k, or 64 k x (64 gate, 64 up) columns
constexpr int STAGE_BYTES = 2 * TILE_BYTES;
constexpr int SMEM = STAGES * STAGE_BYTES + 256;
constexpr int THREADS = 256;                   // TMA, products, two idle warps, four that hand the sums over
static_assert(128 * 128 * 4 <= STAGES * STAGE_BYTES, "the sums take the ring's place");
static_assert(2 * (SMEM + 1024) <= 233472, "two CTAs per SM");
struct Params {
  uint16_t *h, *gu;
  unsigned *status;
  long long ldh;
  int tokens, d_ff, act, tiles_f, k_blocks, shares, up, wide;
  uint32_t idesc;
};
} // namespace mid

template <bool BF16>
__global__ void __launch_bounds__(mid::THREADS, 2)
gated_tile_kernel(const __grid_constant__ CUtensorMap tmap_x, const __grid_constant__ CUtensorMap tmap_w, const mid::Params p) {
  using namespace mid;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  const uint32_t base = smem_u32(smem_raw), bars = base + STAGES * STAGE_BYTES;
  auto full_bar = [&](int s) { return bars + 8u * s; };
  auto empty_bar = [&](int s) { return bars + 8u * (STAGES + s); };
  const uint32_t done = bars + 8u * (2 * STAGES), slot = done + 8;
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const int rank = p.shares > 1 ? static_cast<int>(cluster_ctarank()) : 0, tile = blockIdx.x / p.shares;
  const int row0 = tile / p.tiles_f * 128, f0 = tile % p.tiles_f * BF;
  const int kb0 = p.k_blocks * rank / p.shares, n = p.k_blocks * (rank + 1) / p.shares - kb0;

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(full_bar(s), 1);
      mbar_init(empty_bar(s), 1);
    }
    mbar_init(done, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  if (warp == 1) tmem_alloc_one(slot, 128);
  tcgen05_fence_before();
  __syncthreads();
  tcgen05_fence_after();
  const uint32_t tmem = *reinterpret_cast<volatile uint32_t *>(smem_raw + (slot - base));

  if (warp == 0) {
    if (lane == 0) {
      for (int i = 0; i < n; ++i) {
        const int s = i % STAGES, k = (kb0 + i) * BK;
        if (i >= STAGES && !mbar_wait(empty_bar(s), (i / STAGES - 1) & 1)) {
          report(p.status, kStatusTmaWaitTimeout);
          break;
        }
        mbar_expect_tx(full_bar(s), STAGE_BYTES);
        const uint32_t x = base + s * STAGE_BYTES, w = x + TILE_BYTES;
        tma_load_2d(x, &tmap_x, k, row0, full_bar(s));
        tma_load_2d(w, &tmap_w, f0, k, full_bar(s));
        tma_load_2d(w + TILE_BYTES / 2, &tmap_w, p.up + f0, k, full_bar(s));
      }
      for (int i = max(0, n - STAGES); i < n; ++i)  // everything has been used
        if (!mbar_wait(empty_bar(i % STAGES), (i / STAGES) & 1)) break;
    }
  } else if (warp == 1) {
    const uint32_t leader = attn::elect_one();
    bool ok = true;
    for (int i = 0; i < n && ok; ++i) {
      const int s = i % STAGES;
      ok = __all_sync(0xffffffffu, mbar_wait(full_bar(s), (i / STAGES) & 1));
      if (!ok) break;
      tcgen05_fence_after();
      const uint32_t at = base + s * STAGE_BYTES;
      const uint64_t x = make_smem_desc(at, 16, 1024), w = make_smem_desc(at + TILE_BYTES, TILE_BYTES / 2, 1024);
#pragma unroll
      for (int k = 0; k < BK / 16; ++k)
        attn::mma_ss(tmem, x + (k * 32 >> 4), w + (k * 2048 >> 4), p.idesc, (i | k) ? 1u : 0u, leader);
      attn::commit(empty_bar(s), leader);
    }
    if (ok) attn::commit(done, leader);
    else if (lane == 0) report(p.status, kStatusMmaWaitTimeout);
  }
  if (warp < 4) {
    if (p.shares > 1) {  // the other warps' two barriers
      __syncwarp();
      cluster_sync_all();
      cluster_sync_all();
    }
  } else {
    const bool ok = __all_sync(0xffffffffu, mbar_wait(done, 0));
    if (ok) {
      tcgen05_fence_after();
      const int lane_group = warp & 3;
      attn::leave_row<128, 128>(tmem + (static_cast<uint32_t>(lane_group * 32) << 16), true, base, lane_group * 32 + lane, 0);
    } else if (lane == 0) {
      report(p.status, kStatusEpiWaitTimeout);
    }
    attn::sums_barrier<128>(p.shares);
    // this CTA's part of the tokens; a thread has eight columns of H, whose up projection lies 64 columns behind
    for (int u = threadIdx.x - 128; u < 128 / p.shares * (BF / 8); u += 128) {
      const int r = rank * (128 / p.shares) + u / (BF / 8), unit = u % (BF / 8), token = row0 + r, col = f0 + unit * 8;
      float g[8] = {}, y[8] = {};
#pragma unroll 2
      for (int s = 0; s < p.shares; ++s) {
#pragma unroll
        for (int h = 0; h < 4; ++h) {
          const uint32_t at = base + attn::sum_offset<128>(r, unit * 2 + (h & 1) + (h >> 1) * 16);
          float4 v;
          asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                       : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
                       : "r"(p.shares > 1 ? map_to_cta(at, s) : at));
          float *to = (h >> 1 ? y : g) + (h & 1) * 4;
          to[0] += v.x, to[1] += v.y, to[2] += v.z, to[3] += v.w;
        }
      }
      if (token < p.tokens && col < p.d_ff) {
        float v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = apply_epilogue_fast(g[e], p.act) * y[e];
        store8<BF16>(p.h + token * p.ldh + col, v, p.wide, p.d_ff - col);
        if (p.gu) {
          uint16_t *gu = p.gu + static_cast<long long>(token) * 2 * p.d_ff + col;
          store8<BF16>(gu, g, p.wide, p.d_ff - col);
          store8<BF16>(gu + p.d_ff, y, p.wide, p.d_ff - col);
        }
      }
    }
    attn::sums_barrier<128>(p.shares);
  }
  __syncwarp();
  tcgen05_fence_before();
  __syncthreads();
  if (warp == 1) {
    tcgen05_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(128) : "memory");
  }
}

// ------------------------------------------------------------------------------------------- few tokens
namespace few {
constexpr int BF = 64;                  // columns of H per tile; the M of the product is their gate and up columns
constexpr int BK = 64;
constexpr int W_BOX = BK * 128;         // 64 k x 64 columns
constexpr int W_BYTES = 2 * W_BOX;      // gate, up
__host__ __device__ constexpr int stage_bytes(int nt) { return W_BYTES + nt * 128; }
// 90 to 100 KB of loads in flight; two CTAs per SM
__host__ __device__ constexpr int stages(int nt) { return nt <= 32 ? 5 : nt == 64 ? 4 : 3; }
__host__ __device__ constexpr int smem_bytes(int nt) { return stages(nt) * stage_bytes(nt) + 256; }
static_assert(2 * (smem_bytes(32) + 1024) <= 233472 && 2 * (smem_bytes(128) + 1024) <= 233472, "two CTAs per SM");
constexpr int THREADS = 192;
struct Params {
  uint16_t *h, *gu;
  unsigned *status;
  long long ldh;
  int tokens, d_ff, act, k_blocks, shares;
  int up;  // first column of the up projection in W
  uint32_t idesc;
};
} // namespace few

template <bool BF16, int NT>
__global__ void __launch_bounds__(few::THREADS, 2)
gated_few_kernel(const __grid_constant__ CUtensorMap tmap_x, const __grid_constant__ CUtensorMap tmap_w, const few::Params p) {
  using namespace few;
  constexpr int STAGES = stages(NT), STAGE_BYTES = stage_bytes(NT);
  static_assert(NT * 2 * BF * 4 <= STAGES * STAGE_BYTES, "the sums take the ring's place");
  constexpr int TMEM_COLS = NT < 32 ? 32 : NT;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  const uint32_t base = smem_u32(smem_raw), bars = base + STAGES * STAGE_BYTES;
  auto full_bar = [&](int s) { return bars + 8u * s; };
  auto empty_bar = [&](int s) { return bars + 8u * (STAGES + s); };
  const uint32_t acc_full = bars + 8u * (2 * STAGES), slot = acc_full + 8;
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const int rank = p.shares > 1 ? static_cast<int>(cluster_ctarank()) : 0;
  const int f0 = blockIdx.x / p.shares * BF;
  const int kb0 = p.k_blocks * rank / p.shares, kb1 = p.k_blocks * (rank + 1) / p.shares;

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(full_bar(s), 1);
      mbar_init(empty_bar(s), 1);
    }
    mbar_init(acc_full, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  if (warp == 1) tmem_alloc_one(slot, TMEM_COLS);
  tcgen05_fence_before();
  __syncthreads();
  tcgen05_fence_after();
  const uint32_t tmem = *reinterpret_cast<volatile uint32_t *>(smem_raw + (slot - base));
  float *sums = reinterpret_cast<float *>(smem_raw);  // [NT][gate BF, up BF] once the ring is done with

  if (warp == 0) {
    if (lane == 0) {
      for (int kb = kb0; kb < kb1; ++kb) {
        const int i = kb - kb0, s = i % STAGES;
        if (i >= STAGES && !mbar_wait(empty_bar(s), (i / STAGES - 1) & 1)) {
          report(p.status, kStatusTmaWaitTimeout);
          break;
        }
        mbar_expect_tx(full_bar(s), STAGE_BYTES);
        const uint32_t w = base + s * STAGE_BYTES;
        tma_load_2d(w, &tmap_w, f0, kb * BK, full_bar(s));
        tma_load_2d(w + W_BOX, &tmap_w, p.up + f0, kb * BK, full_bar(s));
        tma_load_2d(w + W_BYTES, &tmap_x, kb * BK, 0, full_bar(s));
      }
      for (int i = max(0, kb1 - kb0 - STAGES); i < kb1 - kb0; ++i)  // everything has been used
        if (!mbar_wait(empty_bar(i % STAGES), (i / STAGES) & 1)) break;
    }
  } else if (warp == 1) {
    const uint32_t leader = attn::elect_one();
    bool ok = true;
    for (int kb = kb0; kb < kb1; ++kb) {
      const int i = kb - kb0, s = i % STAGES;
      ok = __all_sync(0xffffffffu, mbar_wait(full_bar(s), (i / STAGES) & 1));
      if (!ok) break;
      tcgen05_fence_after();
      const uint32_t at = base + s * STAGE_BYTES;
      const uint64_t w = make_smem_desc(at, W_BOX, 1024), x = make_smem_desc(at + W_BYTES, 16, 1024);
#pragma unroll
      for (int k = 0; k < BK / 16; ++k)
        attn::mma_ss(tmem, w + (k * 2048 >> 4), x + (k * 32 >> 4), p.idesc, (i | k) ? 1u : 0u, leader);
      attn::commit(empty_bar(s), leader);
    }
    if (ok) attn::commit(acc_full, leader);
    else if (lane == 0) report(p.status, kStatusMmaWaitTimeout);
  }
  __syncwarp();
  // sums of this CTA's share of k: lane = column of H, a row of `sums` per token
  bool ok = __all_sync(0xffffffffu, mbar_wait(acc_full, 0));
  if (warp >= 2) {
    if (ok) {
      tcgen05_fence_after();
      const int lane_group = warp & 3;
      const uint32_t t = tmem + (static_cast<uint32_t>(lane_group * 32) << 16);
#pragma unroll 1
      for (int c0 = 0; c0 < NT; c0 += 32) {
        uint32_t v[32];
        tmem_ld_32x32(t + c0, v);
        tmem_ld_wait();
#pragma unroll
        for (int e = 0; e < 32; ++e)
          if (c0 + e < NT) sums[(c0 + e) * 2 * BF + lane_group * 32 + lane] = __uint_as_float(v[e]);
      }
    } else if (lane == 0) {
      report(p.status, kStatusEpiWaitTimeout);
    }
  }
  if (p.shares > 1) cluster_sync_all();
  else __syncthreads();
  if (warp >= 2 && ok) {
    // two tokens at a time
    const int c = threadIdx.x % BF, col = f0 + c;
    if (col < p.d_ff) {
      for (int token = rank * 2 + (threadIdx.x - 64) / BF; token < p.tokens; token += 2 * p.shares) {
        const uint32_t mine = base + (token * 2 * BF + c) * 4;
        float g = 0.0f, u = 0.0f;
#pragma unroll 4
        for (int r = 0; r < p.shares; ++r) {
          const uint32_t from = p.shares > 1 ? map_to_cta(mine, r) : mine;
          float x, y;
          asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(x) : "r"(from));
          asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(y) : "r"(from + BF * 4));
          g += x;
          u += y;
        }
        p.h[token * p.ldh + col] = from_f32<BF16>(apply_epilogue_fast(g, p.act) * u);
        if (p.gu) {
          p.gu[static_cast<long long>(token) * 2 * p.d_ff + col] = from_f32<BF16>(g);
          p.gu[static_cast<long long>(token) * 2 * p.d_ff + p.d_ff + col] = from_f32<BF16>(u);
        }
      }
    }
  }
  __syncwarp();
  tcgen05_fence_before();
  if (p.shares > 1) cluster_sync_all();  // the others may still read this CTA's sums
  else __syncthreads();
  if (warp == 1) {
    tcgen05_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(TMEM_COLS) : "memory");
  }
}

} // namespace

const char *gated_check(const GatedProblem &p, bool backward, bool pointers) {
  if (p.dtype != kF16 && p.dtype != kBF16) return "the element type is f16 or bf16";
  if (p.act != kEpiNone && p.act != kEpiRelu && p.act != kEpiSilu) return "unknown activation";
  if (p.tokens < 1 || p.d_in < 1 || p.d_ff < 1) return "extents are at least 1";
  if (p.tokens > (1 << 30) || p.d_in > (1 << 29) || p.d_ff > (1 << 29)) return "extents are at most 2^30 tokens, 2^29 columns";
  if ((p.ldx && p.ldx < p.d_in) || (p.ldw && p.ldw < 2 * p.d_ff) || (p.ldh && p.ldh < p.d_ff))
    return "row pitch smaller than the row";
  if (!pointers) return nullptr;
  const bool padded = gated::Layout(p).padded;
  const uintptr_t unit = padded ? 2 : 16;
  for (const void *q : {p.x, p.w, static_cast<const void *>(p.h), static_cast<const void *>(p.gu),
                        static_cast<const void *>(p.dx), static_cast<const void *>(p.dw)})
    if (reinterpret_cast<uintptr_t>(q) % unit)
      return padded ? "arrays must be aligned to their elements" : "arrays must be 16-byte aligned";
  if ((padded || backward) && reinterpret_cast<uintptr_t>(p.workspace) % 16) return "the workspace must be 16-byte aligned";
  // arrays that start at one address: a tile's results go out while others still read X and W
  if (!backward && (p.h == p.x || p.h == p.w || p.gu == p.x || p.gu == p.w || p.gu == p.h)) return "H and GU may not be X, W or one another";
  if (backward && (p.dx == p.x || p.dx == p.w || p.dw == p.x || p.dw == p.w || p.dx == p.dw)) return "dX and dW may not be X, W or one another";
  return nullptr;
}

size_t gated_workspace_bytes(const GatedProblem &p) { return gated::Layout(p).rest; }

namespace {

// A problem as the kernels get it: extents as the results have them, X and W with rows of whole 16-byte units.
struct Prepared {
  const void *x, *w;
  int64_t ldx, ldw, ldh, up;  // up: first column of the up projection in W
  bool wide;
};

bool tiles(CUtensorMap *tx, CUtensorMap *tw, const GatedProblem &p, const Prepared &q, int rows_x, int rows_w) {
  return make_map(tx, q.x, p.dtype, p.d_in, p.tokens, rows_x, q.ldx) && make_map(tw, q.w, p.dtype, q.up + p.d_ff, p.d_in, rows_w, q.ldw);
}

// `shares` CTAs per cluster
template <typename Params>
cudaError_t launch_cluster(void (*kernel)(CUtensorMap, CUtensorMap, Params), const CUtensorMap &tx, const CUtensorMap &tw,
                           const Params &f, int64_t grid, int threads, int smem, cudaStream_t stream) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(grid));
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = static_cast<unsigned>(f.shares);
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, tx, tw, f);
}

template <typename Params> Params common(const GatedProblem &p, const Prepared &q, int bk, unsigned *status) {
  Params f{};
  f.h = static_cast<uint16_t *>(p.h);
  f.gu = static_cast<uint16_t *>(p.gu);
  f.status = status;
  f.ldh = q.ldh;
  f.tokens = static_cast<int>(p.tokens);
  f.d_ff = static_cast<int>(p.d_ff);
  f.act = p.act;
  f.up = static_cast<int>(q.up);
  f.k_blocks = static_cast<int>((p.d_in + bk - 1) / bk);
  return f;
}

template <bool BF16, int NT>
cudaError_t launch_few(const GatedProblem &p, const Prepared &q, const few::Params &f, int64_t grid, cudaStream_t stream) {
  CUtensorMap tx, tw;
  if (!tiles(&tx, &tw, p, q, NT, few::BK)) return cudaErrorNotSupported;
  const cudaError_t e = attn::allow_smem<gated_few_kernel<BF16, NT>>(few::smem_bytes(NT));
  if (e != cudaSuccess) return e;
  return launch_cluster(gated_few_kernel<BF16, NT>, tx, tw, f, grid, few::THREADS, few::smem_bytes(NT), stream);
}

template <bool BF16>
cudaError_t launch_few_tokens(const GatedProblem &p, const Prepared &q, unsigned *status, cudaStream_t stream) {
  few::Params f = common<few::Params>(p, q, few::BK, status);
  const int nt = p.tokens <= 16 ? 16 : p.tokens <= 32 ? 32 : p.tokens <= 64 ? 64 : 128;
  const int64_t tiles = (p.d_ff + few::BF - 1) / few::BF;
  // Shares of k per tile: as many CTAs as run at once, at least two k blocks each.  One token of 4096 x 11264
  // (176 tiles): 31.5 us with one share, 38 with 2; of 8192 x 1024 (16 tiles): 35 us with one, 10.3 with 8.
  int64_t shares = 2 * sm_count() / tiles;
  if (shares > 8) shares = 8;
  if (shares > f.k_blocks / 2) shares = f.k_blocks / 2;
  f.shares = shares < 1 ? 1 : static_cast<int>(shares);
  const uint32_t fmt = BF16 ? 1u : 0u;
  // f32 accumulator; A (W) is MN-major, B (X) K-major; N >> 3, M >> 4
  f.idesc = (1u << 4) | (fmt << 7) | (fmt << 10) | (1u << 15) | (static_cast<uint32_t>(nt >> 3) << 17) |
            ((128u >> 4) << 24);
  if (nt == 16) return launch_few<BF16, 16>(p, q, f, tiles * f.shares, stream);
  if (nt == 32) return launch_few<BF16, 32>(p, q, f, tiles * f.shares, stream);
  if (nt == 64) return launch_few<BF16, 64>(p, q, f, tiles * f.shares, stream);
  return launch_few<BF16, 128>(p, q, f, tiles * f.shares, stream);
}

template <bool BF16>
cudaError_t launch_tiles(const GatedProblem &p, const Prepared &q, unsigned *status, cudaStream_t stream) {
  CUtensorMap tx, tw;
  if (!tiles(&tx, &tw, p, q, 128, mid::BK)) return cudaErrorNotSupported;
  const cudaError_t e = attn::allow_smem<gated_tile_kernel<BF16>>(mid::SMEM);
  if (e != cudaSuccess) return e;
  mid::Params f = common<mid::Params>(p, q, mid::BK, status);
  f.wide = q.wide;
  f.tiles_f = static_cast<int>((p.d_ff + mid::BF - 1) / mid::BF);
  const int64_t count = (p.tokens + 127) / 128 * f.tiles_f;
  // Shares of k: as many CTAs as run at once, at least twenty k blocks each (adding up costs about as much as eight).
  f.shares = 1;
  while (f.shares < 8 && count * f.shares * 2 <= 2 * sm_count() && f.k_blocks >= 40 * f.shares) f.shares *= 2;
  const uint32_t fmt = BF16 ? 1u : 0u;
  // f32 accumulator; A (X) is K-major, B (W) MN-major; N >> 3, M >> 4
  f.idesc = (1u << 4) | (fmt << 7) | (fmt << 10) | (1u << 16) | ((128u >> 3) << 17) | ((128u >> 4) << 24);
  return launch_cluster(gated_tile_kernel<BF16>, tx, tw, f, count * f.shares, mid::THREADS, mid::SMEM, stream);
}

template <bool BF16>
cudaError_t launch_pairs(const GatedProblem &p, const Prepared &q, unsigned *status, cudaStream_t stream) {
  CUtensorMap tx, tw;
  if (!tiles(&tx, &tw, p, q, pair::BM, pair::BK)) return cudaErrorNotSupported;
  const cudaError_t e = attn::allow_smem<gated_pair_kernel<BF16>>(pair::SMEM_BYTES);
  if (e != cudaSuccess) return e;
  pair::Params f = common<pair::Params>(p, q, pair::BK, status);
  f.wide = q.wide;
  f.tiles_m = static_cast<int>((p.tokens + 2 * pair::BM - 1) / (2 * pair::BM));
  f.tiles_f = static_cast<int>((p.d_ff + pair::BF - 1) / pair::BF);
  f.num_tiles = f.tiles_m * f.tiles_f;
  const uint32_t fmt = BF16 ? 1u : 0u;
  // f32 accumulator; B (W) is MN-major; N = 256, M = 256
  f.idesc = (1u << 4) | (fmt << 7) | (fmt << 10) | (1u << 16) | ((256u >> 3) << 17) | ((256u >> 4) << 24);
  const int clusters = f.num_tiles < sm_count() / 2 ? f.num_tiles : sm_count() / 2;  // a pair of SMs each
  gated_pair_kernel<BF16><<<2 * clusters, pair::THREADS, pair::SMEM_BYTES, stream>>>(tx, tw, f);
  return cudaGetLastError();
}

template <bool BF16>
cudaError_t launch_by_tokens(const GatedProblem &p, const Prepared &q, unsigned *status, cudaStream_t stream) {
  if (p.tokens <= 128) return launch_few_tokens<BF16>(p, q, status, stream);
  // The small tiles while all of them have an SM of their own.  512 tokens of 4096 x 1024 (16 pair tiles): 18.7 us, 28.9
  // by pairs; 1000 of 1000 x 1000 (32): 14.8 and 16.7; 256 of 2048 x 5632 (44): 23.3 and 20.8; 512 of 4096 x 4096 (64):
  // 37.5 and 31.2.  Results stored value by value cost the pairs more, whose threads have a row each: with k up to 2048
  // (4096 of 1025 x 2819: 123 us, 166 by pairs; 1000 of 4097 x 2819: 145 and 133).
  const int64_t pairs = (p.tokens + 255) / 256 * ((p.d_ff + 127) / 128);
  const bool small = pairs <= sm_count() / 4 || (!q.wide && p.d_in <= 2048);
  return small ? launch_tiles<BF16>(p, q, status, stream) : launch_pairs<BF16>(p, q, status, stream);
}

} // namespace

cudaError_t launch_gated(const GatedProblem &p, unsigned *status, cudaStream_t stream, int *launched) {
  const gated::Layout l(p);
  Prepared q{p.x, p.w, gated::pitch(p.ldx, p.d_in), gated::pitch(p.ldw, 2 * p.d_ff), gated::pitch(p.ldh, p.d_ff), p.d_ff, true};
  *launched = 1;
  if (l.padded) {
    char *ws = static_cast<char *>(p.workspace);
    cudaError_t e = gated::launch_pad(p.x, q.ldx, ws + l.x, p.tokens, p.d_in, l.d_in, 1, stream);
    if (e == cudaSuccess) e = gated::launch_pad(p.w, q.ldw, ws + l.w, p.d_in, p.d_ff, l.d_ff, 2, stream);
    if (e != cudaSuccess) return e;
    *launched = 3;
    q = Prepared{ws + l.x, ws + l.w, l.d_in, 2 * l.d_ff, q.ldh, l.d_ff, false};
  }
  return p.dtype == kBF16 ? launch_by_tokens<true>(p, q, status, stream) : launch_by_tokens<false>(p, q, status, stream);
}

} // namespace imex
