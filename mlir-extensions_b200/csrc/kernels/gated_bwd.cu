// Backward pass of the gated feed-forward product (IMEX_OP_GATED_FFN_BWD).
//
// With [G U] = X W kept by the forward pass, one pass over G, U and dH writes [dG dU] = [dH U act'(G), dH act(G)]
// into the workspace, rounded once to the 16-bit type; because W holds both projections side by side,
// dX = [dG dU] W^T and dW = X^T [dG dU] are then one product each.  Large ones go to the framework's CTA-pair GEMM;
// small ones, and extents that are not multiples of eight, to gated_product_kernel: 128 x 128 tiles, two CTAs per SM, k
// shared out between the CTAs of a cluster where there are few tiles, both products in one grid.
#include "gated_common.cuh"

namespace imex {
namespace {

using namespace attn;
using namespace tc;
using namespace tc_host;

struct GradArgs {
  const uint16_t *gu, *dh;
  uint16_t *dgu;
  int64_t ldh, tokens, d_ff;
  int64_t up;  // first column of dU in dGU, half its row
  int act;
};

// act(g) and its derivative
__device__ __forceinline__ void act_both(float g, int act, float &value, float &slope) {
  if (act == kEpiSilu) {
    const float s = __fdividef(1.0f, 1.0f + __expf(-g));
    value = g * s;
    slope = s * (1.0f + g * (1.0f - s));
  } else if (act == kEpiRelu) {
    value = relu_ugt(g);
    slope = !(g <= 0.0f) ? 1.0f : 0.0f;
  } else {
    value = g;
    slope = 1.0f;
  }
}

// 10 bytes per element of H and few operations: bound by memory.  V columns per thread.
template <bool BF16, int V> __global__ void __launch_bounds__(256) gated_grad_kernel(const GradArgs a) {
  struct alignas(2 * V) Pack {
    uint16_t v[V];
  };
  const int64_t per_row = a.up / V, n = a.tokens * per_row;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  for (int64_t e = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x; e < n;
       e += static_cast<int64_t>(gridDim.x) * blockDim.x) {
    const int64_t r = e / per_row, c = (e - r * per_row) * V, at = r * 2 * a.d_ff + c;
    Pack g{}, u{};
    if (c < a.d_ff) {
      g = *reinterpret_cast<const Pack *>(a.gu + at), u = *reinterpret_cast<const Pack *>(a.gu + at + a.d_ff);
      const Pack d = *reinterpret_cast<const Pack *>(a.dh + r * a.ldh + c);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        float value, slope;
        act_both(to_f32<BF16>(g.v[i]), a.act, value, slope);
        const float dh = to_f32<BF16>(d.v[i]);
        g.v[i] = from_f32<BF16>(dh * to_f32<BF16>(u.v[i]) * slope);
        u.v[i] = from_f32<BF16>(dh * value);
      }
    }
    *reinterpret_cast<Pack *>(a.dgu + r * 2 * a.up + c) = g;
    *reinterpret_cast<Pack *>(a.dgu + r * 2 * a.up + c + a.up) = u;
  }
}

// ---- D[128 x 128 tiles] = A . B, f32 sums, 16-bit results
namespace prod {
constexpr int BK = 64;
constexpr int TILE_BYTES = 128 * 128;          // 128 rows or columns x 64 k
constexpr int STAGE_BYTES = 2 * TILE_BYTES;
constexpr int STAGES = 3;
constexpr int SMEM = STAGES * STAGE_BYTES + 256;
constexpr int THREADS = 256;                   // TMA, products, two idle warps, four that hand the sums over
static_assert(128 * 128 * 4 <= STAGES * STAGE_BYTES, "the sums take the ring's place");
static_assert(2 * (SMEM + 1024) <= 233472, "two CTAs per SM");
struct Product {
  uint16_t *d;
  long long ldd;
  int rows, cols, tiles_n, k_blocks, shares;
  int wide;        // results may be stored 16 bytes at a time
  int half, held;  // columns come in halves of `half`, of which `held` exist and are stored side by side
  uint32_t idesc;
};
struct Params {
  Product of[2];      // dX, dW
  unsigned dx_ctas;   // the first CTAs, whole clusters; clusters have the size of the larger number of shares
  unsigned *status;
};
} // namespace prod

// MN_MAJOR: A is stored [k, rows] and B [k, cols] (X^T dGU); else [rows, k] and [cols, k] (dGU W^T).
template <bool BF16, bool MN_MAJOR>
__device__ __forceinline__ void product_tile(const CUtensorMap &tmap_a, const CUtensorMap &tmap_b, const prod::Product &p,
                                             unsigned cta, unsigned *status, uint8_t *smem_raw) {
  using namespace prod;
  const uint32_t base = smem_u32(smem_raw), bars = base + STAGES * STAGE_BYTES;
  auto full_bar = [&](int s) { return bars + 8u * s; };
  auto empty_bar = [&](int s) { return bars + 8u * (STAGES + s); };
  const uint32_t done = bars + 8u * (2 * STAGES), slot = done + 8;
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const Role me(cta, p.shares);
  const int row0 = me.tile / p.tiles_n * 128, col0 = me.tile % p.tiles_n * 128;
  if (row0 >= p.rows) {
    keep_step(me.shares);
    return;
  }
  const int kb0 = static_cast<int>(static_cast<int64_t>(p.k_blocks) * me.rank / me.shares);
  const int n = static_cast<int>(static_cast<int64_t>(p.k_blocks) * (me.rank + 1) / me.shares) - kb0;

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(full_bar(s), 1);
      mbar_init(empty_bar(s), 1);
    }
    mbar_init(done, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(slot), "r"(128) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tcgen05_fence_before();
  __syncthreads();
  tcgen05_fence_after();
  const uint32_t tmem = *reinterpret_cast<volatile uint32_t *>(smem_raw + (slot - base));

  if (warp == 0) {
    asm volatile("griddepcontrol.wait;" ::: "memory");  // dGU is complete
    if (lane == 0) {
      for (int i = 0; i < n; ++i) {
        const int s = i % STAGES, k = (kb0 + i) * BK;
        if (i >= STAGES && !mbar_wait(empty_bar(s), (i / STAGES - 1) & 1)) {
          report(status, kStatusTmaWaitTimeout);
          break;
        }
        mbar_expect_tx(full_bar(s), STAGE_BYTES);
        const uint32_t a = base + s * STAGE_BYTES, b = a + TILE_BYTES;
        if (MN_MAJOR) {
          tma_load_2d(a, &tmap_a, row0, k, full_bar(s));
          tma_load_2d(a + TILE_BYTES / 2, &tmap_a, row0 + 64, k, full_bar(s));
          tma_load_2d(b, &tmap_b, col0, k, full_bar(s));
          tma_load_2d(b + TILE_BYTES / 2, &tmap_b, col0 + 64, k, full_bar(s));
        } else {
          tma_load_2d(a, &tmap_a, k, row0, full_bar(s));
          tma_load_2d(b, &tmap_b, k, col0, full_bar(s));
        }
      }
      for (int i = max(0, n - STAGES); i < n; ++i)  // everything has been used
        if (!mbar_wait(empty_bar(i % STAGES), (i / STAGES) & 1)) break;
    }
  } else if (warp == 1) {
    const uint32_t leader = elect_one();
    bool ok = true;
    for (int i = 0; i < n && ok; ++i) {
      const int s = i % STAGES;
      ok = __all_sync(0xffffffffu, mbar_wait(full_bar(s), (i / STAGES) & 1));
      if (!ok) break;
      tcgen05_fence_after();
      const uint32_t at = base + s * STAGE_BYTES;
      const uint64_t a = make_smem_desc(at, MN_MAJOR ? TILE_BYTES / 2 : 16, 1024);
      const uint64_t b = make_smem_desc(at + TILE_BYTES, MN_MAJOR ? TILE_BYTES / 2 : 16, 1024);
#pragma unroll
      for (int k = 0; k < BK / 16; ++k) {
        const uint64_t off = (MN_MAJOR ? k * 2048 : k * 32) >> 4;
        mma_ss(tmem, a + off, b + off, p.idesc, (i | k) ? 1u : 0u, leader);
      }
      commit(empty_bar(s), leader);
    }
    if (ok) commit(done, leader);
    else if (lane == 0) report(status, kStatusMmaWaitTimeout);
  }
  if (warp < 4) {
    __syncwarp();
    keep_step(me.shares);  // the other warps' two barriers
  } else {
    const bool ok = __all_sync(0xffffffffu, mbar_wait(done, 0));
    if (ok) {
      tcgen05_fence_after();
      const int lane_group = warp & 3;
      leave_row<128, 128>(tmem + (static_cast<uint32_t>(lane_group * 32) << 16), true, base, lane_group * 32 + lane, 0);
    } else if (lane == 0) {
      report(status, kStatusEpiWaitTimeout);
    }
    sums_barrier<128>(me.shares);
    add_up<128, 128>(base, me.first, me.rank, me.shares, threadIdx.x - 128, [&](int r, int unit, float4 x, float4 y) {
      const int col = col0 + unit * 8;
      if (row0 + r >= p.rows || col >= p.cols) return;
      uint16_t *to = p.d + (row0 + r) * p.ldd;
      if (p.wide) {
        store_unit<BF16>(to + col, x, y, 1.0f);
      } else {
        const float v[8] = {x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int h = col + e < p.half ? 0 : 1, c = col + e - h * p.half;
          if (c < p.held) to[h * p.held + c] = from_f32<BF16>(v[e]);
        }
      }
    });
    sums_barrier<128>(me.shares);
  }
  __syncwarp();
  tcgen05_fence_before();
  __syncthreads();
  if (warp == 1) {
    tcgen05_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(128) : "memory");
  }
}

// The role is the same throughout a cluster: dx_ctas is a multiple of its size.
template <bool BF16>
__global__ void __launch_bounds__(prod::THREADS, 2)
gated_product_kernel(const __grid_constant__ CUtensorMap dx_a, const __grid_constant__ CUtensorMap dx_b,
                     const __grid_constant__ CUtensorMap dw_a, const __grid_constant__ CUtensorMap dw_b,
                     const __grid_constant__ prod::Params p) {
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  if (blockIdx.x < p.dx_ctas) product_tile<BF16, false>(dx_a, dx_b, p.of[0], blockIdx.x, p.status, smem_raw);
  else product_tile<BF16, true>(dw_a, dw_b, p.of[1], blockIdx.x - p.dx_ctas, p.status, smem_raw);
}

// The pair GEMM's 256 x 256 tiles move half as much through shared memory per operation, but they need many tiles and
// a long k to pay: 4096 tokens of 4096 x 11264 (256 and 1408 tiles, k 22528 and 4096): 1.20 ms, 1.38 and 1.57 with dX
// or dW by the small kernel.  300 of 1000 x 2720: 58 us and 23; one of 4096 x 11264 (k of dW 1): 397 and 131; 2048 of
// 4096 x 4096 (512 tiles, k 2048): dW saves 40 of 300 us; 4096 of 2048 x 2048 (128 tiles, k 4096): the same.
bool small_product(const GemmProblem &g) {
  const int64_t tiles = ((g.M + 255) / 256) * ((g.N + 255) / 256);
  return tiles <= 64 || g.K <= 2048 || (tiles <= sm_count() && g.K <= 4096);
}

// Shares of k of a tile: as many CTAs as run at once, at least twenty k blocks each (adding up costs about as much as
// eight), at most four (the clusters of both products have one size).  300 tokens of 1000 x 2720 (dX: 24 tiles, k 5440):
// 28.7 us with two, 22.6 with 4; 128 of 2048 x 5632 (16 tiles, k 11264): 47 us with 8, 43 with 4; one of 4096 x 11264: 150
// and 132; 300 of 640 x 8192 (15 tiles): 36 and 39.
bool prepare_product(CUtensorMap *a, CUtensorMap *b, prod::Product *p, const GemmProblem &g, bool mn_major, bool wide,
                     int64_t half, int64_t held) {
  p->d = reinterpret_cast<uint16_t *>(g.C);
  p->ldd = g.ldc;
  p->rows = static_cast<int>(g.M);
  p->cols = static_cast<int>(g.N);
  p->wide = wide;
  p->half = static_cast<int>(half);
  p->held = static_cast<int>(held);
  p->tiles_n = static_cast<int>((g.N + 127) / 128);
  p->k_blocks = static_cast<int>((g.K + prod::BK - 1) / prod::BK);
  const int64_t tiles = (g.M + 127) / 128 * p->tiles_n;
  p->shares = 1;
  while (p->shares < 4 && tiles * p->shares * 2 <= 2 * sm_count() && p->k_blocks >= 40 * p->shares) p->shares *= 2;
  const uint32_t fmt = g.in_dtype == kBF16 ? 1u : 0u;
  p->idesc = (1u << 4) | (fmt << 7) | (fmt << 10) | (mn_major ? 3u << 15 : 0u) | ((128u >> 3) << 17) | ((128u >> 4) << 24);
  return mn_major ? make_map(a, g.A, g.in_dtype, g.M, g.K, prod::BK, g.lda) && make_map(b, g.B, g.in_dtype, g.N, g.K, prod::BK, g.ldb)
                  : make_map(a, g.A, g.in_dtype, g.K, g.M, 128, g.lda) && make_map(b, g.B, g.in_dtype, g.K, g.N, 128, g.ldb);
}
// The products that `dx` and `dw` ask for, in one grid: dW's CTAs, which do not depend on dX's, fill the places that those
// leave.  after_grad: the grid may start while the kernel that writes dGU, the one before it in the stream, still runs.
template <bool BF16>
cudaError_t launch_products(const GemmProblem *dx, const GemmProblem *dw, bool wide, int64_t d_in, int64_t d_ff_wide, int64_t d_ff,
                            bool after_grad, unsigned *status, cudaStream_t stream) {
  CUtensorMap maps[4] = {};
  prod::Params p{};
  p.status = status;
  p.of[0].shares = p.of[1].shares = 1;
  if ((dx && !prepare_product(&maps[0], &maps[1], &p.of[0], *dx, false, wide, gated::eights(d_in), d_in)) ||
      (dw && !prepare_product(&maps[2], &maps[3], &p.of[1], *dw, true, wide, d_ff_wide, d_ff)))
    return cudaErrorNotSupported;
  const int cluster = p.of[0].shares > p.of[1].shares ? p.of[0].shares : p.of[1].shares;
  auto ctas = [&](const prod::Product &q) {
    return ((q.rows + 127ll) / 128 * q.tiles_n * q.shares + cluster - 1) / cluster * cluster;
  };
  p.dx_ctas = static_cast<unsigned>(ctas(p.of[0]));
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(ctas(p.of[0]) + ctas(p.of[1])));
  cfg.blockDim = dim3(prod::THREADS);
  cfg.dynamicSmemBytes = prod::SMEM;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = static_cast<unsigned>(cluster);
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = after_grad ? 2 : 1;
  const cudaError_t e = allow_smem<gated_product_kernel<BF16>>(prod::SMEM);
  return e != cudaSuccess ? e : cudaLaunchKernelEx(&cfg, gated_product_kernel<BF16>, maps[0], maps[1], maps[2], maps[3], p);
}

} // namespace

namespace {
// dGU, then the padded copies or the GEMM's scratch
size_t dgu_bytes(const GatedProblem &p) {
  return gated::round_up(static_cast<size_t>(p.tokens) * 2 * gated::eights(p.d_ff) * 2);
}
template <bool BF16>
cudaError_t launch_passes(const GatedProblem &p, unsigned *status, cudaStream_t stream, int *launched) {
  const gated::Layout l(p, dgu_bytes(p));
  int64_t ldx = gated::pitch(p.ldx, p.d_in), ldw = gated::pitch(p.ldw, 2 * p.d_ff);
  const int64_t ldh = gated::pitch(p.ldh, p.d_ff), ld_dx = ldx, ld_dw = ldw;
  const void *x = p.x, *w = p.w;
  char *ws = static_cast<char *>(p.workspace);
  uint16_t *dgu = reinterpret_cast<uint16_t *>(ws);
  cudaError_t e;
  *launched = 0;
  if (l.padded) {
    e = gated::launch_pad(x, ldx, ws + l.x, p.tokens, p.d_in, l.d_in, 1, stream);
    if (e == cudaSuccess) e = gated::launch_pad(w, ldw, ws + l.w, p.d_in, p.d_ff, l.d_ff, 2, stream);
    if (e != cudaSuccess) return e;
    *launched = 2;
    x = ws + l.x, w = ws + l.w;
    ldx = l.d_in, ldw = 2 * l.d_ff;
  }
  const GradArgs a{static_cast<const uint16_t *>(p.gu), static_cast<const uint16_t *>(p.h), dgu, ldh, p.tokens, p.d_ff, l.d_ff, p.act};
  const int64_t items = p.tokens * (l.padded ? l.d_ff : l.d_ff / 8);
  const int64_t most = sm_count() * 8 * 4;  // resident blocks, four rounds each at the most
  const unsigned blocks = static_cast<unsigned>((items + 255) / 256 < most ? (items + 255) / 256 : most);
  if (l.padded) gated_grad_kernel<BF16, 1><<<blocks, 256, 0, stream>>>(a);
  else gated_grad_kernel<BF16, 8><<<blocks, 256, 0, stream>>>(a);
  if ((e = cudaGetLastError()) != cudaSuccess) return e;
  ++*launched;

  int n = 1;
  GemmProblem dx;
  dx.in_dtype = dx.out_dtype = p.dtype;
  dx.epilogue = kEpiNone;
  dx.accumulate = false;
  dx.bias = nullptr;
  dx.workspace = ws + l.rest;
  dx.workspace_bytes = gemm_tcgen05_workspace_bytes();
  dx.launched = &n;
  GemmProblem dw = dx;
  // dX[tokens, d_in] = dGU[tokens, 2 d_ff] . W^T, W stored [d_in, 2 d_ff]
  dx.A = dgu, dx.B = w, dx.C = static_cast<float *>(p.dx);
  dx.M = p.tokens, dx.N = p.d_in, dx.K = 2 * l.d_ff;
  dx.lda = 2 * l.d_ff, dx.ldb = ldw, dx.ldc = ld_dx;
  dx.trans_a = false, dx.trans_b = true;
  // dW[d_in, 2 d_ff] = X^T . dGU, X stored [tokens, d_in]
  dw.A = x, dw.B = dgu, dw.C = static_cast<float *>(p.dw);
  dw.M = p.d_in, dw.N = 2 * l.d_ff, dw.K = p.tokens;
  dw.lda = ldx, dw.ldb = 2 * l.d_ff, dw.ldc = ld_dw;
  dw.trans_a = true, dw.trans_b = false;
  const bool small_dx = l.padded || small_product(dx), small_dw = l.padded || small_product(dw);
  if (!small_dx) {
    if ((e = launch_gemm_tcgen05_2cta(dx, status, stream)) != cudaSuccess) return e;
    *launched += n;
  }
  if (small_dx || small_dw) {
    e = launch_products<BF16>(small_dx ? &dx : nullptr, small_dw ? &dw : nullptr, !l.padded, p.d_in, l.d_ff, p.d_ff, small_dx, status, stream);
    if (e != cudaSuccess) return e;
    ++*launched;
  }
  if (!small_dw) {
    n = 1;
    if ((e = launch_gemm_tcgen05_2cta(dw, status, stream)) != cudaSuccess) return e;
    *launched += n;
  }
  return cudaSuccess;
}
} // namespace

size_t gated_bwd_workspace_bytes(const GatedProblem &p) {
  const gated::Layout l(p, dgu_bytes(p));
  return l.rest + (l.padded ? 0 : gemm_tcgen05_workspace_bytes());
}

cudaError_t launch_gated_bwd(const GatedProblem &p, unsigned *status, cudaStream_t stream, int *launched) {
  return p.dtype == kBF16 ? launch_passes<true>(p, status, stream, launched) : launch_passes<false>(p, status, stream, launched);
}

} // namespace imex
