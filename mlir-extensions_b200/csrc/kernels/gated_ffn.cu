// The gated feed-forward product H = act(X Wg) * (X Wu) with W = [Wg | Wu] (IMEX_OP_GATED_FFN) and its
// backward pass (IMEX_OP_GATED_FFN_BWD).
//
// Backward: with [G U] = X W kept by the forward pass, one pass over G, U and dH writes
// [dG dU] = [dH U act'(G), dH act(G)] into the workspace; because W holds both projections side by side,
// dX = [dG dU] W^T and dW = X^T [dG dU] are then one product each of the framework's GEMM.
#include "attention_common.cuh"
#include "epilogue.cuh"

namespace imex {
namespace {

using attn::from_f32;
using attn::to_f32;

struct GatedArgs {
  const uint16_t *x, *w;
  uint16_t *h, *gu;
  int64_t ldx, ldw, ldh;
  int64_t tokens, d_in, d_ff;
  int act;
};

// Any extents: 64 x 64 outputs per block, 4 x 4 of both projections per thread.
template <bool BF16> __global__ void __launch_bounds__(256) gated_tile_kernel(const GatedArgs a) {
  __shared__ float xs[16][64 + 4], gs[16][64 + 4], us[16][64 + 4];
  const int tid = threadIdx.x, tx = tid % 16, ty = tid / 16;
  const int64_t m0 = static_cast<int64_t>(blockIdx.y) * 64, n0 = static_cast<int64_t>(blockIdx.x) * 64;
  float g[4][4] = {}, u[4][4] = {};
  for (int64_t k0 = 0; k0 < a.d_in; k0 += 16) {
    for (int e = tid; e < 64 * 16; e += 256) {
      const int m = e / 16, k = e % 16;
      xs[k][m] = m0 + m < a.tokens && k0 + k < a.d_in ? to_f32<BF16>(a.x[(m0 + m) * a.ldx + k0 + k]) : 0.0f;
    }
    for (int e = tid; e < 16 * 64; e += 256) {
      const int k = e / 64, n = e % 64;
      const bool in = n0 + n < a.d_ff && k0 + k < a.d_in;
      const uint16_t *w = a.w + (k0 + k) * a.ldw + n0 + n;
      gs[k][n] = in ? to_f32<BF16>(w[0]) : 0.0f;
      us[k][n] = in ? to_f32<BF16>(w[a.d_ff]) : 0.0f;
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < 16; ++k)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          g[i][j] = fmaf(xs[k][ty * 4 + i], gs[k][tx * 4 + j], g[i][j]);
          u[i][j] = fmaf(xs[k][ty * 4 + i], us[k][tx * 4 + j], u[i][j]);
        }
    __syncthreads();
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int64_t r = m0 + ty * 4 + i, c = n0 + tx * 4 + j;
      if (r >= a.tokens || c >= a.d_ff) continue;
      a.h[r * a.ldh + c] = from_f32<BF16>(apply_epilogue_fast(g[i][j], a.act) * u[i][j]);
      if (a.gu) {
        a.gu[r * 2 * a.d_ff + c] = from_f32<BF16>(g[i][j]);
        a.gu[r * 2 * a.d_ff + a.d_ff + c] = from_f32<BF16>(u[i][j]);
      }
    }
}

struct GradArgs {
  const uint16_t *gu, *dh;
  uint16_t *dgu;
  int64_t ldh, tokens, d_ff;
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
  const int64_t per_row = a.d_ff / V, n = a.tokens * per_row;
  for (int64_t e = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x; e < n;
       e += static_cast<int64_t>(gridDim.x) * blockDim.x) {
    const int64_t r = e / per_row, c = (e - r * per_row) * V, at = r * 2 * a.d_ff + c;
    Pack g = *reinterpret_cast<const Pack *>(a.gu + at), u = *reinterpret_cast<const Pack *>(a.gu + at + a.d_ff);
    const Pack d = *reinterpret_cast<const Pack *>(a.dh + r * a.ldh + c);
#pragma unroll
    for (int i = 0; i < V; ++i) {
      float value, slope;
      act_both(to_f32<BF16>(g.v[i]), a.act, value, slope);
      const float dh = to_f32<BF16>(d.v[i]);
      g.v[i] = from_f32<BF16>(dh * to_f32<BF16>(u.v[i]) * slope);
      u.v[i] = from_f32<BF16>(dh * value);
    }
    *reinterpret_cast<Pack *>(a.dgu + at) = g;
    *reinterpret_cast<Pack *>(a.dgu + at + a.d_ff) = u;
  }
}

int64_t pitch(int64_t ld, int64_t width) { return ld > 0 ? ld : width; }
size_t dgu_bytes(const GatedProblem &p) { return (static_cast<size_t>(p.tokens) * 2 * p.d_ff * 2 + 255) / 256 * 256; }

// The framework's GEMM on the kernel its shapes ask for.
cudaError_t product(GemmProblem &g, unsigned *status, cudaStream_t stream) {
  if (gemm_tcgen05_2cta_preferred(g)) {
    const cudaError_t e = launch_gemm_tcgen05_2cta(g, status, stream);
    if (e != cudaErrorNotSupported) return e;
  }
  return launch_gemm_simt(g, stream);
}

} // namespace

const char *gated_check(const GatedProblem &p) {
  if (p.dtype != kF16 && p.dtype != kBF16) return "the element type is f16 or bf16";
  if (p.act != kEpiNone && p.act != kEpiRelu && p.act != kEpiSilu) return "unknown activation";
  if (p.tokens < 1 || p.d_in < 1 || p.d_ff < 1) return "extents are at least 1";
  if (p.tokens > (1 << 30) || p.d_in > (1 << 29) || p.d_ff > (1 << 29)) return "extents are at most 2^30 tokens, 2^29 columns";
  if ((p.ldx && p.ldx < p.d_in) || (p.ldw && p.ldw < 2 * p.d_ff) || (p.ldh && p.ldh < p.d_ff))
    return "row pitch smaller than the row";
  return nullptr;
}

size_t gated_bwd_workspace_bytes(const GatedProblem &p) { return dgu_bytes(p) + gemm_tcgen05_workspace_bytes(); }

cudaError_t launch_gated(const GatedProblem &p, unsigned *, cudaStream_t stream, int *launched) {
  GatedArgs a{static_cast<const uint16_t *>(p.x), static_cast<const uint16_t *>(p.w), static_cast<uint16_t *>(p.h),
              static_cast<uint16_t *>(p.gu), pitch(p.ldx, p.d_in), pitch(p.ldw, 2 * p.d_ff), pitch(p.ldh, p.d_ff),
              p.tokens, p.d_in, p.d_ff, p.act};
  const dim3 grid(static_cast<unsigned>((p.d_ff + 63) / 64), static_cast<unsigned>((p.tokens + 63) / 64));
  if (p.dtype == kBF16) gated_tile_kernel<true><<<grid, 256, 0, stream>>>(a);
  else gated_tile_kernel<false><<<grid, 256, 0, stream>>>(a);
  *launched = 1;
  return cudaGetLastError();
}

cudaError_t launch_gated_bwd(const GatedProblem &p, unsigned *status, cudaStream_t stream, int *launched) {
  const int64_t ldx = pitch(p.ldx, p.d_in), ldw = pitch(p.ldw, 2 * p.d_ff), ldh = pitch(p.ldh, p.d_ff);
  uint16_t *dgu = static_cast<uint16_t *>(p.workspace);
  GradArgs a{static_cast<const uint16_t *>(p.gu), static_cast<const uint16_t *>(p.h), dgu, ldh, p.tokens, p.d_ff, p.act};
  auto on16 = [](const void *q) { return (reinterpret_cast<uintptr_t>(q) & 15) == 0; };
  const bool wide = p.d_ff % 8 == 0 && ldh % 8 == 0 && on16(p.gu) && on16(p.h) && on16(dgu);
  const int64_t items = p.tokens * (wide ? p.d_ff / 8 : p.d_ff);
  const int64_t most = 148 * 8 * 4;  // resident blocks, four rounds each at the most
  const unsigned blocks = static_cast<unsigned>((items + 255) / 256 < most ? (items + 255) / 256 : most);
  if (p.dtype == kBF16) {
    if (wide) gated_grad_kernel<true, 8><<<blocks, 256, 0, stream>>>(a);
    else gated_grad_kernel<true, 1><<<blocks, 256, 0, stream>>>(a);
  } else {
    if (wide) gated_grad_kernel<false, 8><<<blocks, 256, 0, stream>>>(a);
    else gated_grad_kernel<false, 1><<<blocks, 256, 0, stream>>>(a);
  }
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return e;
  *launched = 1;
  // dX[tokens, d_in] = dGU[tokens, 2 d_ff] . W^T, W stored [d_in, 2 d_ff]
  int n = 1;
  GemmProblem g;
  g.in_dtype = g.out_dtype = p.dtype;
  g.epilogue = kEpiNone;
  g.accumulate = false;
  g.bias = nullptr;
  g.workspace = reinterpret_cast<char *>(p.workspace) + dgu_bytes(p);
  g.workspace_bytes = gemm_tcgen05_workspace_bytes();
  g.launched = &n;
  g.A = dgu, g.B = p.w, g.C = static_cast<float *>(p.dx);
  g.M = p.tokens, g.N = p.d_in, g.K = 2 * p.d_ff;
  g.lda = 2 * p.d_ff, g.ldb = ldw, g.ldc = ldx;
  g.trans_a = false, g.trans_b = true;
  if ((e = product(g, status, stream)) != cudaSuccess) return e;
  *launched += n;
  // dW[d_in, 2 d_ff] = X^T . dGU, X stored [tokens, d_in]
  n = 1;
  g.A = p.x, g.B = dgu, g.C = static_cast<float *>(p.dw);
  g.M = p.d_in, g.N = 2 * p.d_ff, g.K = p.tokens;
  g.lda = ldx, g.ldb = 2 * p.d_ff, g.ldc = ldw;
  g.trans_a = true, g.trans_b = false;
  if ((e = product(g, status, stream)) != cudaSuccess) return e;
  *launched += n;
  return cudaSuccess;
}

} // namespace imex
