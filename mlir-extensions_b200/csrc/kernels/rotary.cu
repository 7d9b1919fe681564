// Rotary positions (IMEX_OP_ROTARY): every pair (a, b) of a head's first rot_dims dimensions becomes
// (a cos t - b sin t, a sin t + b cos t) * factor with t = position * frequency.
//
// The angle is reduced in 64 bits (position * turns, minus its nearest integer: a position of a million
// would leave an f32 product 0.06 rad of rounding) and only then turned into f32 sine and cosine.  They
// are the same for every head, so a block computes them once per token into shared memory and walks the
// token's heads with 16-byte accesses: bound by memory.
#include "attention_common.cuh"

namespace imex {
namespace {

struct RotaryArgs {
  const void *x;
  void *y;
  const int32_t *positions;
  int64_t x_token, x_head, y_token, y_head;
  int heads, pairs, rest, heads_per_block;
  float factor;
  int inverse;
  double turns[128];
};

template <typename T, int N> struct alignas(sizeof(T) * N > 16 ? 16 : sizeof(T) * N) Pack {
  T v[N];
};
__device__ __forceinline__ float widen(float v) { return v; }
__device__ __forceinline__ float widen(__half v) { return __half2float(v); }
__device__ __forceinline__ float widen(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ void narrow(float v, float &o) { o = v; }
__device__ __forceinline__ void narrow(float v, __half &o) { o = __float2half_rn(v); }
__device__ __forceinline__ void narrow(float v, __nv_bfloat16 &o) { o = __float2bfloat16_rn(v); }

// One item = N pairs of one head (or N of its untouched dimensions).
template <typename T, int N, bool INTERLEAVED>
__global__ void __launch_bounds__(256) rotary_kernel(const __grid_constant__ RotaryArgs a) {
  __shared__ float2 cs[128];  // (cos, sin) * factor
  const int64_t token = blockIdx.x;
  const int position = a.positions[token];
  for (int i = threadIdx.x; i < a.pairs; i += blockDim.x) {
    const double turn = static_cast<double>(position) * a.turns[i];
    float s, c;
    sincospif(2.0f * static_cast<float>(turn - rint(turn)), &s, &c);
    cs[i] = make_float2(c * a.factor, (a.inverse ? -s : s) * a.factor);
  }
  __syncthreads();
  const T *x = static_cast<const T *>(a.x) + token * a.x_token;
  T *y = static_cast<T *>(a.y) + token * a.y_token;
  const int per_head = a.pairs / N + a.rest / N;
  const int h0 = blockIdx.y * a.heads_per_block;
  const int items = min(a.heads_per_block, a.heads - h0) * per_head;
  for (int e = threadIdx.x; e < items; e += blockDim.x) {
    const int h = e / per_head, i = (e - h * per_head) * N;
    const T *xh = x + (h0 + h) * a.x_head;
    T *yh = y + (h0 + h) * a.y_head;
    if (i >= a.pairs) {
      const int c = i + a.pairs;
      *reinterpret_cast<Pack<T, N> *>(yh + c) = *reinterpret_cast<const Pack<T, N> *>(xh + c);
      continue;
    }
    if (INTERLEAVED) {
      Pack<T, 2 * N> p = *reinterpret_cast<const Pack<T, 2 * N> *>(xh + 2 * i);
#pragma unroll
      for (int j = 0; j < N; ++j) {
        const float u = widen(p.v[2 * j]), w = widen(p.v[2 * j + 1]);
        const float2 t = cs[i + j];
        narrow(u * t.x - w * t.y, p.v[2 * j]);
        narrow(u * t.y + w * t.x, p.v[2 * j + 1]);
      }
      *reinterpret_cast<Pack<T, 2 * N> *>(yh + 2 * i) = p;
    } else {
      Pack<T, N> p = *reinterpret_cast<const Pack<T, N> *>(xh + i);
      Pack<T, N> q = *reinterpret_cast<const Pack<T, N> *>(xh + i + a.pairs);
#pragma unroll
      for (int j = 0; j < N; ++j) {
        const float u = widen(p.v[j]), w = widen(q.v[j]);
        const float2 t = cs[i + j];
        narrow(u * t.x - w * t.y, p.v[j]);
        narrow(u * t.y + w * t.x, q.v[j]);
      }
      *reinterpret_cast<Pack<T, N> *>(yh + i) = p;
      *reinterpret_cast<Pack<T, N> *>(yh + i + a.pairs) = q;
    }
  }
}

template <typename T, int N> cudaError_t launch_n(const RotaryArgs &a, dim3 grid, int threads, bool inter, cudaStream_t s) {
  if (inter) rotary_kernel<T, N, true><<<grid, threads, 0, s>>>(a);
  else rotary_kernel<T, N, false><<<grid, threads, 0, s>>>(a);
  return cudaGetLastError();
}

// The widest access every row and every part of a head starts and ends on, 16 bytes at most.
template <typename T> cudaError_t launch_typed(RotaryArgs &a, const RotaryProblem &p, cudaStream_t s) {
  int n = 16 / static_cast<int>(sizeof(T));
  auto fits = [&](int m) {
    const int64_t unit = p.interleaved ? 2 * m : m;       // elements of one access
    const int64_t bytes = unit * sizeof(T) > 16 ? 16 : unit * sizeof(T);
    auto at = [&](const void *q) { return reinterpret_cast<uintptr_t>(q) % bytes == 0; };
    const int64_t step = bytes / sizeof(T);
    return a.pairs % m == 0 && a.rest % m == 0 && p.x_token % step == 0 && p.x_head % step == 0 &&
           p.y_token % step == 0 && p.y_head % step == 0 && at(p.x) && at(p.y);
  };
  while (n > 1 && !fits(n)) n /= 2;
  const int per_head = a.pairs / n + a.rest / n;
  // heads of a token are shared out between blocks until there are two blocks per SM
  int64_t splits = 1;
  while (splits < p.heads && p.tokens * splits < 2 * 148) ++splits;
  a.heads_per_block = static_cast<int>((p.heads + splits - 1) / splits);
  const int64_t gy = (p.heads + a.heads_per_block - 1) / a.heads_per_block;
  const int64_t items = static_cast<int64_t>(a.heads_per_block) * per_head;
  const int threads = items >= 256 ? 256 : static_cast<int>((items + 31) / 32 * 32);
  const dim3 grid(static_cast<unsigned>(p.tokens), static_cast<unsigned>(gy));
  if constexpr (sizeof(T) == 2)
    if (n == 8) return launch_n<T, 8>(a, grid, threads, p.interleaved, s);
  if (n == 4) return launch_n<T, 4>(a, grid, threads, p.interleaved, s);
  if (n == 2) return launch_n<T, 2>(a, grid, threads, p.interleaved, s);
  return launch_n<T, 1>(a, grid, threads, p.interleaved, s);
}

} // namespace

const char *rotary_check(const RotaryProblem &p) {
  if (p.dtype != kF32 && p.dtype != kF16 && p.dtype != kBF16) return "the element type is f32, f16 or bf16";
  if (p.tokens < 1 || p.heads < 1 || p.d_head < 1) return "extents are at least 1";
  if (p.rot_dims < 2 || p.rot_dims % 2 || p.rot_dims > 256 || p.rot_dims > p.d_head)
    return "rot_dims is even, 2..256 and at most d_head";
  if (p.tokens > INT32_MAX || p.heads > 65535 || p.d_head > (1 << 20)) return "too many tokens, heads or dimensions";
  if (p.x_token < 0 || p.x_head < 0 || p.y_token < 0 || p.y_head < 0) return "strides are not negative";
  const int64_t e = p.dtype == kF32 ? 4 : 2;
  if (reinterpret_cast<uintptr_t>(p.x) % e || reinterpret_cast<uintptr_t>(p.y) % e ||
      reinterpret_cast<uintptr_t>(p.positions) % 4)
    return "arrays must start on a multiple of their element size";
  // an interleaved pair is read and written as one access
  if (p.interleaved && ((p.x_token | p.x_head | p.y_token | p.y_head) % 2 || reinterpret_cast<uintptr_t>(p.x) % (2 * e) ||
                        reinterpret_cast<uintptr_t>(p.y) % (2 * e)))
    return "interleaved pairs must not straddle: even strides, arrays on a multiple of two elements";
  return nullptr;
}

cudaError_t launch_rotary(const RotaryProblem &p, cudaStream_t stream) {
  RotaryArgs a;
  a.x = p.x, a.y = p.y, a.positions = p.positions;
  a.x_token = p.x_token, a.x_head = p.x_head, a.y_token = p.y_token, a.y_head = p.y_head;
  a.heads = static_cast<int>(p.heads);
  a.pairs = static_cast<int>(p.rot_dims / 2);
  a.rest = static_cast<int>(p.d_head - p.rot_dims);
  a.factor = p.factor;
  a.inverse = p.inverse ? 1 : 0;
  for (int i = 0; i < 128; ++i) a.turns[i] = i < a.pairs ? p.turns[i] : 0.0;
  if (p.dtype == kF32) return launch_typed<float>(a, p, stream);
  if (p.dtype == kF16) return launch_typed<__half>(a, p, stream);
  return launch_typed<__nv_bfloat16>(a, p, stream);
}

} // namespace imex
