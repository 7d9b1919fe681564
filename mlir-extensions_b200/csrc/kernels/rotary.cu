// Rotary positions (IMEX_OP_ROTARY): every pair (a, b) of a head's first rot_dims dimensions becomes
// (a cos t - b sin t, a sin t + b cos t) * factor with t = position * frequency.
//
// The angle is reduced in 64 bits (position * turns, minus its nearest integer: a position of a million
// would leave an f32 product 0.06 rad of rounding) and only then turned into f32 sine and cosine.  They
// are the same for every head, so a block computes them once per token into shared memory and walks the token's
// heads.  Bound by memory: what counts is that enough blocks are resident to cover the chain position - angle -
// barrier - values - store, so a thread holds one item at a time in few registers.
#include "attention_common.cuh"
#include "tcgen05_host.h"

namespace imex {
namespace {

struct RotaryArgs {
  const void *x;
  void *y;
  const int32_t *positions;
  int64_t x_token, x_head, y_token, y_head;
  int64_t tokens;
  int heads, pairs, rest;
  int per_head;         // items of a head
  int lanes;            // threads that share a token: per_head times the heads walked at a time
  int tokens_per_block, heads_per_block;
  float factor;
  int inverse;
  double turns[128];
};

// N neighbouring elements as they lie in memory, moved by one access of 2 to 16 bytes (by plain words: an array of
// __nv_bfloat16 is copied element by element).
template <int BYTES> struct Words;
template <> struct Words<16> { using type = uint4; };
template <> struct Words<8> { using type = uint2; };
template <> struct Words<4> { using type = uint32_t; };
template <> struct Words<2> { using type = uint16_t; };
template <typename T, int N> struct Pack {
  typename Words<N * static_cast<int>(sizeof(T))>::type w;
};
struct F16 { uint16_t bits; };
struct BF16 { uint16_t bits; };

__device__ __forceinline__ uint32_t word(const uint4 &v, int i) { return i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w; }
__device__ __forceinline__ uint32_t word(const uint2 &v, int i) { return i == 0 ? v.x : v.y; }
__device__ __forceinline__ uint32_t word(uint32_t v, int) { return v; }
__device__ __forceinline__ uint32_t word(uint16_t v, int) { return v; }
__device__ __forceinline__ void set_word(uint4 &v, int i, uint32_t x) { (i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w) = x; }
__device__ __forceinline__ void set_word(uint2 &v, int i, uint32_t x) { (i == 0 ? v.x : v.y) = x; }
__device__ __forceinline__ void set_word(uint32_t &v, int, uint32_t x) { v = x; }
__device__ __forceinline__ void set_word(uint16_t &v, int, uint32_t x) { v = static_cast<uint16_t>(x); }

// element j as f32
template <int N> __device__ __forceinline__ float get(const Pack<float, N> &p, int j) { return __uint_as_float(word(p.w, j)); }
template <int N> __device__ __forceinline__ float get(const Pack<F16, N> &p, int j) {
  return attn::to_f32<false>(static_cast<uint16_t>(word(p.w, j / 2) >> (j & 1) * 16));
}
template <int N> __device__ __forceinline__ float get(const Pack<BF16, N> &p, int j) {
  return attn::to_f32<true>(static_cast<uint16_t>(word(p.w, j / 2) >> (j & 1) * 16));
}
// all elements from f32, each rounded once
template <int N> __device__ __forceinline__ void put(Pack<float, N> &p, const float *y) {
#pragma unroll
  for (int j = 0; j < N; ++j) set_word(p.w, j, __float_as_uint(y[j]));
}
__device__ __forceinline__ uint32_t two(F16, float u, float w) {
  uint32_t v;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(v) : "f"(w), "f"(u));
  return v;
}
__device__ __forceinline__ uint32_t two(BF16, float u, float w) {
  uint32_t v;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(v) : "f"(w), "f"(u));
  return v;
}
template <typename T, int N> __device__ __forceinline__ void put(Pack<T, N> &p, const float *y) {
#pragma unroll
  for (int j = 0; j < N; j += 2) set_word(p.w, j / 2, two(T(), y[j], N > 1 ? y[(j + 1) % N] : 0.0f));
}

// One item = N pairs of one head, or N of its untouched dimensions.
template <typename T, int N, bool INTERLEAVED> struct Item {
  // pairs: the first and the second halves (INTERLEAVED: two runs of N elements, which for N = 1 may start anywhere)
  Pack<T, N> a, b;
  __device__ __forceinline__ void load(const T *x, int i, int pairs) {
    if (i >= pairs) {
      a = *reinterpret_cast<const Pack<T, N> *>(x + i + pairs);
    } else if (INTERLEAVED) {
      a = reinterpret_cast<const Pack<T, N> *>(x + 2 * i)[0];
      b = reinterpret_cast<const Pack<T, N> *>(x + 2 * i)[1];
    } else {
      a = *reinterpret_cast<const Pack<T, N> *>(x + i);
      b = *reinterpret_cast<const Pack<T, N> *>(x + i + pairs);
    }
  }
  __device__ __forceinline__ void turn(const float *cos, const float *sin) {
    float c[N], s[N], y[2 * N];
#pragma unroll
    for (int j = 0; j < N; j += 4) {
      if constexpr (N >= 4) {
        const float4 u = *reinterpret_cast<const float4 *>(cos + j), v = *reinterpret_cast<const float4 *>(sin + j);
        c[j] = u.x, c[j + 1] = u.y, c[j + 2] = u.z, c[j + 3] = u.w;
        s[j] = v.x, s[j + 1] = v.y, s[j + 2] = v.z, s[j + 3] = v.w;
      } else {
#pragma unroll
        for (int k = 0; k < N; ++k) c[k] = cos[k], s[k] = sin[k];
      }
    }
#pragma unroll
    for (int j = 0; j < N; ++j) {
      // element e of the pairs in memory order: INTERLEAVED 2j and 2j + 1, else j and N + j
      const int e = INTERLEAVED ? 2 * j : j, f = INTERLEAVED ? 2 * j + 1 : N + j;
      const float u = e < N ? get(a, e % N) : get(b, e % N), w = f < N ? get(a, f % N) : get(b, f % N);
      y[e] = u * c[j] - w * s[j];
      y[f] = u * s[j] + w * c[j];
    }
    put(a, y);
    put(b, y + N);
  }
  __device__ __forceinline__ void store(T *y, int i, int pairs) const {
    if (i >= pairs) {
      *reinterpret_cast<Pack<T, N> *>(y + i + pairs) = a;
    } else if (INTERLEAVED) {
      reinterpret_cast<Pack<T, N> *>(y + 2 * i)[0] = a;
      reinterpret_cast<Pack<T, N> *>(y + 2 * i)[1] = b;
    } else {
      *reinterpret_cast<Pack<T, N> *>(y + i) = a;
      *reinterpret_cast<Pack<T, N> *>(y + i + pairs) = b;
    }
  }
};

// A thread has one place of a head of one token and walks the heads `lanes / per_head` apart.
template <typename T, int N, bool INTERLEAVED>
__global__ void __launch_bounds__(512, 3) rotary_kernel(const __grid_constant__ RotaryArgs a) {
  extern __shared__ float4 shared4[];
  float *cos_sin = reinterpret_cast<float *>(shared4);  // [tokens_per_block][cos, sin][room], times factor
  const int room = (a.pairs + 3) / 4 * 4;
  const int64_t token0 = static_cast<int64_t>(blockIdx.x) * a.tokens_per_block;
  const int tokens = static_cast<int>(min(static_cast<int64_t>(a.tokens_per_block), a.tokens - token0));
  for (int e = threadIdx.x; e < tokens * a.pairs; e += blockDim.x) {
    const int u = e / a.pairs, pair = e - u * a.pairs;
    const double turn = static_cast<double>(a.positions[token0 + u]) * a.turns[pair];
    float s, c;
    sincospif(2.0f * static_cast<float>(turn - rint(turn)), &s, &c);
    cos_sin[2 * u * room + pair] = c * a.factor;
    cos_sin[(2 * u + 1) * room + pair] = (a.inverse ? -s : s) * a.factor;
  }
  __syncthreads();
  const int slot = threadIdx.x / a.lanes, lane = threadIdx.x - slot * a.lanes;
  if (slot >= tokens) return;
  const int h0 = lane / a.per_head, i = (lane - h0 * a.per_head) * N;
  const int h_step = a.lanes / a.per_head, h_first = blockIdx.y * a.heads_per_block;
  const int heads = min(a.heads_per_block, a.heads - h_first);
  const float *cos = cos_sin + 2 * slot * room + i;
  const T *x = static_cast<const T *>(a.x) + (token0 + slot) * a.x_token + (h_first + h0) * a.x_head;
  T *y = static_cast<T *>(a.y) + (token0 + slot) * a.y_token + (h_first + h0) * a.y_head;
  for (int h = h0; h < heads; h += h_step, x += h_step * a.x_head, y += h_step * a.y_head) {
    Item<T, N, INTERLEAVED> item;
    item.load(x, i, a.pairs);
    if (i < a.pairs) item.turn(cos, cos + room);
    item.store(y, i, a.pairs);
  }
}

template <typename T, int N> cudaError_t launch_n(const RotaryArgs &a, dim3 grid, int threads, bool inter, cudaStream_t s) {
  const size_t smem = 2 * static_cast<size_t>(a.tokens_per_block) * ((a.pairs + 3) / 4 * 4) * sizeof(float);
  if (inter) rotary_kernel<T, N, true><<<grid, threads, smem, s>>>(a);
  else rotary_kernel<T, N, false><<<grid, threads, smem, s>>>(a);
  return cudaGetLastError();
}

// The widest access every row and every part of a head starts and ends on, 16 bytes at most.
template <typename T> cudaError_t launch_typed(RotaryArgs &a, const RotaryProblem &p, cudaStream_t s) {
  int n = 16 / static_cast<int>(sizeof(T));
  auto fits = [&](int m) {
    auto at = [&](const void *q) { return reinterpret_cast<uintptr_t>(q) % (m * sizeof(T)) == 0; };
    return a.pairs % m == 0 && a.rest % m == 0 && p.x_token % m == 0 && p.x_head % m == 0 && p.y_token % m == 0 &&
           p.y_head % m == 0 && at(p.x) && at(p.y);
  };
  while (n > 1 && !fits(n)) n /= 2;
  a.per_head = a.pairs / n + a.rest / n;
  // the heads of a token are shared out between blocks until there are two blocks per SM
  int64_t splits = 1;
  while (splits < p.heads && p.tokens * splits < 2 * tc_host::sm_count()) ++splits;
  a.heads_per_block = static_cast<int>((p.heads + splits - 1) / splits);
  const int64_t gy = (p.heads + a.heads_per_block - 1) / a.heads_per_block;
  // about 256 threads (more only where one head has more items), as few rounds over the heads as that allows, evenly
  // filled; several tokens per block when one is small
  int at_once = a.per_head > 256 ? 1 : 256 / a.per_head;
  if (at_once > a.heads_per_block) at_once = a.heads_per_block;
  const int rounds = (a.heads_per_block + at_once - 1) / at_once;
  at_once = (a.heads_per_block + rounds - 1) / rounds;
  a.lanes = at_once * a.per_head;
  a.tokens_per_block = a.lanes > 256 ? 1 : 256 / a.lanes;
  if (a.tokens_per_block > 16) a.tokens_per_block = 16;
  while (a.tokens_per_block > 1 && (p.tokens + a.tokens_per_block - 1) / a.tokens_per_block * gy < 4 * tc_host::sm_count()) --a.tokens_per_block;
  const int threads = (a.lanes * a.tokens_per_block + 31) / 32 * 32;
  const dim3 grid(static_cast<unsigned>((p.tokens + a.tokens_per_block - 1) / a.tokens_per_block), static_cast<unsigned>(gy));
  if constexpr (sizeof(T) == 2)
    if (n == 8) return launch_n<T, 8>(a, grid, threads, p.interleaved, s);
  if (n == 4) return launch_n<T, 4>(a, grid, threads, p.interleaved, s);
  if (n == 2) return launch_n<T, 2>(a, grid, threads, p.interleaved, s);
  return launch_n<T, 1>(a, grid, threads, p.interleaved, s);
}

} // namespace

const char *rotary_check(const RotaryProblem &p, bool pointers) {
  if (p.dtype != kF32 && p.dtype != kF16 && p.dtype != kBF16) return "the element type is f32, f16 or bf16";
  if (p.tokens < 1 || p.heads < 1 || p.d_head < 1) return "extents are at least 1";
  if (p.rot_dims < 2 || p.rot_dims % 2 || p.rot_dims > 256 || p.rot_dims > p.d_head)
    return "rot_dims is even, 2..256 and at most d_head";
  if (p.tokens > INT32_MAX || p.heads > 65535 || p.d_head > 512) return "at most 2^31 - 1 tokens, 65535 heads of 512 dimensions";
  if (p.x_token < 0 || p.x_head < 0 || p.y_token < 0 || p.y_head < 0) return "strides are not negative";
  if (attn::rows_overlap(p.d_head, {{p.y_token, p.tokens}, {p.y_head, p.heads}})) return "the rows of Y overlap";
  if (!pointers) return nullptr;
  const int64_t e = p.dtype == kF32 ? 4 : 2;
  if (reinterpret_cast<uintptr_t>(p.x) % e || reinterpret_cast<uintptr_t>(p.y) % e ||
      reinterpret_cast<uintptr_t>(p.positions) % 4)
    return "arrays must start on a multiple of their element size";
  if (p.x == p.y && ((p.tokens > 1 && p.x_token != p.y_token) || (p.heads > 1 && p.x_head != p.y_head)))
    return "in place, X and Y have the same strides";
  return nullptr;
}

cudaError_t launch_rotary(const RotaryProblem &p, cudaStream_t stream) {
  RotaryArgs a;
  a.x = p.x, a.y = p.y, a.positions = p.positions;
  a.x_token = p.x_token, a.x_head = p.x_head, a.y_token = p.y_token, a.y_head = p.y_head;
  a.tokens = p.tokens;
  a.heads = static_cast<int>(p.heads);
  a.pairs = static_cast<int>(p.rot_dims / 2);
  a.rest = static_cast<int>(p.d_head - p.rot_dims);
  a.factor = p.factor;
  a.inverse = p.inverse ? 1 : 0;
  for (int i = 0; i < 128; ++i) a.turns[i] = i < a.pairs ? p.turns[i] : 0.0;
  if (p.dtype == kF32) return launch_typed<float>(a, p, stream);
  if (p.dtype == kF16) return launch_typed<F16>(a, p, stream);
  return launch_typed<BF16>(a, p, stream);
}

} // namespace imex
