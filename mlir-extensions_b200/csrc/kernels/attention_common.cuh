// What the attention forward and backward kernels share: the mask, 16-bit conversions, checks.
#pragma once
#include "kernels.h"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <cstdint>
#include <utility>

namespace imex {
namespace attn {

// Whether rows of `width` elements that N (stride, extent) pairs repeat may share elements.
template <int N> bool rows_overlap(int64_t width, std::pair<int64_t, int64_t> (&&steps)[N]) {
  std::sort(steps, steps + N);
  for (const auto &s : steps) {
    if (s.second <= 1) continue;
    if (s.first < width) return true;
    width = s.first > (INT64_MAX - width) / (s.second - 1) ? INT64_MAX : width + s.first * (s.second - 1);
  }
  return false;
}

// Both masks leave a row a prefix of the keys: j < min(key_lens[b], i + n_kv - n_q + 1).
__device__ __forceinline__ int key_count(const int32_t *key_lens, int b, int n_kv) {
  return key_lens ? min(max(key_lens[b], 0), n_kv) : n_kv;
}
__device__ __forceinline__ int visible_keys(int i, int keys, int n_q, int n_kv, int causal) {
  if (!causal) return keys;
  const long long c = static_cast<long long>(i) + n_kv - n_q + 1;
  return static_cast<int>(c < 0 ? 0 : (c < keys ? c : keys));
}

template <bool BF16> __device__ __forceinline__ float to_f32(uint16_t b) {
  return BF16 ? __uint_as_float(static_cast<uint32_t>(b) << 16) : __half2float(__ushort_as_half(b));
}
template <bool BF16> __device__ __forceinline__ uint16_t from_f32(float v) {
  return BF16 ? __bfloat16_as_ushort(__float2bfloat16_rn(v)) : __half_as_ushort(__float2half_rn(v));
}

} // namespace attn
} // namespace imex
