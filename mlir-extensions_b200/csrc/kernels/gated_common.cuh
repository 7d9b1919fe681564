// What the gated product and its backward pass share: which problems need padded copies, and those.
#pragma once
#include "epilogue.cuh"
#include "tile_sums.cuh"

namespace imex {
namespace gated {

inline int64_t pitch(int64_t ld, int64_t width) { return ld > 0 ? ld : width; }
inline int64_t eights(int64_t n) { return (n + 7) / 8 * 8; }
inline size_t round_up(size_t n) { return (n + 255) / 256 * 256; }

// TMA moves whole 16-byte units.  Where extents or pitches are not multiples of eight, X and W are copied into the
// workspace with rows of such (the up projection's columns starting on one, too) and results are stored value by value.
struct Layout {
  bool padded;
  int64_t d_in, d_ff;            // extents rounded up
  size_t x, w, rest;             // offsets of the copies, and what is behind them
  explicit Layout(const GatedProblem &p, size_t first = 0) {
    padded = p.d_in % 8 || p.d_ff % 8 || p.ldx % 8 || p.ldw % 8 || p.ldh % 8;
    d_in = eights(p.d_in);
    d_ff = eights(p.d_ff);
    x = first;
    w = x + (padded ? round_up(static_cast<size_t>(p.tokens) * d_in * 2) : 0);
    rest = w + (padded ? round_up(static_cast<size_t>(p.d_in) * 2 * d_ff * 2) : 0);
  }
};

// to[rows][segments * wide] = from[rows][segments * cols] with every segment filled up with zeros; eight values a thread
inline __global__ void __launch_bounds__(256)
gated_pad_kernel(const uint16_t *from, int64_t ld, uint16_t *to, int64_t rows, int64_t cols, int64_t wide, int segments) {
  const int64_t per_row = segments * wide / 8, n = rows * per_row;
  for (int64_t e = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x; e < n;
       e += static_cast<int64_t>(gridDim.x) * blockDim.x) {
    const int64_t r = e / per_row, at = (e - r * per_row) * 8, s = at / wide, c = at - s * wide;
    const uint16_t *x = from + r * ld + s * cols + c;
    uint32_t w[4];
#pragma unroll
    for (int k = 0; k < 4; ++k)
      w[k] = (c + 2 * k < cols ? x[2 * k] : 0u) | (c + 2 * k + 1 < cols ? static_cast<uint32_t>(x[2 * k + 1]) << 16 : 0u);
    reinterpret_cast<uint4 *>(to)[e] = make_uint4(w[0], w[1], w[2], w[3]);
  }
}
inline cudaError_t launch_pad(const void *from, int64_t ld, void *to, int64_t rows, int64_t cols, int64_t wide, int segments,
                              cudaStream_t stream) {
  const int64_t blocks = (rows * segments * wide / 8 + 255) / 256, most = tc_host::sm_count() * 8 * 4;
  gated_pad_kernel<<<static_cast<unsigned>(blocks < most ? blocks : most), 256, 0, stream>>>(
      static_cast<const uint16_t *>(from), ld, static_cast<uint16_t *>(to), rows, cols, wide, segments);
  return cudaGetLastError();
}

} // namespace gated
} // namespace imex
