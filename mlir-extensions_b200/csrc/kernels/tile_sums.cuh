// How CTAs hand over a 128-row tile of f32 sums in TMEM: through their shared memory, where the CTAs of a cluster
// that hold parts of the same sums add them up in order, and out as 16-bit rows with neighbouring threads on
// neighbouring addresses.
#pragma once
#include "attention_tc.cuh"

namespace imex {
namespace attn {

// What a CTA does: share `rank` of the `shares` of tile `tile`, which are neighbours in a cluster from its CTA `first` on.
struct Role {
  int tile, rank, shares, first;
  __device__ Role(unsigned cta, int of) : tile(cta / of), rank(cta % of), shares(of), first(0) {
    if (shares > 1) first = static_cast<int>(cluster_ctarank()) - rank;
  }
};
// CTAs that only fill the last cluster keep step with the two barriers of the others' sums.
__device__ __forceinline__ void keep_step(int shares) {
  if (shares > 1) {
    cluster_sync_all();
    cluster_sync_all();
  }
}

// f32 rows of DH values in shared memory, 16-byte units swizzled by the row
template <int DH> __device__ __forceinline__ uint32_t sum_offset(int row, int unit) {
  return row * (DH * 4) + ((unit ^ (row & 7)) * 16);
}
template <int DH, int COLS>
__device__ __forceinline__ void leave_row(uint32_t taddr, bool has, uint32_t sums, int row, int col0) {
#pragma unroll 1
  for (int c = 0; c < COLS; c += 32) {
    uint32_t v[32];
    if (has) {
      tmem_ld_32x32(taddr + c, v);
      tmem_ld_wait();
    }
#pragma unroll
    for (int e = 0; e < 8; ++e)
      st_shared_v4(sums + sum_offset<DH>(row, (col0 + c) / 4 + e),
                   has ? make_float4(__uint_as_float(v[4 * e]), __uint_as_float(v[4 * e + 1]),
                                     __uint_as_float(v[4 * e + 2]), __uint_as_float(v[4 * e + 3]))
                       : make_float4(0.0f, 0.0f, 0.0f, 0.0f));
  }
}
// This CTA's part (share `rank`) of the rows over all shares, in order, which are the cluster's CTAs from `first` on:
// put(row of the tile, unit of eight columns, the eight sums), neighbouring threads on neighbouring units.  `thread` of
// THREADS; the loads of two steps are in flight together.
template <int DH, int S, int THREADS, typename Put>
__device__ __forceinline__ void add_up_of(uint32_t sums, int first, int rank, int thread, Put &&put) {
  constexpr int UNITS = TILE / S * (DH / 8), STEPS = (UNITS + THREADS - 1) / THREADS;
#pragma unroll 2
  for (int k = 0; k < STEPS; ++k) {
    const int u = thread + k * THREADS;
    const int row = rank * (TILE / S) + u / (DH / 8), unit = u % (DH / 8) * 2;
    float4 v[S][2];
#pragma unroll
    for (int r = 0; r < S; ++r)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint32_t at = sums + sum_offset<DH>(u < UNITS ? row : 0, unit + h);
        asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                     : "=f"(v[r][h].x), "=f"(v[r][h].y), "=f"(v[r][h].z), "=f"(v[r][h].w)
                     : "r"(S > 1 ? map_to_cta(at, first + r) : at));
      }
#pragma unroll
    for (int r = 1; r < S; ++r)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        v[0][h].x += v[r][h].x;
        v[0][h].y += v[r][h].y;
        v[0][h].z += v[r][h].z;
        v[0][h].w += v[r][h].w;
      }
    if (u < UNITS) put(row, unit / 2, v[0][0], v[0][1]);
  }
}
template <int DH, int THREADS, typename Put>
__device__ __forceinline__ void add_up(uint32_t sums, int first, int rank, int shares, int thread, Put &&put) {
  if (shares == 1) add_up_of<DH, 1, THREADS>(sums, first, rank, thread, put);
  else if (shares == 2) add_up_of<DH, 2, THREADS>(sums, first, rank, thread, put);
  else add_up_of<DH, 4, THREADS>(sums, first, rank, thread, put);
}
// Eight sums times a factor as 16-bit values
template <bool BF16> __device__ __forceinline__ void store_unit(uint16_t *to, float4 x, float4 y, float factor) {
  *reinterpret_cast<uint4 *>(to) = make_uint4(pack2<BF16>(x.x * factor, x.y * factor), pack2<BF16>(x.z * factor, x.w * factor),
                                              pack2<BF16>(y.x * factor, y.y * factor), pack2<BF16>(y.z * factor, y.w * factor));
}
// The computing warps' sums are in place everywhere / have been read everywhere.  The first warpgroup takes part
// when there are several CTAs.
template <int THREADS> __device__ __forceinline__ void sums_barrier(int shares) {
  __syncwarp();
  if (shares > 1) cluster_sync_all();
  else asm volatile("bar.sync 1, %0;" ::"n"(THREADS) : "memory");
}

} // namespace attn
} // namespace imex
