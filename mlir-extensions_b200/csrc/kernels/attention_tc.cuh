// Tensor-core pieces shared by the attention forward and backward kernels (sm_100a): 4-D tile loads,
// TMEM accesses, matrix products of 128-row tiles, packed arithmetic, 2^x.
//
// Tiles are 128 rows x d_head of 16-bit values, held as d_head / 64 boxes of 128 rows x 64 columns
// (128-byte rows, 128B-swizzled), as the 4-D tensor maps (d, row, head, batch) deliver them: rows past the
// end of a sequence read zeros.
#pragma once
#include "attention_common.cuh"
#include "tcgen05_host.h"
#include "tcgen05_ptx.cuh"

namespace imex {
namespace attn {

using namespace tc;
using tc_host::allow_smem;

constexpr int TILE = 128;              // rows of a query or key tile
constexpr int BOX_BYTES = TILE * 128;  // 128 rows x 64 columns

// ---- tile loads ---------------------------------------------------------------------------------
__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap *map, int x, int row, int head, int batch,
                                            uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, "
      "{%2, %3, %4, %5}], [%6];" ::"r"(dst),
      "l"(map), "r"(x), "r"(row), "r"(head), "r"(batch), "r"(bar)
      : "memory");
}
template <int DH, int ROWS = TILE>
__device__ __forceinline__ void load_tile(uint32_t dst, const CUtensorMap *map, int row, int head, int batch,
                                          uint32_t bar) {
#pragma unroll
  for (int j = 0; j < DH / 64; ++j) tma_load_4d(dst + j * (ROWS * 128), map, j * 64, row, head, batch, bar);
}

// ---- products -----------------------------------------------------------------------------------
// One thread issues.  The whole warp walks the code with the issuing thread as a predicate: behind a branch on
// the lane every descriptor would be moved into uniform registers one at a time, which costs more than a
// 128 x 128 x 16 product takes.
__device__ __forceinline__ uint32_t elect_one() {
  uint32_t leader;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(leader));
  return leader;
}
__device__ __forceinline__ void mma_ss(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc,
                                       uint32_t accumulate, uint32_t leader) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "setp.ne.b32 q, %5, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
      "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate), "r"(leader)
      : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc, uint32_t idesc,
                                       uint32_t accumulate, uint32_t leader) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "setp.ne.b32 q, %5, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d_tmem),
      "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate), "r"(leader)
      : "memory");
}
__device__ __forceinline__ void commit(uint32_t bar, uint32_t leader) {
  asm volatile(
      "{\n\t.reg .pred q;\n\t"
      "setp.ne.b32 q, %1, 0;\n\t"
      "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(bar),
      "r"(leader)
      : "memory");
}
// The same for CTA pairs: M 256, both CTAs' shared memory; the commit signals the barrier of both.
__device__ __forceinline__ void mma_pair(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc,
                                         uint32_t accumulate, uint32_t leader) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "setp.ne.b32 q, %5, 0;\n\t"
      "@q tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
      "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate), "r"(leader)
      : "memory");
}
__device__ __forceinline__ void commit_pair(uint32_t bar, uint32_t leader) {
  const uint16_t both = 3;
  asm volatile(
      "{\n\t.reg .pred q;\n\t"
      "setp.ne.b32 q, %2, 0;\n\t"
      "@q tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;\n\t}" ::"r"(bar),
      "h"(both), "r"(leader)
      : "memory");
}
// D[128 x BN] = A . B^T over DH, both tiles in shared memory, rows of d_head values (K-major)
template <int DH, int BN>
__device__ __forceinline__ void mma_scores(uint32_t d_tmem, uint32_t a_smem, uint32_t b_smem, uint32_t idesc,
                                           uint32_t leader) {
  const uint64_t a = make_smem_desc(a_smem, 16, 1024), b = make_smem_desc(b_smem, 16, 1024);
#pragma unroll
  for (int k = 0; k < DH / 16; ++k) {
    const uint64_t ao = ((k >> 2) * BOX_BYTES + (k & 3) * 32) >> 4, bo = ((k >> 2) * (BN * 128) + (k & 3) * 32) >> 4;
    mma_ss(d_tmem, a + ao, b + bo, idesc, k ? 1u : 0u, leader);
  }
}
// D[128 x DH] (+)= P . B over BN; P 16-bit pairs in TMEM, PART values of a row in front of each run of PART columns
// (where as many f32 values were); B a tile in shared memory as it lies (MN-major); the 16-row steps [K0, K1) of it
template <int BN, int PART, int K0 = 0, int K1 = BN / 16>
__device__ __forceinline__ void mma_rows(uint32_t d_tmem, uint32_t p_tmem, uint32_t b_smem, uint32_t idesc,
                                         bool accumulate, uint32_t leader) {
  const uint64_t b = make_smem_desc(b_smem, BN * 128, 1024);
#pragma unroll
  for (int k = K0; k < K1; ++k)
    mma_ts(d_tmem, p_tmem + k / (PART / 16) * PART + k % (PART / 16) * 8, b + static_cast<uint64_t>(k * 2048 >> 4), idesc,
           (accumulate || k) ? 1u : 0u, leader);
}
// c = f32; a, b formats; bit 16: B is MN-major; N >> 3; M >> 4
inline uint32_t instruction_desc(bool bf16, bool b_mn_major, int n) {
  const uint32_t fmt = bf16 ? 1u : 0u;
  return (1u << 4) | (fmt << 7) | (fmt << 10) | ((b_mn_major ? 1u : 0u) << 16) | (static_cast<uint32_t>(n >> 3) << 17) |
         (static_cast<uint32_t>(TILE >> 4) << 24);
}

// ---- TMEM ---------------------------------------------------------------------------------------
__device__ __forceinline__ void tmem_st_16(uint32_t taddr, const uint32_t *r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// ---- arithmetic ---------------------------------------------------------------------------------
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// two f32 -> one word of two 16-bit values (a in the low half), round to nearest even
template <bool BF16> __device__ __forceinline__ uint32_t pack2(float a, float b) {
  uint32_t w;
  if (BF16) asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(w) : "f"(b), "f"(a));
  else asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(w) : "f"(b), "f"(a));
  return w;
}
template <bool BF16> __device__ __forceinline__ float2 unpack2(uint32_t w) {
  return make_float2(to_f32<BF16>(static_cast<uint16_t>(w)), to_f32<BF16>(static_cast<uint16_t>(w >> 16)));
}
// packed arithmetic of sm_100: two f32 per 64-bit register
__device__ __forceinline__ uint64_t pack_f32x2(float lo, float hi) {
  uint64_t w;
  asm("mov.b64 %0, {%1, %2};" : "=l"(w) : "f"(lo), "f"(hi));
  return w;
}
__device__ __forceinline__ uint64_t pack_u32x2(uint32_t lo, uint32_t hi) {
  uint64_t w;
  asm("mov.b64 %0, {%1, %2};" : "=l"(w) : "r"(lo), "r"(hi));
  return w;
}
__device__ __forceinline__ void unpack_f32x2(uint64_t w, float &lo, float &hi) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(w));
}
__device__ __forceinline__ uint64_t fma_f32x2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ uint64_t add_f32x2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ uint64_t mul_f32x2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

// ---- host ---------------------------------------------------------------------------------------
// (d, row, head, batch) map of a 16-bit array with element strides, box [1, box_heads, box_rows, 64].
inline bool make_map_4d(CUtensorMap *m, const void *base, int dtype, int64_t d, int64_t rows, int64_t heads,
                        int64_t batch, const Strides3 &s, int box_rows, int box_heads) {
  auto enc = tc_host::encode_fn();
  if (!enc) return false;
  // the stride of an extent of one is never used, but has to be a legal one
  auto stride = [&](int64_t extent, int64_t step) { return static_cast<cuuint64_t>(extent > 1 ? step : d) * 2; };
  cuuint64_t dims[4] = {static_cast<cuuint64_t>(d), static_cast<cuuint64_t>(rows), static_cast<cuuint64_t>(heads),
                        static_cast<cuuint64_t>(batch)};
  cuuint64_t strides[3] = {stride(rows, s.row), stride(heads, s.head), stride(batch, s.batch)};
  cuuint32_t box[4] = {64, static_cast<cuuint32_t>(box_rows), static_cast<cuuint32_t>(box_heads), 1};
  cuuint32_t estr[4] = {1, 1, 1, 1};
  return enc(m, dtype == kBF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4,
             const_cast<void *>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
             CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

} // namespace attn
} // namespace imex
