// Attention backward (IMEX_OP_ATTENTION_BWD) on the 5th-generation tensor cores.
//
//   P = 2^(scale log2(e) Q K^T - log2(e) LSE)       dV = sum_group P^T dO
//   dS = P (dO V^T - delta), delta = rowsum(dO O)   dQ = scale dS K,  dK = scale sum_group dS^T Q
//
// Two kinds of tiles, each with its accumulators in TMEM to the end, so that nothing is added up in memory: no
// atomics, no f32 copy of dQ, and the same bits in every run.  The price is that Q K^T and dO V^T are
// computed twice (7 products instead of 5).
//
//   dq_tile    a CTA owns 128 queries (Q, dO stay in shared memory) and walks the key blocks they see.
//   dkv_tile   a CTA owns 128 keys (K, V stay) and walks the query blocks that see them, of every query head
//              that shares the key head.  It works on the transposed products S^T = K Q^T, dP^T = V dO^T (a
//              thread's row is a key), so that P^T and dS^T are A operands from TMEM and dO and Q are used as
//              they lie.
//
// attention_delta_kernel leaves -delta in the workspace, then one grid (attention_grads_kernel) has dQ's tiles in its
// first CTAs and those of dK / dV, which do not depend on them, behind: they fill the SMs that dQ's last round leaves
// idle.  That grid starts while the row sums are still computed; whoever reads them waits for their grid's end itself.
//
// The walked blocks are as long as the head is wide: 128 rows for d_head 128; 64 rows for d_head 64, where a CTA
// then needs half of the TMEM and of the shared memory, so that two run on an SM and fill each other's waits.
//
// Roles as in the forward kernel: warp 0 loads tiles (TMA), warp 1 issues products, warps 4 and up compute, 32
// columns of a row per thread: four warps per scheduler fill each other's waits better than two with 64 columns each
// (4096 causal, d_head 128: 393 us instead of 425).  P and dS take the places of S and dP in TMEM as 16-bit
// pairs (each thread's in front of its own columns, so that no thread overwrites what another still reads);
// products run in the order they are issued, so overwriting a score tile is ordered by issuing the
// next product behind the one that reads it.  While the warps compute P the tensor core runs the
// previous block's last product and this block's dP; while they compute dS it runs the next block's S.
//
// Where there are fewer tiles than SMs, or few long ones (shared key heads make the blocks of a key tile many,
// the causal mask makes them uneven), the blocks of a tile are shared out between the CTAs of a cluster; each
// leaves its sums in its shared memory, and each adds up a part of the rows over all of them, in order.
//
// Rounding: P and dS once to the 16-bit type, results once.  Masked entries are selected away, padded K rows
// zeroed in shared memory where they are a B operand, so padding may hold anything.
#include "attention_tc.cuh"
#include "tile_sums.cuh"

namespace imex {
namespace {

using namespace attn;
using namespace tc;

constexpr unsigned kPollSleepNs = 40;
constexpr float LOG2E = 1.4426950408889634f;

// Sizes by d_head.  BN: rows of a walked block.
template <int DH> struct Sizes {
  static constexpr int BN = DH;
  static constexpr int CTAS = DH == 128 ? 1 : 2;           // per SM
  static constexpr int CPT = 32;                           // columns of a row per computing thread
  static constexpr int PARTS = BN / CPT;                   // threads that share a row
  static constexpr int THREADS = 128 + TILE * PARTS;
  static constexpr int WARPS = 4 * PARTS;                  // that compute
  static constexpr int TMEM_COLS = 4 * BN;
  static constexpr int RB = TILE * DH * 2, TB = BN * DH * 2;  // bytes of a resident tile and of a walked one
  static constexpr int SA = DH == 128 ? 3 : 4, SB = DH == 128 ? 2 : 3;  // stages: Q (dkv) or K (dq); dO or V
  static constexpr int STAT_STAGES = 2;
  static constexpr int STAT_BYTES = STAT_STAGES * 2 * BN * 4;
  static constexpr int BAR_BYTES = 256;
  static constexpr int SMEM = 2 * RB + (SA + SB) * TB + BAR_BYTES + STAT_BYTES;
};
static_assert(Sizes<128>::SMEM <= 232448, "227 KB a CTA");
static_assert(2 * (Sizes<64>::SMEM + 1024) <= 233472, "two CTAs per SM");

struct BwdParams {
  const uint16_t *o, *dout;
  const float *lse;
  float *neg_delta;  // [batch, q_heads, n_q]
  uint16_t *dq, *dk, *dv;
  const int32_t *key_lens;
  unsigned *status;
  Strides3 so, sdo, sdq, sdk, sdv;
  int batch, q_heads, kv_heads, group, n_q, n_kv, causal;
  // CTAs among which the blocks of a tile of dQ, and of dK and dV, are shared out: 1, 2 or 4.  The larger is the size
  // of all clusters of the grid.
  int shares_q, shares_kv;
  unsigned dq_ctas;  // the first CTAs, whole clusters
  float scale, scale_log2e;
  uint32_t idesc_s, idesc_o;
};

// Barriers and buffers of one CTA, the same for both kernels: two resident tiles, a ring of A tiles and one
// of B tiles.
template <int DH> struct Layout : Sizes<DH> {
  using Z = Sizes<DH>;
  static constexpr int SA = Z::SA, SB = Z::SB, TB = Z::TB, RB = Z::RB;
  uint32_t base;
  __device__ explicit Layout(uint32_t b) : base(b) {}
  __device__ uint32_t resident(int i) const { return base + i * RB; }
  __device__ uint32_t a_tile(int i) const { return base + 2 * RB + (i % SA) * TB; }
  __device__ uint32_t b_tile(int i) const { return base + 2 * RB + (SA + i % SB) * TB; }
  __device__ uint32_t bars() const { return base + 2 * RB + (SA + SB) * TB; }
  __device__ uint32_t res_full() const { return bars(); }
  __device__ uint32_t a_full(int i) const { return bars() + 8 * (1 + i % SA); }
  __device__ uint32_t a_empty(int i) const { return bars() + 8 * (1 + SA + i % SA); }
  __device__ uint32_t a_phase(int i) const { return (i / SA) & 1; }
  __device__ uint32_t b_full(int i) const { return bars() + 8 * (1 + 2 * SA + i % SB); }
  __device__ uint32_t b_empty(int i) const { return bars() + 8 * (1 + 2 * SA + SB + i % SB); }
  __device__ uint32_t b_phase(int i) const { return (i / SB) & 1; }
  static constexpr int FIXED = 1 + 2 * SA + 2 * SB;
  __device__ uint32_t bar(int i) const { return bars() + 8 * (FIXED + i); }
  static constexpr int S_FULL = 0, S_READ = 1, DP_FULL = 2, P_READY = 4, DS_READY = 5, DONE = 7, STAT_FULL = 8, STAT_EMPTY = 10;
  static constexpr int TMEM_SLOT = 12;
  static_assert(8 * (FIXED + 13) <= Z::BAR_BYTES, "the barriers fit");
  __device__ uint32_t stats() const { return bars() + Z::BAR_BYTES; }
};

template <int DH> __device__ __forceinline__ void init_barriers(const Layout<DH> &L) {
  using T = Layout<DH>;
  mbar_init(L.res_full(), 1);
  for (int i = 0; i < T::SA; ++i) mbar_init(L.a_full(i), 1), mbar_init(L.a_empty(i), 1);
  for (int i = 0; i < T::SB; ++i) mbar_init(L.b_full(i), 1), mbar_init(L.b_empty(i), 1);
  mbar_init(L.bar(T::S_FULL), 1);
  mbar_init(L.bar(T::S_READ), T::WARPS);
  for (int i = 0; i < 2; ++i) mbar_init(L.bar(T::DP_FULL + i), 1);
  mbar_init(L.bar(T::P_READY), T::WARPS);
  for (int i = 0; i < 2; ++i) mbar_init(L.bar(T::DS_READY + i), T::WARPS);
  mbar_init(L.bar(T::DONE), 1);
  for (int i = 0; i < T::STAT_STAGES; ++i) mbar_init(L.bar(T::STAT_FULL + i), 32), mbar_init(L.bar(T::STAT_EMPTY + i), T::WARPS);
  asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
}

__device__ __forceinline__ void tmem_alloc(uint32_t slot, uint32_t columns) {
  asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(slot), "r"(columns) : "memory");
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_free(uint32_t tmem, uint32_t columns) {
  asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(columns) : "memory");
}
__device__ __forceinline__ uint32_t ld_shared_u32(uint32_t addr) {
  uint32_t v;
  asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ bool wait_all(uint32_t bar, uint32_t parity) {
  return __all_sync(0xffffffffu, mbar_wait(bar, parity));
}

// The computing warpgroups take registers over from the first one; both shares add up to what the threads have at
// launch (65536 over threads and CTAs, in eights).
template <int DH> struct Registers {
  using Z = Sizes<DH>;
  static constexpr int LAUNCH = 65536 / (Z::THREADS * Z::CTAS) / 8 * 8;
  static constexpr int GIVE = 32;
  static constexpr int TAKE = (LAUNCH + (LAUNCH - GIVE) / Z::PARTS) / 8 * 8;
  static_assert(GIVE + Z::PARTS * TAKE <= (1 + Z::PARTS) * LAUNCH, "no more than there are");
};
template <int DH> __device__ __forceinline__ void give_registers() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(Registers<DH>::GIVE));
}
template <int DH> __device__ __forceinline__ void take_registers() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(Registers<DH>::TAKE));
}

// Blocks [share_of(n, r, s), share_of(n, r + 1, s)) are those of share r of s
__device__ __forceinline__ int share_of(int n, int r, int s) { return static_cast<int>(static_cast<int64_t>(n) * r / s); }

// A resident tile of 128 rows, by the boxes of BN rows that the walked blocks use.
template <int DH>
__device__ __forceinline__ void load_resident(uint32_t dst, const CUtensorMap *map, int row, int head, int batch, uint32_t bar) {
  constexpr int BN = Sizes<DH>::BN;
#pragma unroll
  for (int r = 0; r < TILE; r += BN) load_tile<DH, BN>(dst + r * 128, map, row + r, head, batch, bar);
}

// The producer's two streams of tiles, in the order the products use them.
template <int DH, typename LoadA, typename LoadB>
__device__ __forceinline__ void produce(const Layout<DH> &L, int n, unsigned *status, LoadA &&load_a, LoadB &&load_b) {
  using T = Layout<DH>;
  bool ok = true;
  int na = n > 0, nb = n > 0;  // the first of each is on its way already
  auto a = [&]() {
    if (!ok || na >= n) return;
    if (na >= T::SA && !mbar_wait_relaxed(L.a_empty(na), L.a_phase(na) ^ 1u, kPollSleepNs)) {
      ok = false;
      return;
    }
    mbar_expect_tx(L.a_full(na), T::TB);
    load_a(na, L.a_tile(na), L.a_full(na));
    ++na;
  };
  auto b = [&]() {
    if (!ok || nb >= n) return;
    if (nb >= T::SB && !mbar_wait_relaxed(L.b_empty(nb), L.b_phase(nb) ^ 1u, kPollSleepNs)) {
      ok = false;
      return;
    }
    mbar_expect_tx(L.b_full(nb), T::TB);
    load_b(nb, L.b_tile(nb), L.b_full(nb));
    ++nb;
  };
  for (int j = 1; j < n; ++j) {
    a();
    b();
  }
  if (!ok) report(status, kStatusTmaWaitTimeout);
  // every tile has been used before the CTA may go
  for (int q = max(0, na - T::SA); q < na; ++q)
    if (!mbar_wait_relaxed(L.a_empty(q), L.a_phase(q), kPollSleepNs)) break;
  for (int q = max(0, nb - T::SB); q < nb; ++q)
    if (!mbar_wait_relaxed(L.b_empty(q), L.b_phase(q), kPollSleepNs)) break;
}

// N columns of this thread's row
template <int N> __device__ __forceinline__ void load_columns(uint32_t taddr, uint32_t (&v)[N]) {
  uint32_t x[N / 32][32];
#pragma unroll
  for (int c = 0; c < N / 32; ++c) tmem_ld_32x32(taddr + 32 * c, x[c]);
  tmem_ld_wait();
#pragma unroll
  for (int e = 0; e < N; ++e) v[e] = x[e / 32][e % 32];
}
// N / 2 words of pairs in their place
template <int N> __device__ __forceinline__ void store_pairs(uint32_t taddr, const uint32_t (&w)[N / 2]) {
#pragma unroll
  for (int c = 0; c < N / 32; ++c) tmem_st_16(taddr + 16 * c, w + 16 * c);
  tmem_st_wait();
}

// ------------------------------------------------------------------------------------------- row sums
// -rowsum(dO O), DELTA_ROWS rows per warp: DH / 8 lanes read a row together (a lane per row would touch 32 lines with
// every access).
constexpr int DELTA_ROWS = 16;
template <bool BF16, int DH> __global__ void __launch_bounds__(128) attention_delta_kernel(const BwdParams p) {
  constexpr int GROUP = DH / 8, AT_ONCE = 32 / GROUP, N = DELTA_ROWS / AT_ONCE;  // lanes per row, rows per access, accesses
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int per_head = (p.n_q + 4 * DELTA_ROWS - 1) / (4 * DELTA_ROWS), hb = blockIdx.x / per_head;
  const int b = hb / p.q_heads, head = hb % p.q_heads, lane = threadIdx.x & 31;
  const int row0 = (blockIdx.x % per_head * 4 + (threadIdx.x >> 5)) * DELTA_ROWS + lane / GROUP;
  const uint16_t *o = p.o + b * p.so.batch + head * p.so.head + lane % GROUP * 8;
  const uint16_t *g = p.dout + b * p.sdo.batch + head * p.sdo.head + lane % GROUP * 8;
  float *to = p.neg_delta + static_cast<int64_t>(hb) * p.n_q;
  uint4 x[N], y[N];
#pragma unroll
  for (int k = 0; k < N; ++k) {
    const int row = row0 + k * AT_ONCE;
    x[k] = y[k] = make_uint4(0u, 0u, 0u, 0u);
    if (row < p.n_q) {
      x[k] = *reinterpret_cast<const uint4 *>(o + row * p.so.row);
      y[k] = *reinterpret_cast<const uint4 *>(g + row * p.sdo.row);
    }
  }
#pragma unroll
  for (int k = 0; k < N; ++k) {
    const uint32_t xs[4] = {x[k].x, x[k].y, x[k].z, x[k].w}, ys[4] = {y[k].x, y[k].y, y[k].z, y[k].w};
    float d = 0.0f;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float2 u = unpack2<BF16>(xs[e]), w = unpack2<BF16>(ys[e]);
      d = fmaf(u.x, w.x, d);
      d = fmaf(u.y, w.y, d);
    }
#pragma unroll
    for (int s = 1; s < GROUP; s *= 2) d += __shfl_xor_sync(0xffffffffu, d, s);
    const int row = row0 + k * AT_ONCE;
    if (lane % GROUP == 0 && row < p.n_q) to[row] = -d;
  }
}

// ------------------------------------------------------------------------------------------------ dQ
// TMEM, in units of BN columns: S [0,1), dP / dS of even and odd blocks [1,2) [2,3), dQ [3,4).  S is free for the next
// block as soon as it has been read, dP has two places: the scores and products of block j + 1 run while the
// warps still work on block j, so that the warps only ever wait for each other.  A warp may then be a block ahead
// of another one, hence a barrier each for the dS of even and odd blocks; two ahead it cannot be, because the dP of
// block j + 2 comes behind the product over all of dS j.
template <bool BF16, int DH>
__device__ __forceinline__ void dq_tile(const CUtensorMap &tmap_q, const CUtensorMap &tmap_k, const CUtensorMap &tmap_v,
                                        const CUtensorMap &tmap_do, const BwdParams &p, uint8_t *smem_raw) {
  using T = Layout<DH>;
  const T L(smem_u32(smem_raw));
  constexpr int BN = T::BN, CPT = T::CPT;
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const Role me(blockIdx.x, p.shares_q);
  const int heads_batch = p.batch * p.q_heads, hb = me.tile % heads_batch, b = hb / p.q_heads, head = hb % p.q_heads;
  // under the causal mask the long tiles come first
  const int qt = (p.n_q + TILE - 1) / TILE - 1 - me.tile / heads_batch;
  if (qt < 0) {
    keep_step(me.shares);
    return;
  }
  const int row0 = qt * TILE;
  const int keys = key_count(p.key_lens, b, p.n_kv);
  const int n_all = (visible_keys(min(row0 + TILE, p.n_q) - 1, keys, p.n_q, p.n_kv, p.causal) + BN - 1) / BN;
  const int first = share_of(n_all, me.rank, me.shares), n = share_of(n_all, me.rank + 1, me.shares) - first;  // key blocks

  auto load_a = [&](int j, uint32_t dst, uint32_t bar) { load_tile<DH, BN>(dst, &tmap_k, (first + j) * BN, head / p.group, b, bar); };
  auto load_b = [&](int j, uint32_t dst, uint32_t bar) { load_tile<DH, BN>(dst, &tmap_v, (first + j) * BN, head / p.group, b, bar); };
  if (threadIdx.x == 0) {
    init_barriers<DH>(L);
    if (n > 0) {  // the first tiles, while the others set up
      mbar_expect_tx(L.res_full(), 2 * T::RB);
      load_resident<DH>(L.resident(0), &tmap_q, row0, head, b, L.res_full());
      load_resident<DH>(L.resident(1), &tmap_do, row0, head, b, L.res_full());
      mbar_expect_tx(L.a_full(0), T::TB);
      load_a(0, L.a_tile(0), L.a_full(0));
      mbar_expect_tx(L.b_full(0), T::TB);
      load_b(0, L.b_tile(0), L.b_full(0));
    }
  }
  if (warp == 1) tmem_alloc(L.bar(T::TMEM_SLOT), T::TMEM_COLS);
  tcgen05_fence_before();
  __syncthreads();
  tcgen05_fence_after();
  const uint32_t tmem = ld_shared_u32(L.bar(T::TMEM_SLOT));
  const uint32_t dq_tmem = tmem + 3 * BN;
  auto dp_tmem = [&](int j) { return tmem + BN + (j & 1) * BN; };

  if (warp < 4) {
    give_registers<DH>();
    if (warp == 0) {
      if (lane == 0) produce<DH>(L, n, p.status, load_a, load_b);
    } else if (warp == 1 && n > 0) {
      bool ok = wait_all(L.res_full(), 0);
      const uint32_t leader = elect_one();
      const int pad_block = keys < p.n_kv && keys % BN ? keys / BN - first : -1;
      auto scores = [&](int j) {  // S = Q K_j^T
        ok = ok && wait_all(L.a_full(j), L.a_phase(j));
        if (j == pad_block) {  // rows of K behind the sequence's last key: a B operand of dS K
          const int row = keys % BN, count = (BN - row) * 8;  // 16-byte units per box
          for (int e = lane; e < count * (DH / 64); e += 32) {
            const uint32_t at = L.a_tile(j) + (e / count) * (BN * 128) + row * 128 + (e % count) * 16;
            asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(at), "r"(0) : "memory");
          }
          fence_async_smem();
          __syncwarp();
        }
        if (ok) {
          tcgen05_fence_after();
          mma_scores<DH, BN>(tmem, L.resident(0), L.a_tile(j), p.idesc_s, leader);
          commit(L.bar(T::S_FULL), leader);
        }
      };
      auto products = [&](int j) {  // dP = dO V_j^T
        ok = ok && wait_all(L.b_full(j), L.b_phase(j));
        if (ok) {
          tcgen05_fence_after();
          mma_scores<DH, BN>(dp_tmem(j), L.resident(1), L.b_tile(j), p.idesc_s, leader);
          commit(L.bar(T::DP_FULL + (j & 1)), leader);
          commit(L.b_empty(j), leader);
        }
      };
      scores(0);
      products(0);
      for (int j = 0; j < n && ok; ++j) {
        if (j + 1 < n) {
          ok = wait_all(L.bar(T::S_READ), j & 1);
          scores(j + 1);
          products(j + 1);
        }
        ok = ok && wait_all(L.bar(T::DS_READY + (j & 1)), (j >> 1) & 1);
        if (ok) {
          tcgen05_fence_after();
          mma_rows<BN, CPT>(dq_tmem, dp_tmem(j), L.a_tile(j), p.idesc_o, j > 0, leader);
          commit(L.a_empty(j), leader);
        }
      }
      if (ok) commit(L.bar(T::DONE), leader);
      if (lane == 0 && !ok) report(p.status, kStatusMmaWaitTimeout);
    }
    __syncwarp();
    keep_step(me.shares);  // the computing warps' two barriers
  } else {
    take_registers<DH>();
    const int part = (warp - 4) >> 2, lane_group = warp & 3;
    const int r = lane_group * 32 + lane, i = row0 + r;
    const bool exists = i < p.n_q;
    const uint32_t lanes = static_cast<uint32_t>(lane_group * 32) << 16;
    float lse2 = INFINITY, neg_d = 0.0f;
    asm volatile("griddepcontrol.wait;" ::: "memory");  // the row sums are complete
    if (exists) {
      const int64_t row = (static_cast<int64_t>(b) * p.q_heads + head) * p.n_q + i;
      const float lse = p.lse[row];
      if (lse != -INFINITY) lse2 = lse * LOG2E;  // a row that sees no key: every probability is 2^-inf
      neg_d = __ldcg(p.neg_delta + row);
    }
    const int limit = exists ? visible_keys(i, keys, p.n_q, p.n_kv, p.causal) : INT32_MAX;
    const uint64_t scale2 = pack_f32x2(p.scale_log2e, p.scale_log2e), neg_lse2 = pack_f32x2(-lse2, -lse2);
    const uint64_t neg_delta = pack_f32x2(neg_d, neg_d);
    bool ok = true;
    for (int j = 0; j < n; ++j) {
      ok = wait_all(L.bar(T::S_FULL), j & 1);
      if (!ok) break;
      tcgen05_fence_after();
      const int seen = limit - (first + j) * BN - part * CPT;  // of this thread's keys
      const bool masked = __any_sync(0xffffffffu, seen < CPT);
      uint64_t pr[CPT / 2];
      {
        uint32_t s[CPT];
        load_columns<CPT>(tmem + lanes + part * CPT, s);
        tcgen05_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(L.bar(T::S_READ));
        if (masked) {
#pragma unroll
          for (int e = 0; e < CPT; ++e)
            if (e >= seen) s[e] = __float_as_uint(-INFINITY);
        }
#pragma unroll
        for (int e = 0; e < CPT / 2; ++e) {
          float x0, x1;
          unpack_f32x2(fma_f32x2(pack_u32x2(s[2 * e], s[2 * e + 1]), scale2, neg_lse2), x0, x1);
          pr[e] = pack_f32x2(ex2(x0), ex2(x1));
        }
      }
      ok = wait_all(L.bar(T::DP_FULL + (j & 1)), (j >> 1) & 1);
      if (!ok) break;
      tcgen05_fence_after();
      {
        uint32_t d[CPT], w[CPT / 2];
        load_columns<CPT>(dp_tmem(j) + lanes + part * CPT, d);
        if (masked) {  // (P is 0 there, but 0 times the product with a padded row may be NaN)
#pragma unroll
          for (int e = 0; e < CPT; ++e)
            if (e >= seen) d[e] = 0u;
        }
#pragma unroll
        for (int e = 0; e < CPT / 2; ++e) {
          float x0, x1;
          unpack_f32x2(mul_f32x2(pr[e], add_f32x2(pack_u32x2(d[2 * e], d[2 * e + 1]), neg_delta)), x0, x1);
          w[e] = pack2<BF16>(x0, x1);
        }
        // dS takes the place of this thread's own part of dP
        store_pairs<CPT>(dp_tmem(j) + lanes + part * CPT, w);
      }
      tcgen05_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(L.bar(T::DS_READY + (j & 1)));
    }
    if (ok && n > 0) ok = wait_all(L.bar(T::DONE), 0);
    if (!ok) {
      if (lane == 0) report(p.status, kStatusEpiWaitTimeout);
    } else {
      tcgen05_fence_after();
      constexpr int COLS = DH * 4 / T::WARPS;  // a warpgroup's share of the columns
      leave_row<DH, COLS>(dq_tmem + lanes + part * COLS, n > 0, L.base, r, part * COLS);
    }
    constexpr int CT = T::THREADS - 128;
    sums_barrier<CT>(me.shares);
    uint16_t *dq = p.dq + b * p.sdq.batch + head * p.sdq.head + row0 * p.sdq.row;
    add_up<DH, CT>(L.base, me.first, me.rank, me.shares, threadIdx.x - 128, [&](int row, int unit, float4 x, float4 y) {
      if (row0 + row < p.n_q) store_unit<BF16>(dq + row * p.sdq.row + unit * 8, x, y, p.scale);
    });
    sums_barrier<CT>(me.shares);
  }

  __syncwarp();
  tcgen05_fence_before();
  __syncthreads();
  if (warp == 1) {
    tcgen05_fence_after();
    tmem_free(tmem, T::TMEM_COLS);
  }
}

// ------------------------------------------------------------------------------------------- dK and dV
// TMEM, in units of BN columns: S^T / P^T, dP^T / dS^T, dV, dK
template <bool BF16, int DH>
__device__ __forceinline__ void dkv_tile(const CUtensorMap &tmap_q, const CUtensorMap &tmap_k, const CUtensorMap &tmap_v,
                                         const CUtensorMap &tmap_do, const BwdParams &p, uint8_t *smem_raw) {
  using T = Layout<DH>;
  const T L(smem_u32(smem_raw));
  constexpr int BN = T::BN, CPT = T::CPT;
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const Role me(blockIdx.x - p.dq_ctas, p.shares_kv);
  const int heads_batch = p.batch * p.kv_heads, hb = me.tile % heads_batch, b = hb / p.kv_heads, kv_head = hb % p.kv_heads;
  const int key_tile = me.tile / heads_batch;  // under the causal mask the first keys have the most queries
  if (key_tile >= (p.n_kv + TILE - 1) / TILE) {
    keep_step(me.shares);
    return;
  }
  const int key0 = key_tile * TILE;
  const int keys = key_count(p.key_lens, b, p.n_kv);
  // query i sees key j from i = j - (n_kv - n_q) on
  const int shift = p.causal ? p.n_kv - p.n_q : 0;
  const int tiles_q = (p.n_q + BN - 1) / BN;
  const int first_tile = p.causal ? max(0, key0 - shift) / BN : 0;
  const int per_head = key0 < keys ? max(0, tiles_q - first_tile) : 0;
  const int n_all = per_head * p.group, first = share_of(n_all, me.rank, me.shares);
  const int n = share_of(n_all, me.rank + 1, me.shares) - first;
  auto head_of = [&](int j) { return kv_head * p.group + (first + j) / per_head; };
  auto row_of = [&](int j) { return (first_tile + (first + j) % per_head) * BN; };

  auto load_a = [&](int j, uint32_t dst, uint32_t bar) { load_tile<DH, BN>(dst, &tmap_q, row_of(j), head_of(j), b, bar); };
  auto load_b = [&](int j, uint32_t dst, uint32_t bar) { load_tile<DH, BN>(dst, &tmap_do, row_of(j), head_of(j), b, bar); };
  if (threadIdx.x == 0) {
    init_barriers<DH>(L);
    if (n > 0) {  // the first tiles, while the others set up
      mbar_expect_tx(L.res_full(), 2 * T::RB);
      load_resident<DH>(L.resident(0), &tmap_k, key0, kv_head, b, L.res_full());
      load_resident<DH>(L.resident(1), &tmap_v, key0, kv_head, b, L.res_full());
      mbar_expect_tx(L.a_full(0), T::TB);
      load_a(0, L.a_tile(0), L.a_full(0));
      mbar_expect_tx(L.b_full(0), T::TB);
      load_b(0, L.b_tile(0), L.b_full(0));
    }
  }
  if (warp == 1) tmem_alloc(L.bar(T::TMEM_SLOT), T::TMEM_COLS);
  tcgen05_fence_before();
  __syncthreads();
  tcgen05_fence_after();
  const uint32_t tmem = ld_shared_u32(L.bar(T::TMEM_SLOT));
  const uint32_t dp_tmem = tmem + BN, dv_tmem = tmem + 2 * BN, dk_tmem = tmem + 3 * BN;
  float *stats = reinterpret_cast<float *>(smem_raw + (L.stats() - L.base));
  auto stat_of = [&](int j, int which) { return stats + ((j % T::STAT_STAGES) * 2 + which) * BN; };

  if (warp < 4) {
    give_registers<DH>();
    if (warp == 0) {
      if (lane == 0) produce<DH>(L, n, p.status, load_a, load_b);
    } else if (warp == 1 && n > 0) {
      bool ok = wait_all(L.res_full(), 0);
      const uint32_t leader = elect_one();
      auto scores = [&](int j) {  // S^T = K Q_j^T
        ok = ok && wait_all(L.a_full(j), L.a_phase(j));
        if (ok) {
          tcgen05_fence_after();
          mma_scores<DH, BN>(tmem, L.resident(0), L.a_tile(j), p.idesc_s, leader);
          commit(L.bar(T::S_FULL), leader);
        }
      };
      auto products = [&](int j) {  // dP^T = V dO_j^T
        ok = ok && wait_all(L.b_full(j), L.b_phase(j));
        if (ok) {
          tcgen05_fence_after();
          mma_scores<DH, BN>(dp_tmem, L.resident(1), L.b_tile(j), p.idesc_s, leader);
          commit(L.bar(T::DP_FULL), leader);
        }
      };
      scores(0);
      products(0);
      for (int j = 0; j < n && ok; ++j) {
        ok = wait_all(L.bar(T::P_READY), j & 1);
        if (ok) {
          tcgen05_fence_after();
          mma_rows<BN, CPT>(dv_tmem, tmem, L.b_tile(j), p.idesc_o, j > 0, leader);
          commit(L.b_empty(j), leader);
        }
        if (j + 1 < n) scores(j + 1);
        ok = ok && wait_all(L.bar(T::DS_READY), j & 1);
        if (ok) {
          tcgen05_fence_after();
          mma_rows<BN, CPT>(dk_tmem, dp_tmem, L.a_tile(j), p.idesc_o, j > 0, leader);
          commit(L.a_empty(j), leader);
        }
        if (j + 1 < n) products(j + 1);
      }
      if (ok) commit(L.bar(T::DONE), leader);
      if (lane == 0 && !ok) report(p.status, kStatusMmaWaitTimeout);
    } else if (warp == 2) {
      // row statistics of the query blocks: -log2(e) LSE and -delta.  Queries that do not exist or see no key
      // get -inf for the first, which makes their probabilities 2^-inf.
      asm volatile("griddepcontrol.wait;" ::: "memory");  // the row sums are complete
      bool ok = true;
      for (int j = 0; j < n && ok; ++j) {
        const int64_t row = (static_cast<int64_t>(b) * p.q_heads + head_of(j)) * p.n_q;
        const int i0 = row_of(j);
        float s[BN / 32], d[BN / 32];  // fetched before the wait for a free place
#pragma unroll
        for (int e = 0; e < BN / 32; ++e) {
          const int i = i0 + 32 * e + lane;
          s[e] = -INFINITY, d[e] = 0.0f;
          if (i < p.n_q) {
            const float lse = p.lse[row + i];
            if (lse != -INFINITY) s[e] = -lse * LOG2E;
            d[e] = __ldcg(p.neg_delta + row + i);
          }
        }
        if (j >= T::STAT_STAGES) ok = wait_all(L.bar(T::STAT_EMPTY + j % T::STAT_STAGES), (j / T::STAT_STAGES - 1) & 1);
#pragma unroll
        for (int e = 0; e < BN / 32; ++e) {
          stat_of(j, 0)[32 * e + lane] = s[e];
          stat_of(j, 1)[32 * e + lane] = d[e];
        }
        mbar_arrive(L.bar(T::STAT_FULL + j % T::STAT_STAGES));
      }
    }
    __syncwarp();
    keep_step(me.shares);  // the computing warps' two barriers
  } else {
    take_registers<DH>();
    const int part = (warp - 4) >> 2, lane_group = warp & 3;
    const int r = lane_group * 32 + lane, key = key0 + r;
    const uint32_t lanes = static_cast<uint32_t>(lane_group * 32) << 16;
    // first query that sees this thread's key
    const int from = key < keys ? (p.causal ? max(0, key - shift) : 0) : INT32_MAX;
    const uint64_t scale2 = pack_f32x2(p.scale_log2e, p.scale_log2e);
    bool ok = true;
    for (int j = 0; j < n; ++j) {
      ok = wait_all(L.bar(T::STAT_FULL + j % T::STAT_STAGES), (j / T::STAT_STAGES) & 1) && wait_all(L.bar(T::S_FULL), j & 1);
      if (!ok) break;
      tcgen05_fence_after();
      const int i0 = row_of(j) + part * CPT;
      const bool masked = __any_sync(0xffffffffu, from > i0);
      const int hidden = from - i0;  // of this thread's queries, the first ones (0 or less: none)
      uint64_t pr[CPT / 2];
      {
        uint32_t s[CPT], w[CPT / 2];
        load_columns<CPT>(tmem + lanes + part * CPT, s);
        if (masked) {
#pragma unroll
          for (int e = 0; e < CPT; ++e)
            if (e < hidden) s[e] = __float_as_uint(-INFINITY);
        }
        const ulonglong2 *st = reinterpret_cast<const ulonglong2 *>(stat_of(j, 0) + part * CPT);
#pragma unroll
        for (int e = 0; e < CPT / 2; ++e) {
          float x0, x1;
          unpack_f32x2(fma_f32x2(pack_u32x2(s[2 * e], s[2 * e + 1]), scale2, e & 1 ? st[e / 2].y : st[e / 2].x), x0, x1);
          x0 = ex2(x0);
          x1 = ex2(x1);
          pr[e] = pack_f32x2(x0, x1);
          w[e] = pack2<BF16>(x0, x1);
        }
        store_pairs<CPT>(tmem + lanes + part * CPT, w);
      }
      tcgen05_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(L.bar(T::P_READY));
      ok = wait_all(L.bar(T::DP_FULL), j & 1);
      if (!ok) break;
      tcgen05_fence_after();
      {
        uint32_t d[CPT], w[CPT / 2];
        load_columns<CPT>(dp_tmem + lanes + part * CPT, d);
        if (masked) {  // (P is 0 there, but 0 times the product with a padded row may be NaN)
#pragma unroll
          for (int e = 0; e < CPT; ++e)
            if (e < hidden) d[e] = 0u;
        }
        const ulonglong2 *st = reinterpret_cast<const ulonglong2 *>(stat_of(j, 1) + part * CPT);
#pragma unroll
        for (int e = 0; e < CPT / 2; ++e) {
          float x0, x1;
          unpack_f32x2(mul_f32x2(pr[e], add_f32x2(pack_u32x2(d[2 * e], d[2 * e + 1]), e & 1 ? st[e / 2].y : st[e / 2].x)), x0, x1);
          w[e] = pack2<BF16>(x0, x1);
        }
        store_pairs<CPT>(dp_tmem + lanes + part * CPT, w);
      }
      tcgen05_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(L.bar(T::DS_READY));
      if (lane == 0) mbar_arrive(L.bar(T::STAT_EMPTY + j % T::STAT_STAGES));
    }
    if (ok && n > 0) ok = wait_all(L.bar(T::DONE), 0);
    if (!ok) {
      if (lane == 0) report(p.status, kStatusEpiWaitTimeout);
    } else {
      tcgen05_fence_after();
      // the columns of dV and dK, side by side in TMEM, shared out between the warpgroups
      constexpr int COLS = 2 * DH / T::PARTS;
#pragma unroll
      for (int c = 0; c < COLS; c += DH < COLS ? DH : COLS) {
        const int col = part * COLS + c;
        leave_row<DH, (DH < COLS ? DH : COLS)>(dv_tmem + lanes + col, n > 0, L.base + col / DH * (TILE * DH * 4), r, col % DH);
      }
    }
    // dK and dV may have the place of O, which the row sums' kernel reads: a tile that no query sees gets here at once
    asm volatile("griddepcontrol.wait;" ::: "memory");
    constexpr int CT = T::THREADS - 128;
    sums_barrier<CT>(me.shares);
    uint16_t *dv = p.dv + b * p.sdv.batch + kv_head * p.sdv.head + key0 * p.sdv.row;
    uint16_t *dk = p.dk + b * p.sdk.batch + kv_head * p.sdk.head + key0 * p.sdk.row;
    add_up<DH, CT>(L.base, me.first, me.rank, me.shares, threadIdx.x - 128, [&](int row, int unit, float4 x, float4 y) {
      if (key0 + row < p.n_kv) store_unit<BF16>(dv + row * p.sdv.row + unit * 8, x, y, 1.0f);
    });
    add_up<DH, CT>(L.base + TILE * DH * 4, me.first, me.rank, me.shares, threadIdx.x - 128, [&](int row, int unit, float4 x, float4 y) {
      if (key0 + row < p.n_kv) store_unit<BF16>(dk + row * p.sdk.row + unit * 8, x, y, p.scale);
    });
    sums_barrier<CT>(me.shares);
  }

  __syncwarp();
  tcgen05_fence_before();
  __syncthreads();
  if (warp == 1) {
    tcgen05_fence_after();
    tmem_free(tmem, T::TMEM_COLS);
  }
}

// The role is the same throughout a cluster: dq_ctas is a multiple of its size.
template <bool BF16, int DH>
__global__ void __launch_bounds__(Sizes<DH>::THREADS, Sizes<DH>::CTAS)
attention_grads_kernel(const __grid_constant__ CUtensorMap tmap_q, const __grid_constant__ CUtensorMap tmap_k,
                       const __grid_constant__ CUtensorMap tmap_v, const __grid_constant__ CUtensorMap tmap_do,
                       const __grid_constant__ BwdParams p) {
  extern __shared__ __align__(1024) uint8_t smem_raw[];  // swizzled tiles start on 1024 bytes
  if (blockIdx.x < p.dq_ctas) dq_tile<BF16, DH>(tmap_q, tmap_k, tmap_v, tmap_do, p, smem_raw);
  else dkv_tile<BF16, DH>(tmap_q, tmap_k, tmap_v, tmap_do, p, smem_raw);
}

// CTAs a tile's `blocks` are shared out between, at least `least` blocks each and at most four (clusters of eight CTAs
// that fill their SMs wait long for a place): until they are about as long as the part of `total`, the blocks of dQ and
// of dK / dV, that one of `slots` CTAs has; two shares sooner for the uneven tiles of the causal mask.  Tiles longer than
// the other kind's (shared key heads) come behind all of those, so they are cut finer.  Shares of dQ, dK / dV:
// 1024 x 1024, 8 heads of 64: 32 us with 4, 4, 22.5 with 2, 2; 1000 x 1000 causal, 16 heads on 4 of 128: 49 us with 2, 4,
// 37 with 1, 4; 1000 x 1000, 32 on 8 of 64: 63 us with 1, 2, 55 with 1, 4; 8 of 512 x 512 causal, 32 on 4 of 64: 86 with
// 1, 2, 90 with 1, 4.
int share_count(int64_t blocks, int64_t total, int64_t slots, int least, bool causal, bool longer) {
  int s = 1;
  while (s < 4 && blocks >= least * 2 * s && 10 * blocks * slots * (causal && s == 1 ? 2 : 1) > (longer ? 11 : 16) * total * s) s *= 2;
  return s;
}

template <bool BF16, int DH>
cudaError_t launch_both(const CUtensorMap &tq, const CUtensorMap &tk, const CUtensorMap &tv, const CUtensorMap &tdo,
                        BwdParams f, int64_t batch, cudaStream_t stream) {
  using Z = Sizes<DH>;
  const int64_t slots = tc_host::sm_count() * Z::CTAS;
  const int64_t tiles_q = (f.n_q + TILE - 1) / TILE, tiles_kv = (f.n_kv + TILE - 1) / TILE;
  const int64_t blocks_kv = (f.n_kv + Z::BN - 1) / Z::BN, blocks_q = static_cast<int64_t>((f.n_q + Z::BN - 1) / Z::BN) * f.group;
  const int64_t total = batch * (f.q_heads * tiles_q * blocks_kv + f.kv_heads * tiles_kv * blocks_q);
  f.shares_q = share_count(blocks_kv, total, slots, DH == 64 ? 2 : 4, f.causal, false);
  f.shares_kv = share_count(blocks_q, total, slots, DH == 64 ? 2 : 4, f.causal, blocks_q > blocks_kv);
  const int cluster = f.shares_q > f.shares_kv ? f.shares_q : f.shares_kv;
  auto ctas = [&](int64_t tiles, int shares) { return (tiles * shares + cluster - 1) / cluster * cluster; };
  const int64_t dq_ctas = ctas(batch * f.q_heads * tiles_q, f.shares_q);
  f.dq_ctas = static_cast<unsigned>(dq_ctas);

  const int64_t chunks = (f.n_q + 4 * DELTA_ROWS - 1) / (4 * DELTA_ROWS);
  attention_delta_kernel<BF16, DH><<<static_cast<unsigned>(chunks * batch * f.q_heads), 128, 0, stream>>>(f);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return e;
  // May start while the row sums are still computed.  Its first tiles of Q, K, V and dO are loaded before its wait for
  // them: the row sums' kernel is an ordinary launch, so whatever wrote those was complete before it began.
  e = allow_smem<attention_grads_kernel<BF16, DH>>(Z::SMEM, Registers<DH>::LAUNCH);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(dq_ctas + ctas(batch * f.kv_heads * tiles_kv, f.shares_kv)));
  cfg.blockDim = dim3(Z::THREADS);
  cfg.dynamicSmemBytes = Z::SMEM;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = static_cast<unsigned>(cluster);
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  return cudaLaunchKernelEx(&cfg, attention_grads_kernel<BF16, DH>, tq, tk, tv, tdo, f);
}

} // namespace

cudaError_t launch_attention_bwd(const AttentionProblem &p, unsigned *status, cudaStream_t stream, int *launched) {
  const bool bf16 = p.dtype == kBF16;
  const int rows = static_cast<int>(p.d_head);  // BN
  CUtensorMap tq, tk, tv, tdo;
  if (!make_map_4d(&tq, p.q, p.dtype, p.d_head, p.n_q, p.q_heads, p.batch, p.sq, rows, 1) ||
      !make_map_4d(&tdo, p.dout, p.dtype, p.d_head, p.n_q, p.q_heads, p.batch, p.sdo, rows, 1) ||
      !make_map_4d(&tk, p.k, p.dtype, p.d_head, p.n_kv, p.kv_heads, p.batch, p.sk, rows, 1) ||
      !make_map_4d(&tv, p.v, p.dtype, p.d_head, p.n_kv, p.kv_heads, p.batch, p.sv, rows, 1))
    return cudaErrorNotSupported;
  BwdParams f{};
  f.o = static_cast<const uint16_t *>(p.o);
  f.dout = static_cast<const uint16_t *>(p.dout);
  f.lse = p.lse;
  f.neg_delta = static_cast<float *>(p.workspace);
  f.dq = static_cast<uint16_t *>(p.dq);
  f.dk = static_cast<uint16_t *>(p.dk);
  f.dv = static_cast<uint16_t *>(p.dv);
  f.key_lens = p.key_lens;
  f.status = status;
  f.so = p.so, f.sdo = p.sdo, f.sdq = p.sdq, f.sdk = p.sdk, f.sdv = p.sdv;
  f.batch = static_cast<int>(p.batch);
  f.q_heads = static_cast<int>(p.q_heads);
  f.kv_heads = static_cast<int>(p.kv_heads);
  f.group = static_cast<int>(p.q_heads / p.kv_heads);
  f.n_q = static_cast<int>(p.n_q);
  f.n_kv = static_cast<int>(p.n_kv);
  f.causal = p.causal ? 1 : 0;
  f.scale = p.scale;
  f.scale_log2e = p.scale * LOG2E;
  f.idesc_s = instruction_desc(bf16, false, static_cast<int>(p.d_head));  // BN is d_head
  f.idesc_o = instruction_desc(bf16, true, static_cast<int>(p.d_head));
  *launched = 2;
  if (p.d_head == 64)
    return bf16 ? launch_both<true, 64>(tq, tk, tv, tdo, f, p.batch, stream)
                : launch_both<false, 64>(tq, tk, tv, tdo, f, p.batch, stream);
  return bf16 ? launch_both<true, 128>(tq, tk, tv, tdo, f, p.batch, stream)
              : launch_both<false, 128>(tq, tk, tv, tdo, f, p.batch, stream);
}

} // namespace imex
