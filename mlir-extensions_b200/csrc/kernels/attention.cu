// Attention forward with row statistics (IMEX_OP_ATTENTION) on the 5th-generation tensor cores:
// S = Q K^T, P = 2^(scale log2(e) S - m), O += P V in one pass over the visible keys, with a reference
// maximum m per row that moves only when the row's maximum outgrows it by more than 2^8 (only then are O, in
// TMEM, and the running sum l rescaled); at the end O / l and LSE = ln 2 (m + log2 l).
//
// Both masks leave every row a prefix of the keys, so a tile stops at the last key any of its rows sees and only
// the blocks behind the first row's prefix compare indices.
//
// A tile is 128 query rows of one head, or, when all n_q rows of all query heads of a key head fit into one
// (n_q * group <= 128: decoding, short chunks), those ("packed").
//
//   d_head 64    a CTA holds one tile and half of the SM's TMEM and shared memory, so that two run on an SM. P has
//                TMEM columns of its own, so the next block's scores are computed while the warps still work on
//                this one.
//   d_head 128   S, P and O leave no such room.  A CTA runs two streams instead, each with its own scores S
//                (128 x 128 f32 in TMEM, P takes its place as 16-bit pairs) and accumulator O, so that the tensor
//                core works for one while the other computes exponentials.  The streams are two neighbouring
//                tiles that share every K and V tile ("paired"), or, packed, both hold the one tile and take
//                every other key block; they are merged at the end.
//
// When there are fewer tiles than SMs, or packed ones leave the last round of CTAs nearly empty, the key blocks of a
// tile are shared out between `splits` CTAs, which leave O (unnormalised), m and l in the workspace;
// attention_join_kernel adds them up in order.
//
//   warp 0      TMA producer: Q, then K and V tiles through one ring in the order the products use them.
//   warp 1      issues the products.  Per stream and block: wait for P, O += P V, S = Q K^T of the next
//               block.  Products run in the order they are issued, so one barrier (`scores`) tells the stream
//               that its next scores are there AND that P V before them is done.
//   warps 4-11  stream (warp - 4) / 4, one query row per thread: no shuffles, no exchange.  A row's 128 scores
//               sit in registers, so these two warpgroups take registers over from the first one
//               (72 + 2 * 216 = 3 * 168 a thread at launch).
//
// Rounding: P once to the 16-bit type (l and LSE add up the unrounded values), O once at the end.
// V rows between key_lens[b] and the end of its tile are zeroed in shared memory, so that padding may hold
// anything (0 * NaN would reach the sum); masked scores are selected away.
// Every wait is bounded; one that runs out records a status code and the role leaves its loop.
#include "attention_tc.cuh"

#include <type_traits>

namespace imex {
namespace {

using namespace attn;
using namespace tc;

constexpr int THREADS = 384;
constexpr int REGISTERS = 168;  // a thread at launch, handed over as 72 + 2 * 216
constexpr unsigned kPollSleepNs = 40;
// TMEM columns: S_0 [0,128) S_1 [128,256) O_0 [256,384) O_1 [384,512)
constexpr int TMEM_COLS = 512;
constexpr int O_COL = 256;

constexpr int STAGES = 5;  // K / V tiles of 32 KB beside one (packed) or two (paired) of Q
__host__ __device__ constexpr int q_tiles(bool packed) { return packed ? 1 : 2; }
constexpr int MERGE_BYTES = 2 * TILE * 8;
constexpr int smem_bytes(bool packed) {
  return (q_tiles(packed) + STAGES) * TILE * 256 + 256 + (packed ? MERGE_BYTES : 0);
}

struct FwdParams {
  uint16_t *o;
  float *lse;
  const int32_t *key_lens;
  float *part_o;   // [splits][rows of the problem][DH], unnormalised
  float2 *part_ml; // [splits][rows of the problem]
  unsigned *status;
  Strides3 so;
  int q_heads, group, n_q, n_kv, causal;
  int heads_batch, heads, tiles_q, splits;  // heads: q_heads (paired) or kv_heads (packed)
  int64_t rows;                             // batch * q_heads * n_q
  float scale_log2e;
  uint32_t idesc_s, idesc_o;
};

// What one CTA does.
struct Work {
  int b, head, qt, split;
  int keys;       // keys of the sequence
  int kb0;        // first key block
  int n[2];       // blocks of each stream
};

template <bool PACKED> __device__ __forceinline__ Work work_of(const FwdParams &p) {
  Work w;
  const int hb = blockIdx.x % p.heads_batch, rest = blockIdx.x / p.heads_batch;
  w.b = hb / p.heads;
  w.head = hb % p.heads;
  w.split = rest % p.splits;
  w.qt = p.tiles_q - 1 - rest / p.splits;  // under the causal mask the long tiles come first
  w.keys = key_count(p.key_lens, w.b, p.n_kv);
  auto blocks = [&](int row0, int rows) {  // key blocks that rows [row0, row0 + rows) see
    if (row0 >= p.n_q) return 0;
    return (visible_keys(min(row0 + rows, p.n_q) - 1, w.keys, p.n_q, p.n_kv, p.causal) + TILE - 1) / TILE;
  };
  if (PACKED) {
    const int nb = blocks(0, p.n_q);
    w.kb0 = static_cast<int>(static_cast<int64_t>(nb) * w.split / p.splits);
    const int mine = static_cast<int>(static_cast<int64_t>(nb) * (w.split + 1) / p.splits) - w.kb0;
    w.n[0] = (mine + 1) / 2;
    w.n[1] = mine / 2;
  } else {
    const int n0 = blocks(w.qt * 2 * TILE, TILE), n1 = blocks(w.qt * 2 * TILE + TILE, TILE), nb = max(n0, n1);
    w.kb0 = static_cast<int>(static_cast<int64_t>(nb) * w.split / p.splits);
    const int kb1 = static_cast<int>(static_cast<int64_t>(nb) * (w.split + 1) / p.splits);
    w.n[0] = max(0, min(n0, kb1) - w.kb0);
    w.n[1] = max(0, min(n1, kb1) - w.kb0);
  }
  return w;
}

// ---- one block of a row's keys, a row per thread -----------------------------------------------------
// Scores of keys the row does not see become -inf; seen: of this block's keys, may be negative or large.
__device__ __forceinline__ void mask_scores(uint32_t (&s)[4][32], int seen) {
  if (__any_sync(0xffffffffu, seen < TILE)) {
#pragma unroll
    for (int c = 0; c < 4; ++c)
#pragma unroll
      for (int e = 0; e < 32; ++e)
        if (32 * c + e >= seen) s[c][e] = __float_as_uint(-INFINITY);
  }
}
__device__ __forceinline__ float row_maximum(const uint32_t (&s)[4][32]) {
  float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
  for (int c = 0; c < 4; ++c)
#pragma unroll
    for (int e = 0; e < 32; e += 2) top[c] = max3(top[c], __uint_as_float(s[c][e]), __uint_as_float(s[c][e + 1]));
  return fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
}
// Moves the reference maximum where the row's outgrows it by more than 2^8: O and l shrink by 2^(m - row_max).
// O must not be in use by a product.
template <int DH> __device__ __forceinline__ void move_reference(float &m, float &l, float row_max, uint32_t o_addr) {
  const bool move = row_max > m + 8.0f;
  if (!__any_sync(0xffffffffu, move)) return;
  const float a = move ? ex2(m - row_max) : 1.0f;
#pragma unroll 1
  for (int c = 0; c < DH; c += 32) {
    uint32_t v[32];
    tmem_ld_32x32(o_addr + c, v);
    tmem_ld_wait();
#pragma unroll
    for (int e = 0; e < 32; ++e) v[e] = __float_as_uint(__uint_as_float(v[e]) * a);
    tmem_st_16(o_addr + c, v);
    tmem_st_16(o_addr + c + 16, v + 16);
  }
  l *= a;
  if (move) m = row_max;
}
// P = 2^(scale s - m) as 16-bit pairs to p_addr; ready(half) after each 64 keys; returns the sum of P.
template <bool BF16, typename Ready>
__device__ __forceinline__ float exponentials(const uint32_t (&s)[4][32], float scale_log2e, float m, uint32_t p_addr,
                                              Ready &&ready) {
  const float m_safe = m == -INFINITY ? 0.0f : m;  // a row without a visible key: every exponent is -inf
  const uint64_t scale2 = pack_f32x2(scale_log2e, scale_log2e), neg_m2 = pack_f32x2(-m_safe, -m_safe);
  uint64_t sum[2] = {0ull, 0ull};
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    uint32_t pw[16];
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      float x0, x1;
      unpack_f32x2(fma_f32x2(pack_u32x2(s[c][2 * e], s[c][2 * e + 1]), scale2, neg_m2), x0, x1);
      const float e0 = ex2(x0), e1 = ex2(x1);
      sum[e & 1] = add_f32x2(sum[e & 1], pack_f32x2(e0, e1));
      pw[e] = pack2<BF16>(e0, e1);
    }
    tmem_st_16(p_addr + 16 * c, pw);
    if (c & 1) {
      tmem_st_wait();
      tcgen05_fence_before();
      __syncwarp();
      ready(c >> 1);
    }
  }
  float lo, hi;
  unpack_f32x2(add_f32x2(sum[0], sum[1]), lo, hi);
  return lo + hi;
}
// A row sees no key where the sum is 0; where a score is NaN or +inf it is NaN, and so are LSE and the row.
__device__ __forceinline__ bool sees_any(float l) { return !(l == 0.0f); }
__device__ __forceinline__ float row_lse(float m, float l) {
  return sees_any(l) ? 0.6931471805599453f * (m + log2f(l)) : -INFINITY;
}
// Results go out through shared memory, where Q was: a thread puts its row there as 16-bit units of 16 bytes
// (swizzled by the row), then the warp writes its 32 rows with neighbouring lanes on neighbouring units.
template <bool BF16>
__device__ __forceinline__ void stage_32(uint32_t row_addr, int row, int unit, const float (&x)[32]) {
#pragma unroll
  for (int e = 0; e < 4; ++e)
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(row_addr + (((unit + e) ^ (row & 7)) * 16)),
                 "r"(pack2<BF16>(x[8 * e], x[8 * e + 1])), "r"(pack2<BF16>(x[8 * e + 2], x[8 * e + 3])),
                 "r"(pack2<BF16>(x[8 * e + 4], x[8 * e + 5])), "r"(pack2<BF16>(x[8 * e + 6], x[8 * e + 7]))
                 : "memory");
}
// units [unit0, unit0 + UNITS) of the 32 rows from row0; where(row) is the row's place in O or nullptr
template <int DH, int UNITS, typename Where>
__device__ __forceinline__ void write_rows(uint32_t stage, int row0, int unit0, int lane, Where &&where) {
  __syncwarp();
#pragma unroll 4
  for (int k = 0; k < UNITS; ++k) {
    const int row = row0 + (k * 32 + lane) / UNITS, unit = unit0 + (k * 32 + lane) % UNITS;
    uint4 v;
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                 : "r"(stage + row * (DH * 2) + ((unit ^ (row & 7)) * 16)));
    uint16_t *to = where(row);
    if (to) *reinterpret_cast<uint4 *>(to + unit * 8) = v;
  }
}
// 32 f32 values of a split's row into the workspace
template <int DH>
__device__ __forceinline__ void store_part(const FwdParams &p, const float (&x)[32], int split, int64_t row, int c) {
  float4 *to = reinterpret_cast<float4 *>(p.part_o + (split * p.rows + row) * DH + c);
#pragma unroll
  for (int e = 0; e < 8; ++e) to[e] = make_float4(x[4 * e], x[4 * e + 1], x[4 * e + 2], x[4 * e + 3]);
}
// Rows [first, TILE) of a tile in shared memory to zero, by a whole warp, before products read them
template <int DH> __device__ __forceinline__ void zero_rows(uint32_t tile, int first, int lane) {
  const int count = (TILE - first) * 8;  // 16-byte units per box
  for (int e = lane; e < count * (DH / 64); e += 32) {
    const uint32_t at = tile + (e / count) * BOX_BYTES + first * 128 + (e % count) * 16;
    asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(at), "r"(0) : "memory");
  }
  fence_async_smem();
  __syncwarp();
}

template <bool BF16, bool PACKED>
__global__ void __launch_bounds__(THREADS, 1)
attention_kernel(const __grid_constant__ CUtensorMap tmap_q, const __grid_constant__ CUtensorMap tmap_k,
                 const __grid_constant__ CUtensorMap tmap_v, const FwdParams p) {
  constexpr int DH = 128, TB = TILE * DH * 2;
  extern __shared__ __align__(1024) uint8_t smem_raw[];  // swizzled tiles start on 1024 bytes
  const uint32_t smem_base = smem_u32(smem_raw);
  auto q_smem = [&](int g) { return smem_base + (PACKED ? 0 : g * TB); };
  auto kv_smem = [&](int pos) { return smem_base + (q_tiles(PACKED) + pos % STAGES) * TB; };
  const uint32_t bars = smem_base + (q_tiles(PACKED) + STAGES) * TB;
  const uint32_t q_full = bars;
  auto kv_full = [&](int pos) { return bars + 8u * (1 + pos % STAGES); };
  auto kv_empty = [&](int pos) { return bars + 8u * (1 + STAGES + pos % STAGES); };
  auto kv_phase = [&](int pos) { return static_cast<uint32_t>(pos / STAGES) & 1u; };
  auto scores = [&](int g) { return bars + 8u * (1 + 2 * STAGES + g); };
  auto probs = [&](int g, int half) { return bars + 8u * (3 + 2 * STAGES + 2 * g + half); };
  const uint32_t merge_bar = bars + 8u * (7 + 2 * STAGES);
  const uint32_t tmem_slot = bars + 8u * (8 + 2 * STAGES);
  static_assert(8 * (9 + 2 * STAGES) <= 256, "the barriers fit");
  volatile uint32_t *tmem_slot_ptr = reinterpret_cast<volatile uint32_t *>(smem_raw + (tmem_slot - smem_base));
  float2 *merge = reinterpret_cast<float2 *>(smem_raw + (bars + 256 - smem_base));

  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const Work w = work_of<PACKED>(p);
  const int n_max = max(w.n[0], w.n[1]);

  if (threadIdx.x == 0) {
    mbar_init(q_full, 1);
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(kv_full(s), 1);
      mbar_init(kv_empty(s), 1);
    }
    for (int g = 0; g < 2; ++g) {
      mbar_init(scores(g), 1);
      mbar_init(probs(g, 0), 4);
      mbar_init(probs(g, 1), 4);
    }
    mbar_init(merge_bar, 8);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    if (n_max > 0) {  // Q and the first keys, while the others set up
      if (PACKED) {
        mbar_expect_tx(q_full, p.n_q * p.group * DH * 2);
        load_tile<DH>(q_smem(0), &tmap_q, 0, w.head * p.group, w.b, q_full);
      } else {
        // only of the streams that have blocks: the output of one without (under the causal mask the first rows of more
        // queries than keys see none) takes the place of its Q at once, without a wait for it
        mbar_expect_tx(q_full, (w.n[0] > 0 ? TB : 0) + (w.n[1] > 0 ? TB : 0));
        for (int g = 0; g < 2; ++g)
          if (w.n[g] > 0) load_tile<DH>(q_smem(g), &tmap_q, (w.qt * 2 + g) * TILE, w.head, w.b, q_full);
      }
      mbar_expect_tx(kv_full(0), TB);
      load_tile<DH>(kv_smem(0), &tmap_k, w.kb0 * TILE, PACKED ? w.head : w.head / p.group, w.b, kv_full(0));
    }
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(tmem_slot), "r"(TMEM_COLS)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tcgen05_fence_before();
  __syncthreads();
  tcgen05_fence_after();
  const uint32_t tmem = *tmem_slot_ptr;
  if (p.splits > 1) asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
    if (warp == 0) {
      // ------------------------------------------------------------------ TMA producer
      if (lane == 0 && n_max > 0) {
        const int kv_head = PACKED ? w.head : w.head / p.group;
        int pos = 1;  // the first block of K is on its way already
        bool ok = true;
        auto load = [&](const CUtensorMap *map, int block) {
          if (!ok) return;
          if (pos >= STAGES && !mbar_wait_relaxed(kv_empty(pos), kv_phase(pos) ^ 1u, kPollSleepNs)) {
            report(p.status, kStatusTmaWaitTimeout);
            ok = false;
            return;
          }
          mbar_expect_tx(kv_full(pos), TB);
          load_tile<DH>(kv_smem(pos), map, (w.kb0 + block) * TILE, kv_head, w.b, kv_full(pos));
          ++pos;
        };
        // the order in which the products below use them
        if (PACKED) {
          const int nb = w.n[0] + w.n[1];
          if (nb > 1) load(&tmap_k, 1);
          for (int j = 0; j < nb; ++j) {
            load(&tmap_v, j);
            if (j + 2 < nb) load(&tmap_k, j + 2);
          }
        } else {
          for (int j = 0; j < n_max; ++j) {
            load(&tmap_v, j);
            if (j + 1 < n_max) load(&tmap_k, j + 1);
          }
        }
        // every tile has been used before the CTA may go
        for (int q = max(0, pos - STAGES); q < pos; ++q)
          if (!mbar_wait_relaxed(kv_empty(q), kv_phase(q), kPollSleepNs)) break;
      }
    } else if (warp == 1) {
      // ------------------------------------------------------------------ products
      // the whole warp walks the loop (it zeroes padded V rows together), lane 0 issues
      if (n_max > 0) {
        bool ok = __all_sync(0xffffffffu, mbar_wait(q_full, 0));
        const uint32_t leader = elect_one();
        int pos = 0;
        const int pad_block = w.keys < p.n_kv && w.keys % TILE ? w.keys / TILE - w.kb0 : -1;
        auto wait_tile = [&](int q) {
          if (ok) ok = __all_sync(0xffffffffu, mbar_wait(kv_full(q), kv_phase(q)));
        };
        auto issue_scores = [&](int g, int q) {
          if (ok) {
            tcgen05_fence_after();
            mma_scores<DH, TILE>(tmem + g * TILE, q_smem(g), kv_smem(q), p.idesc_s, leader);
            commit(scores(g), leader);
          }
        };
        auto release = [&](int q) {
          if (ok) commit(kv_empty(q), leader);
        };
        // O_g += P V of the stream's block jl; the last one signals the stream through its scores barrier
        auto issue_rows = [&](int g, int jl, int q) {
          // in two halves, the first while the stream still computes the second
          if (ok) ok = __all_sync(0xffffffffu, mbar_wait(probs(g, 0), jl & 1));
          if (ok) {
            tcgen05_fence_after();
            mma_rows<TILE, TILE, 0, 4>(tmem + O_COL + g * TILE, tmem + g * TILE, kv_smem(q), p.idesc_o, jl > 0, leader);
          }
          if (ok) ok = __all_sync(0xffffffffu, mbar_wait(probs(g, 1), jl & 1));
          if (ok) {
            tcgen05_fence_after();
            mma_rows<TILE, TILE, 4, 8>(tmem + O_COL + g * TILE, tmem + g * TILE, kv_smem(q), p.idesc_o, true, leader);
            if (jl + 1 == w.n[g]) commit(scores(g), leader);
          }
        };
        auto wait_v = [&](int q, int block) {
          wait_tile(q);
          if (block == pad_block) zero_rows<DH>(kv_smem(q), w.keys % TILE, lane);  // V behind the sequence's last key
        };
      if (PACKED) {
          const int nb = w.n[0] + w.n[1];
          for (int g = 0; g < 2 && g < nb; ++g) {
            wait_tile(pos);
            issue_scores(g, pos);
            release(pos++);
          }
          for (int j = 0; j < nb && ok; ++j) {
            const int g = j & 1;
            wait_v(pos, j);
            issue_rows(g, j >> 1, pos);
            release(pos++);
            if (j + 2 < nb) {
              wait_tile(pos);
              issue_scores(g, pos);
              release(pos++);
            }
          }
        } else {
          wait_tile(0);
          for (int g = 0; g < 2; ++g)
            if (w.n[g] > 0) issue_scores(g, 0);
          release(pos++);
          for (int j = 0; j < n_max && ok; ++j) {
            const int v = pos++, k = j + 1 < n_max ? pos++ : -1;
            wait_v(v, j);
            for (int g = 0; g < 2; ++g) {
              if (j < w.n[g]) issue_rows(g, j, v);
              if (g == 1) release(v);
              if (g == 0 && k >= 0) wait_tile(k);
              if (j + 1 < w.n[g]) issue_scores(g, k);
            }
            if (k >= 0) release(k);
          }
        }
        if (!ok && lane == 0) report(p.status, kStatusMmaWaitTimeout);
      }
    }
  } else {
    // ------------------------------------------------------------------ softmax and output
    asm volatile("setmaxnreg.inc.sync.aligned.u32 216;");
    const int g = (warp - 4) >> 2;
    const int lane_group = warp & 3;
    const int r = lane_group * 32 + lane;  // row of the tile = TMEM lane
    const int n = w.n[g];
    const uint32_t t_row = tmem + (static_cast<uint32_t>(lane_group * 32) << 16);
    const uint32_t s_addr = t_row + g * TILE;
    const uint32_t o_addr = t_row + O_COL + g * TILE;
    int head = w.head, i;  // the query this thread's row stands for
    if (PACKED) {
      head = w.head * p.group + r / p.n_q;
      i = r < p.n_q * p.group ? r % p.n_q : p.n_q;
    } else {
      i = w.qt * 2 * TILE + g * TILE + r;
    }
    const bool exists = i < p.n_q;
    const bool idle = PACKED && lane_group * 32 >= p.n_q * p.group;  // a warp without rows only keeps step
    // rows that do not exist compute on whatever is there and are not written
    const int limit = exists ? visible_keys(i, w.keys, p.n_q, p.n_kv, p.causal) : INT32_MAX;
    const float neg_inf = -INFINITY;
    float m = neg_inf, l = 0.0f;  // m: the reference maximum, in units of log2
    bool ok = true;
    for (int j = 0; j < n; ++j) {
      ok = mbar_wait(scores(g), j & 1);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      if (idle) {
        if (lane == 0) {
          mbar_arrive(probs(g, 0));
          mbar_arrive(probs(g, 1));
        }
        continue;
      }
      tcgen05_fence_after();
      uint32_t s[4][32];
#pragma unroll
      for (int c = 0; c < 4; ++c) tmem_ld_32x32(s_addr + 32 * c, s[c]);
      tmem_ld_wait();
      const int seen = limit - (w.kb0 + (PACKED ? 2 * j + g : j)) * TILE;  // of this block's keys
      mask_scores(s, seen);
      const float row_max = row_maximum(s) * p.scale_log2e;
      if (j == 0) m = row_max;
      else move_reference<DH>(m, l, row_max, o_addr);  // (P V of the block before is done: it was issued before these scores)
      l += exponentials<BF16>(s, p.scale_log2e, m, s_addr, [&](int half) {
        if (lane == 0) mbar_arrive(probs(g, half));
      });
    }
    if (ok && n > 0) {
      ok = mbar_wait(scores(g), n & 1);  // the last P V
      ok = __all_sync(0xffffffffu, ok);
    }
    const int64_t row = exists ? (static_cast<int64_t>(w.b) * p.q_heads + head) * p.n_q + i : 0;
    // factors of the two streams' accumulators (paired: only this stream's), first column and number of
    // columns this thread writes
    float a0 = 1.0f, a1 = 0.0f;
    int col0 = 0;
    constexpr int COLS = PACKED ? DH / 2 : DH;
    if (PACKED) {
      merge[g * TILE + r] = make_float2(m, l);
      __syncwarp();
      if (lane == 0) mbar_arrive(merge_bar);
      ok = ok && mbar_wait(merge_bar, 0);
      ok = __all_sync(0xffffffffu, ok);
      const float2 x = merge[r], y = merge[TILE + r];
      m = fmaxf(x.x, y.x);
      const float m_safe = m == neg_inf ? 0.0f : m;
      a0 = ex2(x.x - m_safe), a1 = ex2(y.x - m_safe);
      l = x.y * a0 + y.y * a1;
      col0 = g * COLS;
    }
    if (!ok) {
      if (lane == 0) report(p.status, kStatusEpiWaitTimeout);
    } else {
      tcgen05_fence_after();
      const bool has0 = PACKED ? w.n[0] > 0 : n > 0, has1 = PACKED && w.n[1] > 0;
      const bool some = sees_any(l);
      const float inv = p.splits > 1 ? 1.0f : (some ? 1.0f / l : 0.0f);
      a0 *= inv;
      a1 *= inv;
      if (exists && (!PACKED || g == 0)) {
        if (p.splits > 1) p.part_ml[w.split * p.rows + row] = make_float2(m, l);
        else p.lse[row] = row_lse(m, l);
      }
#pragma unroll 1
      for (int c = col0; c < col0 + COLS; c += 32) {
        uint32_t v0[32], v1[32];
        if (has0) tmem_ld_32x32((PACKED ? t_row + O_COL : o_addr) + c, v0);
        if (has1) tmem_ld_32x32(t_row + O_COL + TILE + c, v1);
        tmem_ld_wait();
        float x[32];
#pragma unroll
        for (int e = 0; e < 32; ++e) {
          x[e] = has0 && some ? __uint_as_float(v0[e]) * a0 : 0.0f;
          if (has1 && some) x[e] = fmaf(__uint_as_float(v1[e]), a1, x[e]);
        }
        if (p.splits == 1) stage_32<BF16>(q_smem(g) + r * (DH * 2), r, c / 8, x);
        else if (exists) store_part<DH>(p, x, w.split, row, c);
        __syncwarp();
      }
      if (p.splits == 1)
        write_rows<DH, COLS / 8>(q_smem(g), lane_group * 32, col0 / 8, lane, [&](int rr) -> uint16_t * {
          const int h = PACKED ? w.head * p.group + rr / p.n_q : w.head;
          const int q = PACKED ? rr % p.n_q : w.qt * 2 * TILE + g * TILE + rr;
          if (PACKED ? rr >= p.n_q * p.group : q >= p.n_q) return nullptr;
          return p.o + w.b * p.so.batch + h * p.so.head + q * p.so.row;
        });
    }
  }

  __syncwarp();
  tcgen05_fence_before();
  __syncthreads();
  if (warp == 1) {
    tcgen05_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(TMEM_COLS) : "memory");
  }
}

// ---- solo: d_head 64, one tile per CTA, two CTAs per SM
namespace solo {
constexpr int DH = 64, STAGES = 5, TB = TILE * DH * 2;
constexpr int THREADS = 256;
constexpr int TMEM_COLS = 256;  // S [0,128) P [128,192) O [192,256)
constexpr int P_COL = 128, O_COL = 192;
constexpr int SMEM = (1 + STAGES) * TB + 256;
constexpr int REGISTERS = 128;  // a thread at launch with two CTAs per SM, handed over as 56 + 200
static_assert(2 * (SMEM + 1024) <= 233472, "two CTAs per SM");
} // namespace solo

template <bool BF16, bool PACKED>
__global__ void __launch_bounds__(solo::THREADS, 2)
attention_solo_kernel(const __grid_constant__ CUtensorMap tmap_q, const __grid_constant__ CUtensorMap tmap_k,
                      const __grid_constant__ CUtensorMap tmap_v, const FwdParams p) {
  constexpr int DH = solo::DH, STAGES = solo::STAGES, TB = solo::TB;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  const uint32_t q_smem = smem_u32(smem_raw);
  auto kv_smem = [&](int pos) { return q_smem + (1 + pos % STAGES) * TB; };
  const uint32_t bars = q_smem + (1 + STAGES) * TB;
  const uint32_t q_full = bars;
  auto kv_full = [&](int pos) { return bars + 8u * (1 + pos % STAGES); };
  auto kv_empty = [&](int pos) { return bars + 8u * (1 + STAGES + pos % STAGES); };
  auto kv_phase = [&](int pos) { return static_cast<uint32_t>(pos / STAGES) & 1u; };
  const uint32_t scores = bars + 8u * (1 + 2 * STAGES), read = scores + 8, probs = scores + 16, rows_done = scores + 32;
  const uint32_t tmem_slot = scores + 40;
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;

  const int hb = blockIdx.x % p.heads_batch, rest = blockIdx.x / p.heads_batch;
  const int b = hb / p.heads, head = hb % p.heads, split = rest % p.splits;
  const int row0 = (p.tiles_q - 1 - rest / p.splits) * TILE;  // under the causal mask the long tiles come first
  // Packed rows that fit into one warp start in another quarter of the tile from CTA to CTA: the warp that has them
  // then sits on another scheduler than that of the SM's other CTA.
  const int rows = PACKED ? p.n_q * p.group : TILE, base = PACKED && rows <= 32 ? blockIdx.x % 4 * 32 : 0;
  const int keys = key_count(p.key_lens, b, p.n_kv);
  const int nb = (visible_keys((PACKED ? p.n_q : min(row0 + TILE, p.n_q)) - 1, keys, p.n_q, p.n_kv, p.causal) + TILE - 1) / TILE;
  const int kb0 = static_cast<int>(static_cast<int64_t>(nb) * split / p.splits);
  const int n = static_cast<int>(static_cast<int64_t>(nb) * (split + 1) / p.splits) - kb0;

  if (threadIdx.x == 0) {
    mbar_init(q_full, 1);
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(kv_full(s), 1);
      mbar_init(kv_empty(s), 1);
    }
    mbar_init(scores, 1);
    mbar_init(read, 4);
    mbar_init(probs, 4);
    mbar_init(probs + 8, 4);
    mbar_init(rows_done, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    if (n > 0) {  // Q and the first keys, while the others set up
      mbar_expect_tx(q_full, rows * DH * 2);
      load_tile<DH>(q_smem + base * (DH * 2), &tmap_q, row0, PACKED ? head * p.group : head, b, q_full);
      mbar_expect_tx(kv_full(0), TB);
      load_tile<DH>(kv_smem(0), &tmap_k, kb0 * TILE, PACKED ? head : head / p.group, b, kv_full(0));
    }
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(tmem_slot), "r"(solo::TMEM_COLS)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tcgen05_fence_before();
  __syncthreads();
  tcgen05_fence_after();
  const uint32_t tmem = *reinterpret_cast<volatile uint32_t *>(smem_raw + (tmem_slot - q_smem));
  if (p.splits > 1) asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
    if (warp == 0) {
      if (lane == 0 && n > 0) {
        const int kv_head = PACKED ? head : head / p.group;
        int pos = 1;  // the first block of K is on its way already
        bool ok = true;
        auto load = [&](const CUtensorMap *map, int block) {
          if (!ok) return;
          if (pos >= STAGES && !mbar_wait_relaxed(kv_empty(pos), kv_phase(pos) ^ 1u, kPollSleepNs)) {
            report(p.status, kStatusTmaWaitTimeout);
            ok = false;
            return;
          }
          mbar_expect_tx(kv_full(pos), TB);
          load_tile<DH>(kv_smem(pos), map, (kb0 + block) * TILE, kv_head, b, kv_full(pos));
          ++pos;
        };
        for (int j = 0; j < n; ++j) {
          if (j + 1 < n) load(&tmap_k, j + 1);
          load(&tmap_v, j);
        }
        for (int q = max(0, pos - STAGES); q < pos; ++q)  // every tile has been used
          if (!mbar_wait_relaxed(kv_empty(q), kv_phase(q), kPollSleepNs)) break;
      }
    } else if (warp == 1 && n > 0) {
      const uint32_t leader = elect_one();
      bool ok = __all_sync(0xffffffffu, mbar_wait(q_full, 0));
      int pos = 0;
      const int pad_block = keys < p.n_kv && keys % TILE ? keys / TILE - kb0 : -1;
      auto wait = [&](uint32_t bar, uint32_t parity) {
        if (ok) ok = __all_sync(0xffffffffu, mbar_wait(bar, parity));
      };
      auto next_scores = [&]() {
        wait(kv_full(pos), kv_phase(pos));
        if (ok) {
          tcgen05_fence_after();
          mma_scores<DH, TILE>(tmem, q_smem, kv_smem(pos), p.idesc_s, leader);
          commit(scores, leader);
          commit(kv_empty(pos), leader);
        }
        ++pos;
      };
      next_scores();
      for (int j = 0; j < n && ok; ++j) {
        if (j + 1 < n) {
          wait(read, j & 1);
          next_scores();
        }
        wait(kv_full(pos), kv_phase(pos));
        if (j == pad_block) zero_rows<DH>(kv_smem(pos), keys % TILE, lane);  // V behind the sequence's last key
        for (int half = 0; half < 2; ++half) {
          wait(probs + 8 * half, j & 1);
          if (!ok) break;
          tcgen05_fence_after();
          const uint32_t o = tmem + solo::O_COL, q = tmem + solo::P_COL;
          if (half == 0) mma_rows<TILE, TILE, 0, 4>(o, q, kv_smem(pos), p.idesc_o, j > 0, leader);
          else mma_rows<TILE, TILE, 4, 8>(o, q, kv_smem(pos), p.idesc_o, true, leader);
        }
        if (ok) {
          commit(rows_done, leader);
          commit(kv_empty(pos), leader);
        }
        ++pos;
      }
      if (!ok && lane == 0) report(p.status, kStatusMmaWaitTimeout);
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 200;");
    const int lane_group = warp & 3, r = lane_group * 32 + lane;
    // head and query of a row of the tile; rows that do not exist compute on whatever is there and are not written
    auto head_of = [&](int row) { return PACKED ? head * p.group + (row - base) / p.n_q : head; };
    auto query_of = [&](int row) {
      return PACKED ? (row >= base && row - base < rows ? (row - base) % p.n_q : p.n_q) : row0 + row;
    };
    const int i = query_of(r);
    const bool exists = i < p.n_q;
    const bool idle = PACKED && !__any_sync(0xffffffffu, exists);  // a warp without rows only keeps step
    const uint32_t t_row = tmem + (static_cast<uint32_t>(lane_group * 32) << 16);
    const int limit = exists ? visible_keys(i, keys, p.n_q, p.n_kv, p.causal) : INT32_MAX;
    float m = -INFINITY, l = 0.0f;
    bool ok = true;
    auto wait = [&](uint32_t bar, uint32_t parity) { return __all_sync(0xffffffffu, mbar_wait(bar, parity)); };
    for (int j = 0; j < n; ++j) {
      if (!(ok = wait(scores, j & 1))) break;
      if (idle) {
        if (lane == 0) mbar_arrive(read);
        if (j > 0 && !(ok = wait(rows_done, (j - 1) & 1))) break;
        if (lane == 0) {
          mbar_arrive(probs);
          mbar_arrive(probs + 8);
        }
        continue;
      }
      tcgen05_fence_after();
      uint32_t s[4][32];
#pragma unroll
      for (int c = 0; c < 4; ++c) tmem_ld_32x32(t_row + 32 * c, s[c]);
      tmem_ld_wait();
      tcgen05_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(read);
      mask_scores(s, limit - (kb0 + j) * TILE);
      const float row_max = row_maximum(s) * p.scale_log2e;
      if (j == 0) {
        m = row_max;
      } else {
        if (!(ok = wait(rows_done, (j - 1) & 1))) break;  // P and O are free
        tcgen05_fence_after();
        move_reference<DH>(m, l, row_max, t_row + solo::O_COL);
      }
      l += exponentials<BF16>(s, p.scale_log2e, m, t_row + solo::P_COL, [&](int half) {
        if (lane == 0) mbar_arrive(probs + 8 * half);
      });
    }
    if (ok && n > 0) ok = wait(rows_done, (n - 1) & 1);
    if (!ok) {
      if (lane == 0) report(p.status, kStatusEpiWaitTimeout);
    } else {
      tcgen05_fence_after();
      const int64_t row = exists ? (static_cast<int64_t>(b) * p.q_heads + head_of(r)) * p.n_q + i : 0;
      const bool some = sees_any(l);
      const float f = p.splits > 1 ? 1.0f : (some ? 1.0f / l : 0.0f);
      if (exists) {
        if (p.splits > 1) p.part_ml[split * p.rows + row] = make_float2(m, l);
        else p.lse[row] = row_lse(m, l);
      }
#pragma unroll 1
      for (int c = 0; c < DH; c += 32) {
        uint32_t v[32];
        if (n > 0) tmem_ld_32x32(t_row + solo::O_COL + c, v);
        tmem_ld_wait();
        float x[32];
#pragma unroll
        for (int e = 0; e < 32; ++e) x[e] = n > 0 && some ? __uint_as_float(v[e]) * f : 0.0f;
        if (p.splits == 1) stage_32<BF16>(q_smem + r * (DH * 2), r, c / 8, x);
        else if (exists) store_part<DH>(p, x, split, row, c);
        __syncwarp();
      }
      if (p.splits == 1)
        write_rows<DH, DH / 8>(q_smem, lane_group * 32, 0, lane, [&](int rr) -> uint16_t * {
          const int q = query_of(rr);
          return q < p.n_q ? p.o + b * p.so.batch + head_of(rr) * p.so.head + q * p.so.row : nullptr;
        });
    }
  }

  __syncwarp();
  tcgen05_fence_before();
  __syncthreads();
  if (warp == 1) {
    tcgen05_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(solo::TMEM_COLS) : "memory");
  }
}

// O and LSE of a row from its splits (64 at most).  One warp per row: a lane has the maximum and sum of two splits, then
// the warp adds up the rows in order, eight loads in flight.
template <bool BF16, int DH> __global__ void __launch_bounds__(128) attention_join_kernel(const FwdParams p) {
  // started while the last tiles still run
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int64_t row = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  if (row >= p.rows) return;
  float2 ml[2];
#pragma unroll
  for (int k = 0; k < 2; ++k)
    ml[k] = lane + 32 * k < p.splits ? p.part_ml[(lane + 32 * k) * p.rows + row] : make_float2(-INFINITY, 0.0f);
  float m = fmaxf(ml[0].x, ml[1].x);
#pragma unroll
  for (int s = 16; s; s /= 2) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, s));
  const float m_safe = m == -INFINITY ? 0.0f : m;
  const float a0 = ex2(ml[0].x - m_safe), a1 = ex2(ml[1].x - m_safe);
  float l = fmaf(ml[0].y, a0, ml[1].y * a1);
#pragma unroll
  for (int s = 16; s; s /= 2) l += __shfl_xor_sync(0xffffffffu, l, s);
  constexpr int V = DH / 32;
  using Vec = typename std::conditional<V == 4, float4, float2>::type;
  float x[V] = {};
  const float *from = p.part_o + row * DH + lane * V;
  for (int s0 = 0; s0 < p.splits; s0 += 8) {
    Vec v[8];
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (s0 + k < p.splits) v[k] = *reinterpret_cast<const Vec *>(from + (s0 + k) * p.rows * DH);
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (s0 + k < p.splits) {
        const int s = s0 + k;
        const float a = __shfl_sync(0xffffffffu, s < 32 ? a0 : a1, s & 31);
        const float *e = reinterpret_cast<const float *>(&v[k]);
#pragma unroll
        for (int c = 0; c < V; ++c) x[c] = fmaf(e[c], a, x[c]);
      }
  }
  const float inv = sees_any(l) ? 1.0f / l : 0.0f;
  const int i = static_cast<int>(row % p.n_q);
  const int64_t bh = row / p.n_q;
  uint16_t *to = p.o + (bh / p.q_heads) * p.so.batch + (bh % p.q_heads) * p.so.head + i * p.so.row + lane * V;
  uint32_t w[V / 2];
#pragma unroll
  for (int e = 0; e < V; e += 2) w[e / 2] = pack2<BF16>(x[e] * inv, x[e + 1] * inv);
  if (V == 4) *reinterpret_cast<uint2 *>(to) = make_uint2(w[0], w[V / 2 - 1]);
  else *reinterpret_cast<uint32_t *>(to) = w[0];
  if (lane == 0) p.lse[row] = row_lse(m, l);
}

bool is_packed(const AttentionProblem &p) { return p.n_q * (p.q_heads / p.kv_heads) <= TILE; }
int64_t tiles_per_head(const AttentionProblem &p) {
  if (is_packed(p)) return 1;
  const int64_t rows = p.d_head == 64 ? TILE : 2 * TILE;
  return (p.n_q + rows - 1) / rows;
}
int64_t tile_count(const AttentionProblem &p) {
  return p.batch * (is_packed(p) ? p.kv_heads : p.q_heads) * tiles_per_head(p);
}
// Shares of a tile's key blocks, at least four blocks each, none of fewer than twelve: the number with the shortest sum
// of rounds, where a CTA's start and end cost about as much as seven blocks (four where two CTAs share an SM and one
// works on) and the joining as three.  8 query heads on one key head, one query: 8192 keys 57 us with one share, 13
// with 16; 64 tiles of 1000 keys: 12.6 us with one, 14.6 with two.  One query of 8000 keys, packed: 128 tiles (one
// round) 84 us with one share, 90 with 2; 160 tiles (two rounds) 139 and 119 with 3; 80 tiles of 4000 keys: 35 with
// one, 39 with 3.  Tiles that are not packed are split only to fill one round: a share leaves 128 KB in the workspace.
int split_count(const AttentionProblem &p) {
  const int64_t blocks = (p.n_kv + TILE - 1) / TILE, tiles = tile_count(p);
  const int64_t slots = (p.d_head == 64 ? 2 : 1) * tc_host::sm_count(), ends = p.d_head == 64 ? 4 : 7;
  if (blocks < 12 || (tiles >= slots && !is_packed(p))) return 1;
  int64_t best = 1, best_cost = INT64_MAX;
  for (int64_t s = 1; s <= 64 && s <= blocks / 4; ++s) {
    const int64_t rounds = (tiles * s + slots - 1) / slots;
    const int64_t cost = rounds * ((blocks + s - 1) / s + ends) + (s > 1 ? 3 : 0);
    if (cost < best_cost && (is_packed(p) || s == 1 || rounds == 1)) best = s, best_cost = cost;
  }
  return static_cast<int>(best);
}

bool same(const Strides3 &a, const Strides3 &b) { return a.batch == b.batch && a.head == b.head && a.row == b.row; }
bool aligned(const void *x) { return (reinterpret_cast<uintptr_t>(x) & 15) == 0; }

template <auto kernel>
cudaError_t launch_tiles(const CUtensorMap &tq, const CUtensorMap &tk, const CUtensorMap &tv, const FwdParams &f,
                         unsigned grid, int threads, int smem, int registers, cudaStream_t stream) {
  const cudaError_t e = allow_smem<kernel>(smem, registers);
  if (e != cudaSuccess) return e;
  kernel<<<grid, threads, smem, stream>>>(tq, tk, tv, f);
  return cudaGetLastError();
}
template <bool BF16, int DH, bool PACKED>
cudaError_t launch_typed(const CUtensorMap &tq, const CUtensorMap &tk, const CUtensorMap &tv, const FwdParams &f,
                         unsigned grid, cudaStream_t stream) {
  cudaError_t e;
  if constexpr (DH == 64)
    e = launch_tiles<attention_solo_kernel<BF16, PACKED>>(tq, tk, tv, f, grid, solo::THREADS, solo::SMEM, solo::REGISTERS, stream);
  else
    e = launch_tiles<attention_kernel<BF16, PACKED>>(tq, tk, tv, f, grid, THREADS, smem_bytes(PACKED), REGISTERS, stream);
  if (e != cudaSuccess || f.splits == 1) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>((f.rows + 3) / 4));
  cfg.blockDim = dim3(128);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, attention_join_kernel<BF16, DH>, f);
}
template <bool BF16, int DH>
cudaError_t launch_rows(const CUtensorMap &tq, const CUtensorMap &tk, const CUtensorMap &tv, const FwdParams &f,
                        unsigned grid, bool packed, cudaStream_t stream) {
  return packed ? launch_typed<BF16, DH, true>(tq, tk, tv, f, grid, stream)
                : launch_typed<BF16, DH, false>(tq, tk, tv, f, grid, stream);
}

} // namespace

const char *attention_check(const AttentionProblem &p, bool backward, bool pointers) {
  if (p.dtype != kF16 && p.dtype != kBF16) return "the element type is f16 or bf16";
  if (p.batch < 1 || p.q_heads < 1 || p.kv_heads < 1 || p.n_q < 1 || p.n_kv < 1)
    return "batch, heads and lengths are at least 1";
  if (p.q_heads % p.kv_heads) return "q_heads must be a multiple of kv_heads";
  if (p.d_head != 64 && p.d_head != 128) return "d_head is 64 or 128";
  if (!(p.scale > 0.0f) || p.scale > 1.0e30f) return "sm_scale must be positive and at most 1e30";
  if (p.batch > 65535 || p.q_heads > 65535 || p.n_q > (1 << 30) || p.n_kv > (1 << 30) ||
      p.batch * p.q_heads * ((p.n_q + TILE - 1) / TILE) > INT32_MAX / 64 ||
      p.batch * p.kv_heads * ((p.n_kv + TILE - 1) / TILE) > INT32_MAX / 64)
    return "too many sequences, heads or rows";
  const Strides3 *s[8] = {&p.sq, &p.sk, &p.sv, &p.so, &p.sdo, &p.sdq, &p.sdk, &p.sdv};
  const bool of_keys[8] = {false, true, true, false, false, false, true, true};
  const bool written[8] = {false, false, false, !backward, false, true, true, true};
  for (int i = 0; i < (backward ? 8 : 4); ++i) {
    const int64_t extent[3] = {p.batch, of_keys[i] ? p.kv_heads : p.q_heads, of_keys[i] ? p.n_kv : p.n_q};
    const int64_t step[3] = {s[i]->batch, s[i]->head, s[i]->row};
    for (int j = 0; j < 3; ++j) {
      if (step[j] < 0 || step[j] % 8 || step[j] >= (1ll << 38)) return "strides are multiples of 8 elements, below 2^38";
      if (extent[j] > 1 && step[j] == 0) return "strides of extents above 1 are not zero";
    }
    if (written[i] && rows_overlap(p.d_head, {{step[0], extent[0]}, {step[1], extent[1]}, {step[2], extent[2]}}))
      return "the rows of an output overlap";
  }
  if (!pointers) return nullptr;
  if (!aligned(p.q) || !aligned(p.k) || !aligned(p.v) || !aligned(p.o) ||
      (backward && (!aligned(p.dout) || !aligned(p.dq) || !aligned(p.dk) || !aligned(p.dv))))
    return "arrays must be 16-byte aligned";
  if (reinterpret_cast<uintptr_t>(p.lse) % 4 || reinterpret_cast<uintptr_t>(p.key_lens) % 4)
    return "LSE and key_lens must start on a multiple of 4 bytes";
  if (attention_workspace_bytes(p, backward) && !aligned(p.workspace)) return "the workspace must be 16-byte aligned";
  // Arrays that start at one address share their first row at least.  A tile's O goes out after its Q has been read;
  // everything else is read by tiles that may run later.
  if (!backward && (p.o == p.k || p.o == p.v || (p.o == p.q && !same(p.so, p.sq)))) return "O may not be K or V, nor Q with other strides";
  if (backward)
    for (const void *d : {p.dq, p.dk, p.dv})
      if (d == p.q || d == p.k || d == p.v || d == p.dout || (d == p.dq) + (d == p.dk) + (d == p.dv) > 1)
        return "dQ, dK and dV may not be Q, K, V, dO or one another";
  return nullptr;
}

size_t attention_workspace_bytes(const AttentionProblem &p, bool backward) {
  const size_t rows = static_cast<size_t>(p.batch) * p.q_heads * p.n_q;
  auto up = [](size_t n) { return (n + 255) / 256 * 256; };
  if (backward) return up(rows * sizeof(float));
  const size_t splits = split_count(p);
  return splits == 1 ? 0 : up(splits * rows * sizeof(float2)) + up(splits * rows * p.d_head * sizeof(float));
}

cudaError_t launch_attention(const AttentionProblem &p, unsigned *status, cudaStream_t stream, int *launched) {
  const bool packed = is_packed(p), bf16 = p.dtype == kBF16;
  const int64_t group = p.q_heads / p.kv_heads;
  CUtensorMap tq, tk, tv;
  if (!make_map_4d(&tq, p.q, p.dtype, p.d_head, p.n_q, p.q_heads, p.batch, p.sq,
                   packed ? static_cast<int>(p.n_q) : TILE, packed ? static_cast<int>(group) : 1) ||
      !make_map_4d(&tk, p.k, p.dtype, p.d_head, p.n_kv, p.kv_heads, p.batch, p.sk, TILE, 1) ||
      !make_map_4d(&tv, p.v, p.dtype, p.d_head, p.n_kv, p.kv_heads, p.batch, p.sv, TILE, 1))
    return cudaErrorNotSupported;
  FwdParams f{};
  f.o = static_cast<uint16_t *>(p.o);
  f.lse = p.lse;
  f.key_lens = p.key_lens;
  f.status = status;
  f.so = p.so;
  f.q_heads = static_cast<int>(p.q_heads);
  f.group = static_cast<int>(group);
  f.n_q = static_cast<int>(p.n_q);
  f.n_kv = static_cast<int>(p.n_kv);
  f.causal = p.causal ? 1 : 0;
  f.heads = static_cast<int>(packed ? p.kv_heads : p.q_heads);
  f.heads_batch = f.heads * static_cast<int>(p.batch);
  f.tiles_q = static_cast<int>(tiles_per_head(p));
  f.splits = split_count(p);
  f.rows = p.batch * p.q_heads * p.n_q;
  f.scale_log2e = p.scale * 1.4426950408889634f;
  f.idesc_s = instruction_desc(bf16, false, TILE);
  f.idesc_o = instruction_desc(bf16, true, static_cast<int>(p.d_head));
  if (f.splits > 1) {
    f.part_ml = static_cast<float2 *>(p.workspace);
    const size_t ml = (static_cast<size_t>(f.splits) * f.rows * sizeof(float2) + 255) / 256 * 256;
    f.part_o = reinterpret_cast<float *>(static_cast<char *>(p.workspace) + ml);
  }
  const unsigned grid = static_cast<unsigned>(tile_count(p) * f.splits);
  *launched = f.splits > 1 ? 2 : 1;
  if (p.d_head == 64)
    return bf16 ? launch_rows<true, 64>(tq, tk, tv, f, grid, packed, stream)
                : launch_rows<false, 64>(tq, tk, tv, f, grid, packed, stream);
  return bf16 ? launch_rows<true, 128>(tq, tk, tv, f, grid, packed, stream)
              : launch_rows<false, 128>(tq, tk, tv, f, grid, packed, stream);
}

} // namespace imex
