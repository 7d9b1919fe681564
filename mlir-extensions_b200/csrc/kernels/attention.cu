// Attention forward with row statistics (IMEX_OP_ATTENTION): checks and a plain kernel, one block
// per query row, one pass over its visible keys with the running maximum and sum.
#include "attention_common.cuh"

namespace imex {
namespace {

using namespace attn;

struct FwdArgs {
  const uint16_t *q, *k, *v;
  uint16_t *o;
  float *lse;
  const int32_t *key_lens;
  Strides3 sq, sk, sv, so;
  int q_heads, group, n_q, n_kv, d, causal;
  float scale;
};

template <bool BF16> __global__ void __launch_bounds__(128) attention_rows_kernel(const FwdArgs a) {
  __shared__ float qs[128], ps[128], red[4];
  const int i = blockIdx.x, h = blockIdx.y, b = blockIdx.z, t = threadIdx.x;
  const uint16_t *q = a.q + b * a.sq.batch + h * a.sq.head + i * a.sq.row;
  const uint16_t *k = a.k + b * a.sk.batch + (h / a.group) * a.sk.head;
  const uint16_t *v = a.v + b * a.sv.batch + (h / a.group) * a.sv.head;
  if (t < a.d) qs[t] = to_f32<BF16>(q[t]);
  __syncthreads();
  const int limit = visible_keys(i, key_count(a.key_lens, b, a.n_kv), a.n_q, a.n_kv, a.causal);
  float m = -INFINITY, l = 0.0f, acc = 0.0f;
  for (int j0 = 0; j0 < limit; j0 += 128) {
    float s = -INFINITY;
    if (j0 + t < limit) {
      s = 0.0f;
      const uint16_t *kr = k + (j0 + t) * a.sk.row;
      for (int c = 0; c < a.d; ++c) s = fmaf(qs[c], to_f32<BF16>(kr[c]), s);
      s *= a.scale;
    }
    float x = s;
    for (int o = 16; o; o >>= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, o));
    if ((t & 31) == 0) red[t >> 5] = x;
    __syncthreads();
    const float m1 = fmaxf(m, fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3])));
    const float p = expf(s - m1), r = expf(m - m1);
    ps[t] = p;
    __syncthreads();
    acc *= r;
    l *= r;
    m = m1;
    const int n = min(128, limit - j0);
    for (int j = 0; j < n; ++j) {
      l += ps[j];
      if (t < a.d) acc = fmaf(ps[j], to_f32<BF16>(v[(j0 + j) * a.sv.row + t]), acc);
    }
    __syncthreads();
  }
  if (t < a.d)
    a.o[b * a.so.batch + h * a.so.head + i * a.so.row + t] = from_f32<BF16>(limit > 0 ? acc / l : 0.0f);
  if (t == 0)
    a.lse[(static_cast<int64_t>(b) * a.q_heads + h) * a.n_q + i] = limit > 0 ? m + logf(l) : -INFINITY;
}

bool aligned(const void *x) { return (reinterpret_cast<uintptr_t>(x) & 15) == 0; }

} // namespace

const char *attention_check(const AttentionProblem &p, bool backward, bool pointers) {
  if (p.dtype != kF16 && p.dtype != kBF16) return "the element type is f16 or bf16";
  if (p.batch < 1 || p.q_heads < 1 || p.kv_heads < 1 || p.n_q < 1 || p.n_kv < 1)
    return "batch, heads and lengths are at least 1";
  if (p.q_heads % p.kv_heads) return "q_heads must be a multiple of kv_heads";
  if (p.d_head != 64 && p.d_head != 128) return "d_head is 64 or 128";
  if (!(p.scale > 0.0f) || p.scale > 3.0e38f) return "sm_scale must be positive and finite";
  if (p.batch > 65535 || p.q_heads > 65535 || p.n_q > (1 << 30) || p.n_kv > (1 << 30))
    return "at most 65535 sequences and heads, 2^30 rows";
  const Strides3 *s[8] = {&p.sq, &p.sk, &p.sv, &p.so, &p.sdo, &p.sdq, &p.sdk, &p.sdv};
  for (int i = 0; i < (backward ? 8 : 4); ++i)
    if (s[i]->batch < 0 || s[i]->head < 0 || s[i]->row < 0 || s[i]->batch % 8 || s[i]->head % 8 || s[i]->row % 8 ||
        s[i]->batch >= (1ll << 38) || s[i]->head >= (1ll << 38) || s[i]->row >= (1ll << 38))
      return "strides are multiples of 8 elements, below 2^38";
  if (!pointers) return nullptr;
  if (!aligned(p.q) || !aligned(p.k) || !aligned(p.v) || !aligned(p.o) ||
      (backward && (!aligned(p.dout) || !aligned(p.dq) || !aligned(p.dk) || !aligned(p.dv))))
    return "arrays must be 16-byte aligned";
  return nullptr;
}

size_t attention_workspace_bytes(const AttentionProblem &p, bool backward) {
  if (!backward) return 0;
  return (static_cast<size_t>(p.batch) * p.q_heads * p.n_q * sizeof(float) + 255) / 256 * 256;
}

cudaError_t launch_attention(const AttentionProblem &p, unsigned *, cudaStream_t stream, int *launched) {
  FwdArgs a{static_cast<const uint16_t *>(p.q), static_cast<const uint16_t *>(p.k), static_cast<const uint16_t *>(p.v),
            static_cast<uint16_t *>(p.o), p.lse, p.key_lens, p.sq, p.sk, p.sv, p.so, static_cast<int>(p.q_heads),
            static_cast<int>(p.q_heads / p.kv_heads), static_cast<int>(p.n_q), static_cast<int>(p.n_kv),
            static_cast<int>(p.d_head), p.causal ? 1 : 0, p.scale};
  const dim3 grid(static_cast<unsigned>(p.n_q), static_cast<unsigned>(p.q_heads), static_cast<unsigned>(p.batch));
  if (p.dtype == kBF16) attention_rows_kernel<true><<<grid, 128, 0, stream>>>(a);
  else attention_rows_kernel<false><<<grid, 128, 0, stream>>>(a);
  *launched = 1;
  return cudaGetLastError();
}

} // namespace imex
