// Attention backward (IMEX_OP_ATTENTION_BWD), plain kernels: one block per query row for dQ (which also
// leaves delta = rowsum(dO O) in the workspace), one block per key for dK and dV.  The probabilities are
// recomputed from LSE.
#include "attention_common.cuh"

namespace imex {
namespace {

using namespace attn;

struct BwdArgs {
  const uint16_t *q, *k, *v, *o, *dout;
  const float *lse;
  float *delta;
  uint16_t *dq, *dk, *dv;
  const int32_t *key_lens;
  Strides3 sq, sk, sv, so, sdo, sdq, sdk, sdv;
  int q_heads, group, n_q, n_kv, d, causal;
  float scale;
};

template <bool BF16> __global__ void __launch_bounds__(128) attention_dq_rows_kernel(const BwdArgs a) {
  __shared__ float qs[128], gs[128], ds[128], red[4];
  const int i = blockIdx.x, h = blockIdx.y, b = blockIdx.z, t = threadIdx.x;
  const uint16_t *k = a.k + b * a.sk.batch + (h / a.group) * a.sk.head;
  const uint16_t *v = a.v + b * a.sv.batch + (h / a.group) * a.sv.head;
  float part = 0.0f;
  if (t < a.d) {
    qs[t] = to_f32<BF16>(a.q[b * a.sq.batch + h * a.sq.head + i * a.sq.row + t]);
    gs[t] = to_f32<BF16>(a.dout[b * a.sdo.batch + h * a.sdo.head + i * a.sdo.row + t]);
    part = gs[t] * to_f32<BF16>(a.o[b * a.so.batch + h * a.so.head + i * a.so.row + t]);
  }
  for (int o = 16; o; o >>= 1) part += __shfl_xor_sync(0xffffffffu, part, o);
  if ((t & 31) == 0) red[t >> 5] = part;
  __syncthreads();
  const float delta = red[0] + red[1] + red[2] + red[3];
  const int64_t row = (static_cast<int64_t>(b) * a.q_heads + h) * a.n_q + i;
  if (t == 0) a.delta[row] = delta;
  const float lse = a.lse[row];
  const int limit = visible_keys(i, key_count(a.key_lens, b, a.n_kv), a.n_q, a.n_kv, a.causal);
  float acc = 0.0f;
  for (int j0 = 0; j0 < limit; j0 += 128) {
    float x = 0.0f;
    if (j0 + t < limit) {
      const uint16_t *kr = k + (j0 + t) * a.sk.row, *vr = v + (j0 + t) * a.sv.row;
      float s = 0.0f, dp = 0.0f;
      for (int c = 0; c < a.d; ++c) {
        s = fmaf(qs[c], to_f32<BF16>(kr[c]), s);
        dp = fmaf(gs[c], to_f32<BF16>(vr[c]), dp);
      }
      x = expf(s * a.scale - lse) * (dp - delta);
    }
    ds[t] = x;
    __syncthreads();
    const int n = min(128, limit - j0);
    if (t < a.d)
      for (int j = 0; j < n; ++j) acc = fmaf(ds[j], to_f32<BF16>(k[(j0 + j) * a.sk.row + t]), acc);
    __syncthreads();
  }
  if (t < a.d) a.dq[b * a.sdq.batch + h * a.sdq.head + i * a.sdq.row + t] = from_f32<BF16>(acc * a.scale);
}

template <bool BF16> __global__ void __launch_bounds__(128) attention_dkv_rows_kernel(const BwdArgs a) {
  __shared__ float ks[128], vs[128], ps[128], ds[128];
  const int j = blockIdx.x, hk = blockIdx.y, b = blockIdx.z, t = threadIdx.x;
  const int keys = key_count(a.key_lens, b, a.n_kv);
  float dk = 0.0f, dv = 0.0f;
  if (j < keys) {
    if (t < a.d) {
      ks[t] = to_f32<BF16>(a.k[b * a.sk.batch + hk * a.sk.head + j * a.sk.row + t]);
      vs[t] = to_f32<BF16>(a.v[b * a.sv.batch + hk * a.sv.head + j * a.sv.row + t]);
    }
    __syncthreads();
    for (int h = hk * a.group; h < (hk + 1) * a.group; ++h) {
      const uint16_t *q = a.q + b * a.sq.batch + h * a.sq.head;
      const uint16_t *g = a.dout + b * a.sdo.batch + h * a.sdo.head;
      for (int i0 = 0; i0 < a.n_q; i0 += 128) {
        float p = 0.0f, x = 0.0f;
        const int i = i0 + t;
        if (i < a.n_q && j < visible_keys(i, keys, a.n_q, a.n_kv, a.causal)) {
          float s = 0.0f, dp = 0.0f;
          for (int c = 0; c < a.d; ++c) {
            s = fmaf(to_f32<BF16>(q[i * a.sq.row + c]), ks[c], s);
            dp = fmaf(to_f32<BF16>(g[i * a.sdo.row + c]), vs[c], dp);
          }
          const int64_t row = (static_cast<int64_t>(b) * a.q_heads + h) * a.n_q + i;
          p = expf(s * a.scale - a.lse[row]);
          x = p * (dp - a.delta[row]);
        }
        ps[t] = p;
        ds[t] = x;
        __syncthreads();
        const int n = min(128, a.n_q - i0);
        if (t < a.d)
          for (int r = 0; r < n; ++r) {
            dv = fmaf(ps[r], to_f32<BF16>(g[(i0 + r) * a.sdo.row + t]), dv);
            dk = fmaf(ds[r], to_f32<BF16>(q[(i0 + r) * a.sq.row + t]), dk);
          }
        __syncthreads();
      }
    }
  }
  if (t < a.d) {
    a.dk[b * a.sdk.batch + hk * a.sdk.head + j * a.sdk.row + t] = from_f32<BF16>(dk * a.scale);
    a.dv[b * a.sdv.batch + hk * a.sdv.head + j * a.sdv.row + t] = from_f32<BF16>(dv);
  }
}

} // namespace

cudaError_t launch_attention_bwd(const AttentionProblem &p, unsigned *, cudaStream_t stream, int *launched) {
  auto in = [](const void *x) { return static_cast<const uint16_t *>(x); };
  auto out = [](void *x) { return static_cast<uint16_t *>(x); };
  BwdArgs a{in(p.q), in(p.k), in(p.v), in(p.o), in(p.dout), p.lse, static_cast<float *>(p.workspace),
            out(p.dq), out(p.dk), out(p.dv), p.key_lens, p.sq, p.sk, p.sv, p.so, p.sdo, p.sdq, p.sdk, p.sdv,
            static_cast<int>(p.q_heads), static_cast<int>(p.q_heads / p.kv_heads), static_cast<int>(p.n_q),
            static_cast<int>(p.n_kv), static_cast<int>(p.d_head), p.causal ? 1 : 0, p.scale};
  const dim3 gq(static_cast<unsigned>(p.n_q), static_cast<unsigned>(p.q_heads), static_cast<unsigned>(p.batch));
  const dim3 gk(static_cast<unsigned>(p.n_kv), static_cast<unsigned>(p.kv_heads), static_cast<unsigned>(p.batch));
  if (p.dtype == kBF16) {
    attention_dq_rows_kernel<true><<<gq, 128, 0, stream>>>(a);
    attention_dkv_rows_kernel<true><<<gk, 128, 0, stream>>>(a);
  } else {
    attention_dq_rows_kernel<false><<<gq, 128, 0, stream>>>(a);
    attention_dkv_rows_kernel<false><<<gk, 128, 0, stream>>>(a);
  }
  *launched = 2;
  return cudaGetLastError();
}

} // namespace imex
