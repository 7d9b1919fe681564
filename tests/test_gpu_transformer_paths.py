"""The ways through the attention and gated feed-forward kernels that only some shapes take, each against its formula in
64 bits; the tolerances are those of test_gpu_transformer_ops.py."""
import numpy as np
import pytest
import torch

from __graft_entry__ import load_package
from test_gpu_transformer_ops import Attention, Output, _bits, _dt

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def pkg():
    return load_package()


@pytest.fixture()
def sess(pkg):
    s = pkg.Session(device=0)
    yield s
    s.close()


# ------------------------------------------------------------------------------------------- attention
@pytest.mark.parametrize("n_q,n_kv", [(300, 150), (600, 400), (256, 128), (1000, 800)])
@pytest.mark.parametrize("kind", ["bf16", "f16"])
def test_rows_before_the_first_key_of_a_tile_pair(pkg, sess, n_q, n_kv, kind):
    """d_head 128, more queries than keys under the causal mask: of a CTA's two tiles the first sees no key and the
    second does.  Every launch comes behind other work that leaves the caches cold; the rows without a key are
    exactly 0 each time."""
    a = Attention(2, 4, 2, n_q, n_kv, 128, kind, causal=True)
    a.check(a.run(pkg, sess))
    B = pkg.blob
    ptrs = [sess.upload(_bits(t)) for t in (a.q, a.k, a.v)]
    kernel = sess.kernel(B.attention("cold", *a.dims, dtype=_dt(pkg, kind), causal=True))
    assert sess.workspace_bytes(kernel) == 0
    spoil = torch.empty(64 << 20, device="cuda")
    for _ in range(20):
        spoil.fill_(1.0)
        torch.cuda.synchronize()
        o, lse = Output(sess, a.q.numel(), kind), Output(sess, 8 * n_q, "f32")
        sess.launch(kernel, ptrs + [o.ptr, lse.ptr])
        assert (o.get(a.q.shape)[:, :, :n_q - n_kv] == 0).all()
        assert np.isneginf(lse.get((2, 4, n_q)).numpy()[:, :, :n_q - n_kv]).all()
        for x in (o, lse):
            sess.free(x.base)


# The blocks of a tile of dQ, and of one of dK and dV, are shared out between 1, 2 or 4 CTAs each, in one grid whose
# clusters have the size of the larger number; CTAs that only fill the last cluster of dQ's tiles have none.
SHARES = [
    # q_heads, kv_heads, n_q, n_kv, d, causal: shares of dQ, of dK and dV
    (1, 1, 300, 100, 64, True),       # 1, 2, an empty CTA
    (8, 1, 1, 100, 64, True),         # 1, 4
    (3, 1, 130, 100, 64, True),       # 1, 4, two empty CTAs
    (1, 1, 1, 300, 64, False),        # 2, 1, an empty CTA behind dK and dV
    (8, 1, 1, 200, 64, False),        # 2, 4
    (1, 1, 520, 200, 64, True),       # 2, 4, two empty CTAs
    (1, 1, 1, 700, 64, False),        # 4, 1, two empty CTAs
    (4, 1, 1, 500, 64, True),         # 4, 2
    (8, 1, 1, 500, 64, False),        # 4, 4
    (3, 1, 300, 100, 128, False),     # 1, 2, an empty CTA
    (8, 1, 130, 100, 128, True),      # 1, 4
    (1, 1, 1, 1000, 128, True),       # 2, 1
    (8, 1, 1, 1000, 128, True),       # 2, 2
    (8, 1, 130, 1000, 128, True),     # 2, 4
    (1, 1, 3, 2100, 128, True),       # 4, 1
]


@pytest.mark.parametrize("case", SHARES, ids=lambda c: "-".join(str(x) for x in c))
@pytest.mark.parametrize("lens", [False, True], ids=["", "lens"])
def test_attention_gradients_by_shares(pkg, sess, case, lens):
    """Also with what the workspace holds replaced by NaN before every launch: the row sums of the launch are read, not
    those of the one before."""
    q_heads, kv_heads, n_q, n_kv, d, causal = case
    a = Attention(2 if lens else 1, q_heads, kv_heads, n_q, n_kv, d, "bf16", causal, [n_kv, n_kv // 3] if lens else None, "tokens")
    got = a.run(pkg, sess)
    first = {n: got[n].clone() for n in ("dq", "dk", "dv")}
    o, lse = a.laid(got["o"]), got["lse"].clone()
    a.check(got)
    B = pkg.blob
    kernel = sess.kernel(B.attention_bwd("again", *a.dims, causal=causal, key_lens=lens, layout="tokens"))
    need = sess.workspace_bytes(kernel)
    nan, work = np.full(need // 4, np.nan, np.float32), sess.alloc(need)
    outs = [Output(sess, t.numel(), "bf16") for t in (a.q, a.k, a.v)]
    args = [sess.upload(_bits(a.laid(t))) for t in (a.q, a.k, a.v)]
    args += [sess.upload(_bits(o)), sess.upload(_bits(a.laid(a.do))), sess.upload(lse.numpy())] + [x.ptr for x in outs]
    args += [sess.upload(np.array(a.lens, np.int32))] if lens else []
    spoil = torch.empty(64 << 20, device="cuda")
    for _ in range(5):
        pkg.runtime.gpuMemCopy(sess.stream, work, nan.ctypes.data, need)
        spoil.fill_(1.0)
        torch.cuda.synchronize()
        sess.launch(kernel, args + [work])
        for x, n, t in zip(outs, first, (a.q, a.k, a.v)):
            assert torch.equal(a.back(x.get(-1), t.shape), first[n]), n
