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
