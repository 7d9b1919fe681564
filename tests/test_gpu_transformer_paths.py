"""The ways through the attention and gated feed-forward kernels that only some shapes take, each against its formula in
64 bits; the tolerances are those of test_gpu_transformer_ops.py."""
import subprocess
import sys

import numpy as np
import pytest
import torch

from __graft_entry__ import ROOT, load_package
from test_gpu_transformer_ops import HALF_STEP, SENTINEL, TORCH, Attention, Output, _bits, _dt, _launch, _rand

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


# --------------------------------------------------------------------------------------- gated product
class Gated:
    """A problem on the GPU with rows behind one another or `pitch` elements further apart, exact results and tolerances
    as in test_gpu_transformer_ops.py."""

    def __init__(self, m, d, f, kind, pitch=0):
        self.m, self.d, self.f, self.kind = m, d, f, kind
        self.u = HALF_STEP[kind]
        self.pitches = dict(ldx=d + pitch, ldw=2 * f + pitch, ldh=f + pitch) if pitch else {}
        self.x, self.w, self.dh = self.new(m, d, 1, pitch), self.new(d, 2 * f, 2, pitch, d ** -0.5), self.new(m, f, 3, pitch)

    def new(self, rows, cols, seed, pitch, std=1.0):
        g = torch.Generator("cuda").manual_seed(seed)
        return (torch.randn((rows, cols + pitch), generator=g, device="cuda") * std).to(TORCH[self.kind])[:, :cols]

    def like(self, t):
        """A result of t's shape and pitch, NaN, also between its rows."""
        whole = torch.full((t.shape[0], t.stride(0)), float("nan"), dtype=t.dtype, device="cuda")
        return whole, whole[:, :t.shape[1]]

    def launches(self, pkg, desc, tensors, outs, times=1):
        """The results of `times` launches, each with NaN in the workspace before it; the same bits each time."""
        with pkg.Session(device=torch.cuda.current_device(), adopt_stream=1) as s:
            kernel = s.kernel(desc)
            need = s.workspace_bytes(kernel)
            work = [torch.empty(need, dtype=torch.uint8, device="cuda")] if need else []
            run = s.bind(kernel, [t.data_ptr() for t in tensors + [o[1] for o in outs] + work])
            first = None
            for _ in range(times):
                for t in work + [o[0] for o in outs]:
                    t.fill_(255 if t.dtype == torch.uint8 else float("nan"))
                run()
                got = [o[1].clone() for o in outs]
                first = first or got
                assert all(torch.equal(a.view(torch.int16), b.view(torch.int16)) for a, b in zip(first, got))
            for whole, t in outs:
                assert torch.isnan(whole[:, t.shape[1]:]).all(), "written between the rows"
            s.wait()
        return first

    def forward(self, pkg, save=True, times=1):
        outs = [self.like(self.dh)] + ([self.like(torch.empty((self.m, 2 * self.f), dtype=self.x.dtype, device="cuda"))] if save else [])
        desc = pkg.blob.gated_ffn("g", self.m, self.d, self.f, _dt(pkg, self.kind), save_gu=save, **self.pitches)
        got = self.launches(pkg, desc, [self.x, self.w], outs, times)
        x, w, f = self.x.double(), self.w.double(), self.f
        z = x @ w
        acc = 2.0 ** -24 * (self.d + 8) * (x.abs() @ w.abs()) + 2.0 ** -25
        a, up = torch.nn.functional.silu(z[:, :f]), z[:, f:]
        want = a * up
        tol = 1.1 * acc[:, :f] * (up.abs() + acc[:, f:]) + a.abs() * acc[:, f:] + (self.u + 4e-6) * want.abs() + 2.0 ** -25
        assert ((got[0].double() - want).abs() <= tol * 1.01).all()
        if save:
            assert ((got[1].double() - z).abs() <= (acc + self.u * z.abs()) * 1.01).all()

    def backward(self, pkg, times=3):
        f, tiny = self.f, 2.0 ** -25
        gu = (self.x.float() @ self.w.float()).to(TORCH[self.kind])
        desc = pkg.blob.gated_ffn_bwd("gb", self.m, self.d, f, _dt(pkg, self.kind), **self.pitches)
        dx, dw = self.launches(pkg, desc, [self.x, self.w, gu, self.dh], [self.like(self.x), self.like(self.w)], times)
        z = gu.double().requires_grad_(True)
        dz, = torch.autograd.grad(torch.nn.functional.silu(z[:, :f]) * z[:, f:], z, self.dh.double())
        x, w = self.x.double(), self.w.double()
        e = (self.u + 1e-5) * dz.abs() + tiny
        for got, want, size, terms in ((dx, dz @ w.t(), e @ w.abs().t(), dz.abs() @ w.abs().t()),
                                       (dw, x.t() @ dz, x.abs().t() @ e, x.abs().t() @ dz.abs())):
            tol = size + self.u * want.abs() + 2.0 ** -24 * (max(self.m, 2 * f) + 8) * terms + tiny
            assert ((got.double() - want).abs() <= tol * 1.01).all()


@pytest.mark.parametrize("m,d,f,kind,pitch", [
    (2048, 4096, 2064, "bf16", 0),   # dX by CTA pairs, then dW's small tiles
    (2305, 1000, 4808, "f16", 0),    # dX by small tiles, then dW by CTA pairs
    (2400, 2056, 2200, "bf16", 0),   # both by CTA pairs
    (2400, 2056, 2200, "f16", 8),
    (300, 1000, 2720, "f16", 0),     # both by small tiles in one grid, dX's k in four shares
    (257, 520, 2600, "bf16", 0),     # fifteen tiles of dX
    (150, 296, 1400, "bf16", 16),    # dX's k in two
    (2600, 256, 104, "f16", 0),      # dW's k in two
    (70, 4100, 30, "f16", 3),        # copied operands
])
def test_gated_gradients_by_products(pkg, m, d, f, kind, pitch):
    Gated(m, d, f, kind, pitch).backward(pkg)


def test_large_products_on_a_second_device(pkg):
    """Sessions on two devices in one process: what a kernel needs is asked for on each."""
    if torch.cuda.device_count() < 2:
        pytest.skip("one CUDA device")
    for device in (0, 1):
        with torch.cuda.device(device):
            Gated(2400, 2056, 2200, "bf16").backward(pkg, times=1)


# ----------------------------------------------------------------------------- values that are not finite
@pytest.mark.parametrize("q_heads,kv_heads,n_q,n_kv,d,causal", [
    (2, 2, 140, 140, 64, True), (4, 2, 300, 300, 128, True), (2, 1, 3, 260, 64, False), (4, 1, 2, 515, 128, True),
    (4, 1, 1, 3000, 128, False), (2, 1, 2, 2500, 64, True), (1, 1, 200, 2000, 128, True)])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), 1e38], ids=str)
def test_scores_that_are_not_finite_make_their_rows_nan(pkg, sess, q_heads, kv_heads, n_q, n_kv, d, causal, bad):
    """A NaN or infinite key, or one whose scores overflow (the sum of products leaves f32): O and LSE of the rows that
    see it are NaN, the other rows are what they are without it.  A query of NaN: its row alone."""
    a = Attention(1, q_heads, kv_heads, n_q, n_kv, d, "bf16", causal)
    a.q[0, 0] = a.q[0, 0].abs() + 4.0
    key = n_kv - n_q + n_q // 2 if causal else n_kv // 2
    a.k[0, 0, key] = bad
    row = n_q // 3
    a.q[0, 1 % q_heads, row] = float("nan")
    got = a.run(pkg, sess, backward=False)
    sees = torch.arange(n_q) >= (key - (n_kv - n_q) if causal else 0)
    nan = torch.zeros((q_heads, n_q), dtype=torch.bool)
    nan[:q_heads // kv_heads] |= sees
    if bad != bad or bad == float("inf"):
        touched = nan.clone()
    else:  # the overflow of the head whose queries are positive; the others' may cancel
        touched = torch.zeros_like(nan)
        touched[0] = nan[0]
    touched[1 % q_heads, row] = True
    nan[1 % q_heads, row] = True
    assert torch.isnan(got["lse"][0][touched]).all() and torch.isnan(got["o"][0][touched]).all()
    a.k[0, 0, key], a.q[0, 1 % q_heads, row] = 0.0, 0.0
    ref, tol = a.exact()
    off = (got["o"].double() - ref["o"]).abs()[0] / tol["o"][0]
    assert (off[~nan] <= 1.0).all()
    assert (got["lse"].double() - ref["lse"]).abs()[0][~nan].le(2e-5 + 1e-6 * ref["lse"][0][~nan].abs()).all()


@pytest.mark.parametrize("d,n_q,n_kv", [(64, 140, 140), (128, 1, 2000)])
def test_a_score_of_minus_infinity_has_no_weight(pkg, sess, d, n_q, n_kv):
    a = Attention(1, 2, 1, n_q, n_kv, d, "bf16")
    a.q = a.q.abs() + 1.0
    a.k[0, 0, 7] = -3e38
    a.check(a.run(pkg, sess, backward=False))


# ------------------------------------------------------------------------------------ arrays in one another's place
def _refusals(cases):
    """(builder call, number of pointers, what is done to them, message): refused before anything is launched, by one line
    on stdout and abort().  A process each, side by side."""
    runs = []
    for make, n, patch, message in cases:
        text = ("from __graft_entry__ import load_package\npkg = load_package()\nB = pkg.blob\ns = pkg.Session(device=0)\n"
                "k = s.kernel(B.%s)\np = [s.alloc(1 << 16) for _ in range(%d)]\n%s\ns.launch(k, p)\n" % (make, n, patch))
        runs.append((subprocess.Popen([sys.executable, "-c", text], cwd=ROOT, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True),
                     make, patch, message))
    for process, make, patch, message in runs:
        out, _ = process.communicate(timeout=300)
        assert process.returncode == -6 and message in out, (make, patch, out)


def test_outputs_in_the_place_of_inputs_are_refused():
    """No value is looked at: all buffers are large enough for what would run."""
    attention, wide = "attention('a', 2, 2, 2, 8, 8, 64%s)", ", strides={'o': (2048, 1024, 128)}"
    back, grads = "attention_bwd('a', 1, 1, 1, 8, 8, 64)", "dQ, dK and dV may not be"
    _refusals([
        (attention % "", 5, "p[3] = p[1]", "O may not be K or V"),
        (attention % "", 5, "p[3] = p[2]", "O may not be K or V"),
        (attention % wide, 5, "p[3] = p[0]", "nor Q with other strides"),
        (back, 10, "p[6] = p[0]", grads), (back, 10, "p[7] = p[4]", grads), (back, 10, "p[8] = p[2]", grads), (back, 10, "p[8] = p[7]", grads),
        ("gated_ffn('a', 4, 16, 16)", 3, "p[2] = p[0]", "H and GU may not be"),
        ("gated_ffn('a', 4, 16, 16, save_gu=True)", 4, "p[3] = p[2]", "H and GU may not be"),
        ("gated_ffn_bwd('a', 4, 16, 16)", 7, "p[6] = s.alloc(s.workspace_bytes(k)); p[4] = p[0]", "dX and dW may not be"),
        ("gated_ffn_bwd('a', 4, 16, 16)", 7, "p[6] = s.alloc(s.workspace_bytes(k)); p[5] = p[1]", "dX and dW may not be"),
        ("rotary('a', 4, 2, 64, [1.0], x_strides=(192, 64))", 3, "p[2] = p[0]", "in place, X and Y have the same strides"),
    ])


@pytest.mark.parametrize("q_heads,kv_heads,n_q,n_kv,d", [(4, 2, 300, 300, 64), (4, 2, 300, 300, 128), (4, 1, 1, 3000, 128), (2, 2, 200, 2000, 64)])
def test_attention_output_in_the_place_of_q(pkg, sess, q_heads, kv_heads, n_q, n_kv, d):
    a = Attention(1, q_heads, kv_heads, n_q, n_kv, d, "bf16", True)
    want = a.run(pkg, sess, backward=False)
    kernel = sess.kernel(pkg.blob.attention("in_place", *a.dims, causal=True))
    q, k, v = (sess.upload(_bits(t)) for t in (a.q, a.k, a.v))
    lse = Output(sess, q_heads * n_q, "f32")
    need = sess.workspace_bytes(kernel)
    sess.launch(kernel, [q, k, v, q, lse.ptr] + ([sess.alloc(need)] if need else []))
    assert np.array_equal(sess.download(q, a.q.shape, np.int16), _bits(want["o"]))


def test_gradients_in_the_place_of_what_is_read_before_them(pkg):
    """The gated product's GU and dH, and attention's O, have been read when the gradients are written."""
    a = Gated(300, 264, 264, "bf16")
    gu = (a.x.float() @ a.w.float()).to(torch.bfloat16)
    desc = pkg.blob.gated_ffn_bwd("gb", 300, 264, 264)
    outs = [a.like(a.x), a.like(a.w)]
    want = a.launches(pkg, desc, [a.x, a.w, gu, a.dh], outs)
    with pkg.Session(device=0, adopt_stream=1) as s:
        kernel = s.kernel(desc)
        work, dh = torch.empty(s.workspace_bytes(kernel), dtype=torch.uint8, device="cuda"), a.dh.clone()
        s.launch(kernel, [t.data_ptr() for t in (a.x, a.w, gu, dh, dh, outs[1][1], work)])
    assert torch.equal(dh, want[0]) and torch.equal(outs[1][1], want[1])
    t = lambda *shape: torch.randn(shape, device="cuda").to(torch.bfloat16)  # noqa: E731
    q, k, v, o, do = (t(2, 4, 333, 128) for _ in range(5))
    lse = torch.full((2, 4, 333), 6.0, device="cuda")
    grads = [torch.empty_like(q) for _ in range(3)]
    with pkg.Session(device=0, adopt_stream=1) as s:
        kernel = s.kernel(pkg.blob.attention_bwd("b", 2, 4, 4, 333, 333, 128))
        work = torch.empty(s.workspace_bytes(kernel), dtype=torch.uint8, device="cuda")
        s.launch(kernel, [x.data_ptr() for x in [q, k, v, o, do, lse] + grads + [work]])
        s.launch(kernel, [x.data_ptr() for x in [q, k, v, o, do, lse, o] + grads[1:] + [work]])
    assert torch.equal(o, grads[0])


def test_missing_and_surplus_arrays_are_refused():
    """A null is no array; one array too many would take the workspace's place."""
    split, back = "attention('a', 1, 1, 1, 1, 3000, 64%s)", "attention_bwd('a', 1, 1, 1, 8, 8, 64%s)"
    _refusals([
        ("attention('a', 1, 1, 1, 8, 8, 64, key_lens=True)", 6, "p[5] = 0", "needs 6 pointer arguments, got 5"),
        ("gated_ffn('a', 4, 16, 16, save_gu=True)", 4, "p[3] = 0", "needs 4 pointer arguments, got 3"),
        (split % "", 6, "p[5] = 0", "needs 6 pointer arguments, got 5"),
        (split % "", 7, "", "takes 6 pointer arguments, the last its workspace, got 7"),
        (split % ", key_lens=True", 8, "", "takes 7 pointer arguments, the last its workspace, got 8"),
        (back % "", 11, "", "takes 10 pointer arguments, the last its workspace, got 11"),
        ("gated_ffn('a', 4, 15, 16)", 5, "", "takes 4 pointer arguments, the last its workspace, got 5"),
        ("gated_ffn_bwd('a', 4, 16, 16)", 8, "", "takes 7 pointer arguments, the last its workspace, got 8"),
        ("rotary('a', 4, 2, 64, [1.0])", 3, "p[1] = 0", "needs 3 pointer arguments, got 2"),
    ])


def test_a_workspace_where_none_is_needed_is_not_used(pkg, sess):
    a = Attention(1, 2, 2, 20, 30, 64, "bf16")
    kernel = sess.kernel(pkg.blob.attention("a", *a.dims))
    assert sess.workspace_bytes(kernel) == 0
    o, lse, spare = Output(sess, a.q.numel(), "bf16"), Output(sess, 40, "f32"), Output(sess, 64, "f32")
    sess.launch(kernel, [sess.upload(_bits(t)) for t in (a.q, a.k, a.v)] + [o.ptr, lse.ptr, spare.ptr])
    a.check({"o": o.get(a.q.shape), "lse": lse.get((1, 2, 20))})
    assert (_bits(spare.get(-1)) == SENTINEL).all()


# -------------------------------------------------------------------------- keys shared out between CTAs, and joined
SPLIT = [
    # batch, q_heads, kv_heads, n_q, n_kv, d, kind, causal, lens, layout
    (4, 4, 2, 1, 3000, 64, "bf16", False, [3000, 0, 1, 300], "heads"),        # six shares, most of them empty
    (4, 4, 2, 1, 3000, 128, "f16", True, [3000, 0, 1, 300], "tokens"),
    (3, 8, 1, 5, 2600, 64, "f16", True, [2600, 130, 1999], "tokens"),         # the last key inside a later share's block
    (3, 8, 1, 5, 2600, 128, "bf16", False, [2600, 130, 1999], "heads"),
    (1, 1, 1, 1, 33000, 64, "bf16", False, None, "heads"),                    # 52 shares
    (1, 2, 1, 1, 33000, 128, "bf16", True, None, "heads"),
    (2, 1, 1, 1, 33000, 128, "f16", False, [31111, 5], "heads"),
    (1, 2, 2, 300, 2000, 64, "bf16", True, None, "heads"),                    # a tile per 128 queries
    (1, 2, 2, 300, 2000, 128, "f16", True, None, "tokens"),
    (2, 3, 1, 140, 1800, 128, "bf16", False, [1800, 500], "tokens"),
    (2, 3, 1, 140, 1800, 64, "f16", True, [0, 1733], "heads"),
    (1, 1, 1, 700, 5000, 128, "bf16", True, None, "heads"),                   # ten shares of pairs that end unequally
    (1, 1, 1, 3000, 2600, 128, "bf16", True, None, "heads"),                  # the first queries see no key
]


@pytest.mark.parametrize("case", SPLIT, ids=lambda c: "-".join(str(x) for x in c).replace(" ", ""))
def test_attention_with_keys_shared_out(pkg, sess, case):
    a = Attention(*case)
    if a.lens is not None:
        a.poison_padding()
    desc = pkg.blob.attention("a", *a.dims, dtype=_dt(pkg, a.kind), causal=a.causal, key_lens=a.lens is not None, layout=a.layout)
    assert sess.workspace_bytes(sess.kernel(desc)) > 0, "one share"
    a.check(a.run(pkg, sess))


@pytest.mark.parametrize("m,d,f,kind,pitch", [
    (2100, 136, 2824, "bf16", 0),    # 207 tiles on 74 pairs of CTAs, two k blocks
    (4200, 264, 2824, "f16", 0),     # 391 tiles, three bands of row blocks, three k blocks
    (5000, 8, 1160, "bf16", 0),      # one k block
    (2600, 1000, 2000, "bf16", 8),   # rows with a pitch
    (2500, 2051, 1301, "f16", 0),    # copied operands, results stored value by value
])
@pytest.mark.parametrize("save", [False, True], ids=["", "kept"])
def test_gated_pairs_of_ctas_walk_several_tiles(pkg, m, d, f, kind, pitch, save):
    Gated(m, d, f, kind, pitch).forward(pkg, save, times=3)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("place", [0, 1, 2], ids=["dq", "dk", "dv"])
def test_attention_gradients_in_the_place_of_o(pkg, d, place):
    """Also those of keys that no query sees, whose zeros depend on nothing: they go out when O has been read.  Cold caches
    before every launch."""
    t = lambda *shape: torch.randn(shape, device="cuda").to(torch.bfloat16)  # noqa: E731
    dims = (8, 16, 16, 600, 600, d)
    q, k, v, kept, do = (t(8, 16, 600, d) for _ in range(5))
    lse, lens = torch.full((8, 16, 600), 6.0, device="cuda"), torch.tensor([0, 600, 1, 0, 100, 0, 0, 599], dtype=torch.int32, device="cuda")
    want, o, spoil = [torch.empty_like(q) for _ in range(3)], torch.empty_like(q), torch.empty(64 << 20, device="cuda")
    got = [o if i == place else torch.empty_like(q) for i in range(3)]
    with pkg.Session(device=0, adopt_stream=1) as s:
        kernel = s.kernel(pkg.blob.attention_bwd("b", *dims, key_lens=True))
        work = torch.empty(s.workspace_bytes(kernel), dtype=torch.uint8, device="cuda")
        s.launch(kernel, [x.data_ptr() for x in [q, k, v, kept, do, lse] + want + [lens, work]])
        run = s.bind(kernel, [x.data_ptr() for x in [q, k, v, o, do, lse] + got + [lens, work]])
        for _ in range(10):
            o.copy_(kept)
            spoil.fill_(1.0)
            run()
            assert all(torch.equal(a, b) for a, b in zip(got, want))
        s.wait()


# ------------------------------------------------------------------------------------------------ far offsets
def test_offsets_beyond_32_bits(pkg):
    """Sequences, rows and tokens more than 2^31 elements apart: the same bits as side by side."""
    B, step = pkg.blob, 2 ** 30 + 8
    big = torch.zeros(3 * step + 4096 * 64, dtype=torch.bfloat16, device="cuda")   # 6.5 GB
    at = lambda offset, shape, strides: torch.as_strided(big, shape, strides, offset)  # noqa: E731
    new = lambda *shape: torch.randn(shape, device="cuda").to(torch.bfloat16)  # noqa: E731
    with pkg.Session(device=0, adopt_stream=1) as s:
        def launch(desc, tensors):
            kernel = s.kernel(desc)
            need = s.workspace_bytes(kernel)
            work = [torch.empty(need, dtype=torch.uint8, device="cuda")] if need else []
            s.launch(kernel, [t.data_ptr() for t in tensors + work])

        # attention: four sequences of 40 rows of 64, each array in a part of its own of every 2^30
        dims, far = (4, 2, 2, 40, 40, 64), (step, 40 * 64, 64)
        near = {n: new(4, 2, 40, 64) for n in ("q", "k", "v", "do")}
        outs = {n: torch.empty_like(near["q"]) for n in ("o", "dq", "dk", "dv")}
        lse = torch.empty((4, 2, 40), device="cuda")
        names = ("q", "k", "v", "o", "do", "dq", "dk", "dv")
        wide = {n: at(i * 8192, (4, 2, 40, 64), (step, 40 * 64, 64, 1)) for i, n in enumerate(names)}
        for n, t in near.items():
            wide[n].copy_(t)
        strides = {n: far for n in names}
        both = dict(near, **outs)
        for t, kw in ((both, {}), (wide, {"strides": strides})):
            launch(B.attention("a", *dims, causal=True, **kw), [t[n] for n in ("q", "k", "v", "o")] + [lse])
            launch(B.attention_bwd("b", *dims, causal=True, **kw), [t[n] for n in ("q", "k", "v", "o", "do")] + [lse] + [t[n] for n in ("dq", "dk", "dv")])
        for n in outs:
            assert torch.equal(outs[n], wide[n]), n
        # gated product: X, H and dH with their rows 2^30 apart (dX has X's pitch)
        m, d, f = 4, 128, 136
        x, w, dh, gu = new(m, d), new(d, 2 * f), new(m, f), torch.empty((m, 2 * f), dtype=torch.bfloat16, device="cuda")
        h, dx, dw = torch.empty_like(dh), torch.empty_like(x), torch.empty_like(w)
        xs, hs, dhs, dxs = (at(i * 8192, (m, c), (step, 1)) for i, c in enumerate((d, f, f, d)))
        xs.copy_(x), dhs.copy_(dh)
        dw2, gu2 = torch.empty_like(dw), torch.empty_like(gu)
        launch(B.gated_ffn("g", m, d, f, save_gu=True), [x, w, h, gu])
        launch(B.gated_ffn_bwd("gb", m, d, f), [x, w, gu, dh, dx, dw])
        launch(B.gated_ffn("g", m, d, f, save_gu=True, ldx=step, ldh=step), [xs, w, hs, gu2])
        launch(B.gated_ffn_bwd("gb", m, d, f, ldx=step, ldh=step), [xs, w, gu, dhs, dxs, dw2])
        for a, b in ((h, hs), (gu, gu2), (dx, dxs), (dw, dw2)):
            assert torch.equal(a, b)
        # rotary: tokens 2^30 apart
        x, y, pos = new(4, 3, 64), torch.empty((4, 3, 64), dtype=torch.bfloat16, device="cuda"), torch.arange(4, dtype=torch.int32, device="cuda")
        xs, ys = (at(i * 8192, (4, 3, 64), (step, 64, 1)) for i in range(2))
        xs.copy_(x)
        freqs = B.rotary_frequencies(64)
        launch(B.rotary("r", 4, 3, 64, freqs), [x, pos, y])
        launch(B.rotary("r", 4, 3, 64, freqs, x_strides=(step, 64), y_strides=(step, 64)), [xs, pos, ys])
        assert torch.equal(y, ys)


def test_many_rows_of_one_head_pass_32_bits(pkg):
    """2^24 + 100 keys of 128: offsets inside one head beyond 2^31 elements, one query, by shares.  All weights are equal but
    for the last keys', so O is known."""
    n, d = 2 ** 24 + 100, 128
    k, v = torch.zeros((1, 1, n, d), dtype=torch.bfloat16, device="cuda"), torch.ones((1, 1, n, d), dtype=torch.bfloat16, device="cuda")
    q = torch.ones((1, 1, 1, d), dtype=torch.bfloat16, device="cuda")
    k[0, 0, -3:] = 2.0           # scores 256 / sqrt(128) = 22.6: three keys against 2^24 of weight 1
    v[0, 0, -3:] = -3.0
    o, lse = torch.empty_like(q), torch.empty((1, 1, 1), device="cuda")
    with pkg.Session(device=0, adopt_stream=1) as s:
        kernel = s.kernel(pkg.blob.attention("a", 1, 1, 1, 1, n, d))
        work = torch.empty(s.workspace_bytes(kernel), dtype=torch.uint8, device="cuda")
        s.launch(kernel, [t.data_ptr() for t in (q, k, v, o, lse, work)])
    heavy = 3 * np.exp(256 / np.sqrt(128.0))
    total = n - 3 + heavy
    want = (n - 3 - 3 * heavy) / total
    # P of the heavy keys is 1 (the reference maximum) and exact; those of the light ones e^-22.6 rounded to bf16, all
    # the same way: half a step of their share of the sum; then O's own half step
    assert abs(o.double().cpu() - want).max() <= 2.0 ** -8 * ((n - 3) / total + abs(want)) + 1e-4
    assert abs(lse.item() - np.log(total)) <= 2e-5 + 1e-6 * np.log(total) + 1e-4


# ---------------------------------------------------------------------------------------------- several at once
def test_sessions_on_several_streams_at_once(pkg):
    """Three streams with a session, buffers and workspaces each, all operators back to back on each: the results of
    every stream are those of the calls alone."""
    B, chains = pkg.blob, []
    new = lambda *shape: torch.randn(shape, device="cuda").to(torch.bfloat16)  # noqa: E731
    torch.manual_seed(5)
    torch.cuda.synchronize()
    for i, (d, n, heads, kv) in enumerate([(64, 520, 12, 3), (128, 400, 8, 2), (64, 300, 16, 16)]):
        stream = torch.cuda.Stream()
        s = pkg.Session(device=0, adopt_stream=stream.cuda_stream)
        q, do, k, v = new(2, heads, n, d), new(2, heads, n, d), new(2, kv, n, d), new(2, kv, n, d)
        q1, k1, v1 = new(2, heads, 1, d), new(2, kv, 2500, d), new(2, kv, 2500, d)
        x, w, dh = new(n, 256), new(256, 2 * 520), new(n, 520)
        out = {name: torch.empty_like(t) for name, t in dict(o=q, dq=q, dk=k, dv=v, o1=q1, dx=x, dw=w, h=dh, turned=q).items()}
        out["gu"] = torch.empty((n, 2 * 520), dtype=torch.bfloat16, device="cuda")
        out["lse"], out["lse1"] = torch.empty((2, heads, n), device="cuda"), torch.empty((2, heads, 1), device="cuda")
        pos = torch.arange(2 * heads * n, dtype=torch.int32, device="cuda")
        dims, dims1 = (2, heads, kv, n, n, d), (2, heads, kv, 1, 2500, d)
        calls = [(B.rotary("r", 2 * heads * n, 1, d, B.rotary_frequencies(d)), [q, pos, out["turned"]]),
                 (B.attention("a", *dims, causal=True), [q, k, v, out["o"], out["lse"]]),
                 (B.attention("a1", *dims1), [q1, k1, v1, out["o1"], out["lse1"]]),
                 (B.gated_ffn("g", n, 256, 520, save_gu=True), [x, w, out["h"], out["gu"]]),
                 (B.attention_bwd("b", *dims, causal=True), [q, k, v, out["o"], do, out["lse"], out["dq"], out["dk"], out["dv"]]),
                 (B.gated_ffn_bwd("gb", n, 256, 520), [x, w, out["gu"], dh, out["dx"], out["dw"]])]
        launches, keep = [], [stream]
        for desc, args in calls:
            kernel = s.kernel(desc)
            need = s.workspace_bytes(kernel)
            args = args + ([torch.empty(need, dtype=torch.uint8, device="cuda")] if need else [])
            keep.append(args)
            launches.append(s.bind(kernel, [t.data_ptr() for t in args]))
        chains.append((s, launches, out, keep))
    torch.cuda.synchronize()
    alone = []
    for s, launches, out, _ in chains:
        for run in launches:
            run()
        s.wait()
        alone.append({n: t.clone() for n, t in out.items()})
    torch.cuda.synchronize()
    for _ in range(30):
        for j in range(len(chains[0][1])):
            for s, launches, _, _ in chains:
                launches[j]()
    for (s, _, out, _), want in zip(chains, alone):
        s.wait()
        for n in out:
            assert torch.equal(out[n], want[n]), n
        s.close()


def test_captured_gradients_by_products_and_shares(pkg):
    """The mixed orders of the gated backward pass and clusters of attention's, captured and replayed on other inputs: the
    bits of direct launches."""
    B, stream = pkg.blob, torch.cuda.Stream()
    with torch.cuda.stream(stream), pkg.Session(device=0, adopt_stream=stream.cuda_stream) as s:
        new = lambda *shape: torch.randn(shape, device="cuda").to(torch.bfloat16)  # noqa: E731
        ins, outs, launches, keep = [], [], [], []

        def bind(desc, args):
            kernel = s.kernel(desc)
            need = s.workspace_bytes(kernel)
            keep.append(args + ([torch.empty(need, dtype=torch.uint8, device="cuda")] if need else []))
            launches.append(s.bind(kernel, [t.data_ptr() for t in keep[-1]]))
        for m, d, f in ((2048, 4096, 2064), (2305, 1000, 4808), (2400, 2056, 2200), (300, 1000, 2720), (70, 410, 30), (33, 41, 65)):
            x, w, gu, dh = new(m, d), new(d, 2 * f), new(m, 2 * f), new(m, f)
            h, kept, dx, dw = torch.empty_like(dh), torch.empty_like(gu), torch.empty_like(x), torch.empty_like(w)
            bind(B.gated_ffn("g", m, d, f, save_gu=True), [x, w, h, kept])
            bind(B.gated_ffn_bwd("gb", m, d, f), [x, w, gu, dh, dx, dw])
            ins += [x, w, gu, dh]
            outs += [h, kept, dx, dw]
        for q_heads, kv_heads, n_q, n_kv, d, causal in SHARES:
            q, do, o = (new(1, n_q, q_heads, d) for _ in range(3))
            k, v = (new(1, n_kv, kv_heads, d) for _ in range(2))
            lse = torch.full((1, q_heads, n_q), 5.0, device="cuda")
            grads = [torch.empty_like(t) for t in (q, k, v)]
            bind(B.attention_bwd("b", 1, q_heads, kv_heads, n_q, n_kv, d, causal=causal, layout="tokens"), [q, k, v, o, do, lse] + grads)
            ins += [q, k, v, o, do]
            outs += grads
        for run in launches:
            run()
        stream.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            for run in launches:
                run()
        for t in ins:
            t.copy_(new(*t.shape))
        for run in launches:
            run()
        stream.synchronize()
        want = [t.clone() for t in outs]
        for t in outs:
            t.zero_()
        for _ in range(3):
            graph.replay()
        stream.synchronize()
        s.wait()
        assert all(torch.equal(a.view(torch.int16), b.view(torch.int16)) for a, b in zip(outs, want))


@pytest.mark.parametrize("m,d,f", [(130, 64, 72), (130, 33, 41)])
def test_the_slope_of_relu_at_zero_is_zero(pkg, sess, m, d, f):
    x, w = _rand((m, d), "f16", 1), _rand((d, 2 * f), "f16", 2, d ** -0.5)
    gu, dh = _rand((m, 2 * f), "f16", 3), _rand((m, f), "f16", 4)
    gu[:, :f][::2] = 0.0
    gu[:, :f][::4] = -0.0
    dx, dw = Output(sess, m * d, "f16"), Output(sess, d * 2 * f, "f16")
    _launch(sess, pkg.blob.gated_ffn_bwd("gb", m, d, f, pkg.blob.F16, pkg.blob.EPI_RELU),
            [sess.upload(_bits(t)) for t in (x, w, gu, dh)] + [dx.ptr, dw.ptr])
    g, u = gu[:, :f].double(), gu[:, f:].double()
    dz = torch.cat([dh.double() * u * (g > 0), dh.double() * g.clamp(min=0)], 1)
    e = (2.0 ** -11 + 1e-5) * dz.abs() + 2.0 ** -25
    for got, want, size, terms in ((dx.get((m, d)), dz @ w.double().t(), e @ w.double().abs().t(), dz.abs() @ w.double().abs().t()),
                                   (dw.get((d, 2 * f)), x.double().t() @ dz, x.double().abs().t() @ e, x.double().abs().t() @ dz.abs())):
        tol = size + 2.0 ** -11 * want.abs() + 2.0 ** -24 * (max(m, 2 * f) + 8) * terms + 2.0 ** -25
        assert ((got.double() - want).abs() <= tol * 1.01).all()
