"""Attention with row statistics and its backward pass, the gated feed-forward product and its backward pass, and
rotary positions, through the C ABI, against their formulas in 64 bits.

Tolerances count roundings.  u is half a step of the 16-bit type (bf16 2^-8, f16 2^-11).  The kernels round the
probabilities (and dS) once to the 16-bit type before the second product and every result once, so

    |O  - exact| <= u P|V| + u |O|                      and for f16, whose smallest step is 2^-24, 2^-25 sum |V|
    |dV - exact| <= u P^T|dO| + u |dV|                  (f16: 2^-25 sum |dO|)
    |dQ - exact| <= scale E |K| + u |dQ|,   |dK - exact| <= scale E^T |Q| + u |dK|
         E = u |dS| + P (u |dO| . |O|) + 2^-25 (f16)    since delta = dO . O is taken from the rounded O

plus what 32-bit arithmetic leaves: F = 2e-5 relative on P (a score is a sum of d_head products, |S| up to ten or so:
d_head 2^-24 sum |q||k| scale, the exponential 2^-22) and on sums of up to a few thousand terms."""
import math
import subprocess
import sys

import numpy as np
import pytest
import torch

from __graft_entry__ import ROOT, load_package

pytestmark = pytest.mark.gpu

F = 2e-5
HALF_STEP = {"bf16": 2.0 ** -8, "f16": 2.0 ** -11, "f32": 2.0 ** -24}
TORCH = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
SENTINEL = 0x3A5C


@pytest.fixture(scope="module")
def pkg():
    return load_package()


@pytest.fixture()
def sess(pkg):
    s = pkg.Session(device=0)
    yield s
    s.close()


def _dt(pkg, kind):
    return {"bf16": pkg.blob.BF16, "f16": pkg.blob.F16, "f32": pkg.blob.F32}[kind]


def _bits(t):
    t = t.contiguous()
    return t.view(torch.int16 if t.element_size() == 2 else torch.int32).numpy()


def _rand(shape, kind, seed, std=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * std).to(TORCH[kind])


class Output:
    """A device buffer filled with a sentinel, with guard elements before and behind the result."""
    GUARD = 64

    def __init__(self, sess, n, kind):
        self.sess, self.n, self.kind = sess, n, kind
        self.np = np.uint32 if kind == "f32" else np.uint16
        self.base = sess.upload(np.full(n + 2 * self.GUARD, SENTINEL, self.np))
        self.ptr = self.base + self.GUARD * self.np().itemsize

    def get(self, shape):
        raw = self.sess.download(self.base, (self.n + 2 * self.GUARD,), self.np)
        assert (raw[:self.GUARD] == SENTINEL).all() and (raw[-self.GUARD:] == SENTINEL).all(), "written outside"
        body = raw[self.GUARD:-self.GUARD].copy()
        if self.kind == "f32":
            return torch.from_numpy(body.view(np.float32)).reshape(shape)
        return torch.from_numpy(body.view(np.int16)).view(TORCH[self.kind]).reshape(shape)


def _launch(sess, desc, args):
    kernel = sess.kernel(desc)
    need = sess.workspace_bytes(kernel)
    if need:  # whatever is in the workspace must not matter
        args = args + [sess.upload(np.full(need, 0xFF, np.uint8))]
    sess.launch(kernel, args)


# ------------------------------------------------------------------------------------------- attention
class Attention:
    """A problem, its inputs (as [batch, heads, rows, d]), the exact results and the kernels' ones."""

    def __init__(self, batch, q_heads, kv_heads, n_q, n_kv, d, kind="bf16", causal=False, lens=None, layout="heads",
                 scale=None, seed=1, std=1.0):
        self.dims = (batch, q_heads, kv_heads, n_q, n_kv, d)
        self.kind, self.causal, self.lens, self.layout = kind, causal, lens, layout
        self.scale = d ** -0.5 if scale is None else scale
        self.q, self.do = (_rand((batch, q_heads, n_q, d), kind, seed + i, std if i == 0 else 1.0) for i in (0, 3))
        self.k, self.v = (_rand((batch, kv_heads, n_kv, d), kind, seed + i) for i in (1, 2))

    def poison_padding(self):
        for b, n in enumerate(self.lens):
            self.k[b, :, n:] = float("nan")
            self.v[b, :, n:] = float("inf")

    def exact(self):
        batch, q_heads, kv_heads, n_q, n_kv, d = self.dims
        g = q_heads // kv_heads
        q, do = self.q.double(), self.do.double()
        k, v = (t.double().clone() for t in (self.k, self.v))
        for b, n in enumerate(self.lens or []):
            k[b, :, n:] = 0
            v[b, :, n:] = 0
        k, v = (t.repeat_interleave(g, 1) for t in (k, v))
        s = (q @ k.transpose(2, 3)) * self.scale
        j = torch.arange(n_kv)
        seen = torch.ones((batch, 1, n_q, n_kv), dtype=torch.bool)
        if self.causal:
            seen &= (j[None] <= torch.arange(n_q)[:, None] + (n_kv - n_q))
        if self.lens is not None:
            seen &= (j[None] < torch.tensor(self.lens)[:, None])[:, None, None]
        s = s.masked_fill(~seen, -math.inf)
        lse = torch.logsumexp(s, 3)
        p = torch.exp(s - torch.where(lse == -math.inf, torch.zeros_like(lse), lse)[..., None])
        o = p @ v
        dp = do @ v.transpose(2, 3)
        ds = p * (dp - (do * o).sum(3, keepdim=True))
        per = (batch, kv_heads, g, n_kv, d)
        grads = {"dq": ds @ k * self.scale, "dk": (ds.transpose(2, 3) @ q * self.scale).view(per).sum(2),
                 "dv": (p.transpose(2, 3) @ do).view(per).sum(2)}
        u, tiny = HALF_STEP[self.kind], 2.0 ** -25 if self.kind == "f16" else 0.0
        pt = tiny * seen
        e = (u + F) * ds.abs() + p * ((u + F) * (do.abs() * o.abs()).sum(3, keepdim=True) + F * (do.abs() @ v.abs().transpose(2, 3))) + pt
        tol = {"o": ((u + F) * p + pt) @ v.abs() + (u + F) * o.abs() + 2.0 ** -25,
               "dq": e @ k.abs() * self.scale + (u + F) * grads["dq"].abs() + 2.0 ** -25,
               "dk": (e.transpose(2, 3) @ q.abs() * self.scale).view(per).sum(2) + (u + F) * grads["dk"].abs() + 2.0 ** -25,
               "dv": (((u + F) * p + pt).transpose(2, 3) @ do.abs()).view(per).sum(2) + (u + F) * grads["dv"].abs() + 2.0 ** -25}
        return {"o": o, "lse": lse, **grads}, tol

    def laid(self, t):
        return t if self.layout == "heads" else t.transpose(1, 2).contiguous()

    def back(self, t, shape):
        b, h, n, d = shape
        return t.reshape(b, h, n, d) if self.layout == "heads" else t.reshape(b, n, h, d).transpose(1, 2)

    def run(self, pkg, sess, backward=True, **more):
        batch, q_heads, kv_heads, n_q, n_kv, d = self.dims
        B = pkg.blob
        kw = dict(dtype=_dt(pkg, self.kind), sm_scale=self.scale, causal=self.causal, key_lens=self.lens is not None,
                  layout=self.layout, **more)
        dq, dk, dv = (sess.upload(_bits(self.laid(t))) for t in (self.q, self.k, self.v))
        lens = [sess.upload(np.array(self.lens, np.int32))] if self.lens is not None else []
        o, lse = Output(sess, self.q.numel(), self.kind), Output(sess, batch * q_heads * n_q, "f32")
        _launch(sess, B.attention("attn", *self.dims, **kw), [dq, dk, dv, o.ptr, lse.ptr] + lens)
        got = {"o": self.back(o.get(-1), self.q.shape), "lse": lse.get((batch, q_heads, n_q))}
        if backward:
            ddo = sess.upload(_bits(self.laid(self.do)))
            outs = {n: Output(sess, t.numel(), self.kind) for n, t in (("dq", self.q), ("dk", self.k), ("dv", self.v))}
            _launch(sess, B.attention_bwd("attn_bwd", *self.dims, **kw),
                    [dq, dk, dv, o.ptr, ddo, lse.ptr] + [x.ptr for x in outs.values()] + lens)
            for n, x in outs.items():
                got[n] = self.back(x.get(-1), (self.q if n == "dq" else self.k).shape)
        return got

    def check(self, got):
        ref, tol = self.exact()
        lse, want = got.pop("lse").double(), ref.pop("lse")
        assert torch.equal(lse == -math.inf, want == -math.inf)
        seen = want > -math.inf
        assert (lse - want)[seen].abs().le(2e-5 + 1e-6 * want[seen].abs()).all()
        for n, t in got.items():
            assert torch.isfinite(t).all(), n
            off = (t.double() - ref[n]).abs() / tol[n]
            assert off.max() <= 1.0, "%s: %.3g of the tolerance at %s" % (n, off.max(), np.unravel_index(int(off.argmax()), off.shape))


ATTENTION = [
    # batch, q_heads, kv_heads, n_q, n_kv, d, kind, causal, lens, layout
    (1, 1, 1, 1, 1, 64, "f16", False, None, "heads"),
    (1, 1, 1, 1, 1, 128, "bf16", True, None, "tokens"),
    (2, 3, 1, 5, 7, 64, "bf16", False, None, "tokens"),
    (1, 2, 2, 128, 128, 128, "bf16", True, None, "heads"),
    (1, 2, 2, 128, 128, 64, "f16", False, None, "heads"),
    (1, 2, 1, 129, 257, 64, "bf16", True, None, "tokens"),
    (2, 4, 2, 200, 200, 128, "f16", True, None, "tokens"),
    (3, 2, 2, 65, 300, 64, "f16", False, [0, 300, 131], "heads"),
    (3, 4, 1, 97, 97, 128, "bf16", True, [97, 1, 0], "tokens"),
    (1, 2, 1, 300, 20, 64, "bf16", True, None, "heads"),      # the first 280 rows see no key
    (2, 2, 2, 257, 130, 128, "f16", True, [130, 64], "heads"),
    (2, 8, 1, 1, 1000, 128, "bf16", False, [1000, 333], "heads"),
    (2, 8, 2, 3, 515, 64, "f16", True, None, "tokens"),
    (1, 6, 2, 40, 600, 64, "bf16", True, None, "tokens"),
    (1, 1, 1, 640, 640, 64, "f16", True, None, "heads"),
    (1, 3, 1, 385, 513, 128, "bf16", False, None, "tokens"),
]


@pytest.mark.parametrize("case", ATTENTION, ids=lambda c: "-".join(str(x) for x in c).replace(" ", ""))
def test_attention_and_its_gradients(pkg, sess, case):
    a = Attention(*case)
    a.check(a.run(pkg, sess))


@pytest.mark.parametrize("d,n_q,n_kv", [(64, 140, 140), (128, 130, 300), (64, 1, 200)])
def test_attention_padding_may_hold_anything(pkg, sess, d, n_q, n_kv):
    a = Attention(4, 4, 2, n_q, n_kv, d, "bf16", lens=[n_kv, 1, 0, n_kv - 7])
    a.poison_padding()
    a.check(a.run(pkg, sess))


def test_attention_lengths_out_of_range_are_clamped(pkg, sess):
    a = Attention(2, 1, 1, 30, 40, 64, "f16", lens=[-5, 1000])
    got = a.run(pkg, sess)
    a.lens = [0, 40]
    a.check(got)


@pytest.mark.parametrize("std,scale", [(30.0, None), (1.0, 2.0), (1e-3, 0.01)])
def test_attention_with_sharp_and_flat_rows(pkg, sess, std, scale):
    """Scores of some hundreds: every row has its maximum at a key of its own.  |S| is up to 600, so the f32 rounding
    of a score alone moves P by 600 * 2^-22: the 32-bit share of the tolerance grows with it."""
    a = Attention(1, 2, 1, 150, 400, 64, "bf16", scale=scale, std=std)
    global F
    keep, F = F, 3e-4
    try:
        got = a.run(pkg, sess)
        got["lse"] = got["lse"].double()
        ref, _ = a.exact()
        assert (got["lse"] - ref["lse"]).abs().max() <= 1e-6 * ref["lse"].abs().max() + 2e-5
        got["lse"] = ref["lse"]
        a.check(got)
    finally:
        F = keep


def test_attention_row_maxima_that_keep_growing(pkg, sess):
    """Keys in the order of their scores: the running maximum moves in every tile."""
    a = Attention(1, 1, 1, 64, 1024, 64, "bf16", scale=1.0)
    a.q = torch.ones_like(a.q) * 0.5
    a.k = (torch.arange(1024.0) / 128).floor().mul(0.5)[None, None, :, None].expand(1, 1, 1024, 64).to(torch.bfloat16).contiguous()
    a.check(a.run(pkg, sess))


def test_attention_inside_a_packed_projection(pkg, sess):
    """Q, K and V as slices of one [tokens, heads + 2 kv_heads, d] array, and their gradients into another one."""
    n, hq, hkv, d = 150, 4, 2, 64
    a = Attention(1, hq, hkv, n, n, d, "bf16", causal=True)
    B, width = pkg.blob, hq + 2 * hkv
    packed = torch.cat([t[0].transpose(0, 1) for t in (a.q, a.k, a.v)], 1).contiguous()
    base = sess.upload(_bits(packed))
    row = width * d
    at = {"q": 0, "k": hq * d, "v": (hq + hkv) * d}
    inside = (n * row, d, row)
    strides = {x: inside for x in ("q", "k", "v", "dq", "dk", "dv")}
    o, lse = Output(sess, n * hq * d, "bf16"), Output(sess, hq * n, "f32")
    dims = (1, hq, hkv, n, n, d)
    ptrs = [base + 2 * at[x] for x in ("q", "k", "v")]
    _launch(sess, B.attention("p", *dims, causal=True, layout="tokens", strides={x: inside for x in ("q", "k", "v")}),
            ptrs + [o.ptr, lse.ptr])
    grads = Output(sess, n * row, "bf16")
    ddo = sess.upload(_bits(a.do[0].transpose(0, 1)))
    _launch(sess, B.attention_bwd("pb", *dims, causal=True, layout="tokens", strides=strides),
            ptrs + [o.ptr, ddo, lse.ptr] + [grads.ptr + 2 * at[x] for x in ("q", "k", "v")])
    g = grads.get((n, width, d)).transpose(0, 1)[None]
    a.check({"o": o.get((1, n, hq, d)).transpose(1, 2), "lse": lse.get((1, hq, n)), "dq": g[:, :hq],
             "dk": g[:, hq:hq + hkv], "dv": g[:, hq + hkv:]})


def test_attention_gaps_between_rows_stay_untouched(pkg, sess):
    n, d, row = 70, 64, 96
    a = Attention(1, 1, 1, n, n, d, "f16")
    s = {x: (0, 0, row) for x in ("o", "dq", "dk", "dv")}
    B = pkg.blob
    ins = [sess.upload(_bits(t)) for t in (a.q, a.k, a.v)]
    o, lse = Output(sess, n * row, "f16"), Output(sess, n, "f32")
    _launch(sess, B.attention("g", *a.dims, dtype=B.F16, strides={"o": s["o"]}), ins + [o.ptr, lse.ptr])
    outs = [Output(sess, n * row, "f16") for _ in range(3)]
    _launch(sess, B.attention_bwd("gb", *a.dims, dtype=B.F16, strides=s),
            ins + [o.ptr, sess.upload(_bits(a.do)), lse.ptr] + [x.ptr for x in outs])
    got = {}
    for name, x in zip(("o", "dq", "dk", "dv"), [o] + outs):
        t = x.get((n, row))
        assert (t[:, d:].contiguous().view(torch.int16) == SENTINEL).all(), name
        got[name] = t[:, :d][None, None]
    got["lse"] = lse.get((1, 1, n))
    a.check(got)


def test_attention_gradients_against_differences(pkg, sess):
    """The loss sum(dO * O) in 64 bits, moved along a direction, against the kernels' gradients along it: dQ, dK and
    dV are held to the tolerance of each element times the direction's."""
    a = Attention(1, 2, 1, 33, 50, 64, "f16", causal=True)
    got, (_, tol) = a.run(pkg, sess), a.exact()
    for n, src in (("dq", "q"), ("dk", "k"), ("dv", "v")):
        x = getattr(a, src)
        step = torch.randn(x.shape, generator=torch.Generator().manual_seed(9)).double()
        loss = []
        for h in (1e-4, -1e-4):
            setattr(a, src, x.double() + h * step)
            loss.append((a.exact()[0]["o"] * a.do.double()).sum())
        setattr(a, src, x)
        want = (loss[0] - loss[1]) / 2e-4
        assert abs((got[n].double() * step).sum() - want) <= (tol[n] * step.abs()).sum() + 1e-6 * abs(want)


def test_attention_runs_give_the_same_bits(pkg, sess):
    a = Attention(2, 8, 2, 333, 333, 128, "bf16", causal=True, layout="tokens")
    first = a.run(pkg, sess)
    for _ in range(3):
        again = a.run(pkg, sess)
        for n in first:
            assert torch.equal(first[n].contiguous().view(torch.int16), again[n].contiguous().view(torch.int16)), n


@pytest.mark.parametrize("d,kind", [(64, "f16"), (128, "bf16")])
def test_attention_gradients_with_warps_out_of_step(pkg, d, kind):
    """Many CTAs, short and long ones beside each other, every launch behind other work that leaves the caches cold:
    the gradients of the first and of later launches are the same bits, none of them NaN."""
    torch.manual_seed(3)
    dims = (4, 16, 16, 1000, 1000, d)
    new = lambda: torch.randn((4, 1000, 16, d), device="cuda").to(TORCH[kind])  # noqa: E731
    with pkg.Session(device=0, adopt_stream=1) as sess:
        B = pkg.blob
        q, k, v, do, o = new(), new(), new(), new(), torch.empty((4, 1000, 16, d), dtype=TORCH[kind], device="cuda")
        lse, lens = torch.empty((4, 16, 1000), device="cuda"), torch.tensor([0, 1000, 777, 850], dtype=torch.int32, device="cuda")
        kw = dict(dtype=_dt(pkg, kind), key_lens=True, layout="tokens")
        grads = [torch.empty_like(q) for _ in range(3)]

        def bind(desc, args):
            kernel = sess.kernel(desc)
            need = sess.workspace_bytes(kernel)
            if need:
                args = args + [torch.empty(need, dtype=torch.uint8, device="cuda")]
            return sess.bind(kernel, [t.data_ptr() for t in args]), args
        forward, keep = bind(B.attention("a", *dims, **kw), [q, k, v, o, lse, lens])
        backward, keep2 = bind(B.attention_bwd("b", *dims, **kw), [q, k, v, o, do, lse] + grads + [lens])
        forward()
        first, spoil = None, torch.empty(64 << 20, device="cuda")
        for _ in range(25):
            spoil.fill_(1.0)
            for g in grads:
                g.fill_(float("nan"))
            backward()
            got = [g.clone() for g in grads]
            assert all(torch.isfinite(g).all() for g in got)
            first = first or got
            assert all(torch.equal(a.view(torch.int16), b.view(torch.int16)) for a, b in zip(first, got))


@pytest.mark.parametrize("op,arg,by,message", [
    ("attention", 0, 8, "16-byte aligned"), ("attention", 3, 8, "16-byte aligned"), ("attention", 4, 2, "multiple of 4 bytes"),
    ("attention_bwd", 7, 8, "16-byte aligned"), ("attention_bwd", 5, 2, "multiple of 4 bytes"),
    ("attention_bwd", -1, 8, "the workspace must be")])
def test_misaligned_arrays_are_refused(op, arg, by, message):
    """Before anything is launched, by the error convention: one line on stdout, then abort()."""
    text = ("from __graft_entry__ import load_package\npkg = load_package()\nB = pkg.blob\ns = pkg.Session(device=0)\n"
            "k = s.kernel(B.%s('a', 1, 1, 1, 8, 8, 64))\nn = %d\np = [s.alloc(4096) for _ in range(n)]\n"
            "p[%d] += %d\ns.launch(k, p)\n" % (op, 5 if op == "attention" else 10, arg, by))
    r = subprocess.run([sys.executable, "-c", text], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert r.returncode == -6 and message in r.stdout, r.stdout + r.stderr


# --------------------------------------------------------------------------------------- gated product
def _act(g, act):
    return {0: g, 1: g.clamp(min=0), 2: torch.nn.functional.silu(g)}[act]


GATED = [
    # tokens, d_in, d_ff, kind, act
    (1, 8, 8, "f16", 2), (1, 1, 1, "bf16", 2), (3, 5, 7, "f16", 2), (1, 1024, 704, "bf16", 2), (2, 512, 136, "f16", 1),
    (16, 264, 1000, "bf16", 2), (17, 256, 256, "f16", 0), (33, 200, 128, "bf16", 2), (64, 1000, 360, "f16", 2),
    (65, 128, 72, "bf16", 1), (127, 64, 8, "f16", 2), (128, 136, 264, "bf16", 2), (129, 520, 392, "f16", 2),
    (300, 1000, 104, "bf16", 2), (513, 72, 513, "bf16", 2), (700, 256, 384, "f16", 2), (40, 33, 65, "bf16", 0),
    (513, 2600, 200, "bf16", 2), (200, 5201, 70, "f16", 2), (520, 96, 1704, "bf16", 2), (1300, 41, 801, "f16", 1), (520, 2049, 1701, "f16", 2),
]


@pytest.mark.parametrize("case", GATED, ids=lambda c: "-".join(str(x) for x in c))
@pytest.mark.parametrize("save", [False, True], ids=["", "kept"])
def test_gated_ffn(pkg, sess, case, save):
    m, d, f, kind, act = case
    x, w = _rand((m, d), kind, 1), _rand((d, 2 * f), kind, 2, d ** -0.5)
    h, gu = Output(sess, m * f, kind), Output(sess, m * 2 * f, kind)
    args = [sess.upload(_bits(x)), sess.upload(_bits(w)), h.ptr] + ([gu.ptr] if save else [])
    _launch(sess, pkg.blob.gated_ffn("g", m, d, f, _dt(pkg, kind), act, save_gu=save), args)
    z, size = x.double() @ w.double(), x.double().abs() @ w.double().abs()
    g, up = z[:, :f], z[:, f:]
    u = HALF_STEP[kind]
    acc = 2.0 ** -24 * (d + 8) * size + 2.0 ** -25   # any order of d additions, each product exact
    a = _act(g, act)
    want = a * up
    # |silu'| <= 1.1; the fast exponential and division of silu keep 4e-6
    tol = 1.1 * acc[:, :f] * (up.abs() + acc[:, f:]) + a.abs() * acc[:, f:] + (u + 4e-6) * want.abs() + 2.0 ** -25
    assert ((h.get((m, f)).double() - want).abs() <= tol * 1.01).all()
    if save:
        assert ((gu.get((m, 2 * f)).double() - z).abs() <= (acc + u * z.abs()) * 1.01).all()
    else:
        assert (gu.get(-1).view(torch.int16) == SENTINEL).all()


@pytest.mark.parametrize("case", GATED, ids=lambda c: "-".join(str(x) for x in c))
def test_gated_ffn_gradients(pkg, sess, case):
    m, d, f, kind, act = case
    x, w = _rand((m, d), kind, 1), _rand((d, 2 * f), kind, 2, d ** -0.5)
    gu, dh = (x.float() @ w.float()).to(TORCH[kind]), _rand((m, f), kind, 3)
    dx, dw = Output(sess, m * d, kind), Output(sess, d * 2 * f, kind)
    _launch(sess, pkg.blob.gated_ffn_bwd("gb", m, d, f, _dt(pkg, kind), act),
            [sess.upload(_bits(t)) for t in (x, w, gu, dh)] + [dx.ptr, dw.ptr])
    z = gu.double().requires_grad_(True)
    dz, = torch.autograd.grad(_act(z[:, :f], act) * z[:, f:], z, dh.double())
    u, tiny = HALF_STEP[kind], 2.0 ** -25
    # [dG dU] is rounded once to 16 bits (and computed to 1e-5), the sums once more
    e = (u + 1e-5) * dz.abs() + tiny
    for got, want, size, terms in ((dx.get((m, d)), dz @ w.double().t(), e @ w.double().abs().t(), dz.abs() @ w.double().abs().t()),
                                   (dw.get((d, 2 * f)), x.double().t() @ dz, x.double().abs().t() @ e, x.double().abs().t() @ dz.abs())):
        tol = size + u * want.abs() + 2.0 ** -24 * (max(m, 2 * f) + 8) * terms + tiny
        assert ((got.double() - want).abs() <= tol * 1.01).all()


@pytest.mark.parametrize("m,d,f,ldx,ldw,ldh", [(1, 128, 136, 160, 304, 144), (20, 128, 136, 160, 304, 144),
                                               (200, 128, 136, 160, 304, 144), (2100, 128, 640, 136, 1288, 648),
                                               (20, 128, 136, 131, 275, 137), (200, 99, 135, 131, 272, 144),
                                               (2100, 64, 601, 65, 1210, 603), (520, 2056, 1704, 2057, 3409, 1705)])
def test_gated_ffn_row_pitches(pkg, sess, m, d, f, ldx, ldw, ldh):
    x, w = _rand((m, ldx), "bf16", 1), _rand((d, ldw), "bf16", 2, d ** -0.5)
    h = Output(sess, m * ldh, "bf16")
    _launch(sess, pkg.blob.gated_ffn("g", m, d, f, pkg.blob.BF16, ldx=ldx, ldw=ldw, ldh=ldh),
            [sess.upload(_bits(x)), sess.upload(_bits(w)), h.ptr])
    z = x[:, :d].double() @ w[:, :2 * f].double()
    got = h.get((m, ldh))
    assert (got[:, f:].contiguous().view(torch.int16) == SENTINEL).all()
    want = torch.nn.functional.silu(z[:, :f]) * z[:, f:]
    assert ((got[:, :f].double() - want).abs() <= 2.0 ** -8 * want.abs() + 1e-4).all()
    gu, dh = z.to(torch.bfloat16), _rand((m, ldh), "bf16", 3)
    dx, dw = Output(sess, m * ldx, "bf16"), Output(sess, d * ldw, "bf16")
    _launch(sess, pkg.blob.gated_ffn_bwd("gb", m, d, f, pkg.blob.BF16, ldx=ldx, ldw=ldw, ldh=ldh),
            [sess.upload(_bits(t)) for t in (x, w, gu, dh)] + [dx.ptr, dw.ptr])
    zz = gu.double().requires_grad_(True)
    dz, = torch.autograd.grad(torch.nn.functional.silu(zz[:, :f]) * zz[:, f:], zz, dh[:, :f].double())
    for out, width, held, want, size in ((dx, d, ldx, dz @ w[:, :2 * f].double().t(), dz.abs() @ w[:, :2 * f].double().abs().t()),
                                         (dw, 2 * f, ldw, x[:, :d].double().t() @ dz, x[:, :d].double().abs().t() @ dz.abs())):
        t = out.get((-1, held))
        assert (t[:, width:].contiguous().view(torch.int16) == SENTINEL).all()
        assert ((t[:, :width].double() - want).abs() <= 1.01 * 2.0 ** -8 * (want.abs() + size) + 1e-5).all()


@pytest.mark.parametrize("m", [5, 200])
def test_gated_ffn_odd_extents_take_arrays_at_any_element(pkg, sess, m):
    d, f = 33, 69
    x, w = _rand((m, d), "f16", 1), _rand((d, 2 * f), "f16", 2, d ** -0.5)
    gu, dh = (x.float() @ w.float()).half(), _rand((m, f), "f16", 3)
    runs = []
    for lead in (0, 1, 3):
        up = lambda t: sess.upload(_bits(torch.cat([torch.zeros(lead, dtype=t.dtype), t.flatten()]))) + 2 * lead
        outs = [Output(sess, n + lead, "f16") for n in (m * f, m * 2 * f, m * d, d * 2 * f)]
        at = [o.ptr + 2 * lead for o in outs]
        _launch(sess, pkg.blob.gated_ffn("g", m, d, f, pkg.blob.F16, save_gu=True), [up(x), up(w), at[0], at[1]])
        _launch(sess, pkg.blob.gated_ffn_bwd("b", m, d, f, pkg.blob.F16), [up(x), up(w), up(gu), up(dh), at[2], at[3]])
        runs.append([o.get(-1)[lead:] for o in outs])
        assert all(o.get(-1)[:lead].view(torch.int16).eq(SENTINEL).all() for o in outs)
    assert all(torch.isfinite(a).all() and torch.equal(a, b) for r in runs[1:] for a, b in zip(runs[0], r))


@pytest.mark.parametrize("op,d,arg,message", [("gated_ffn", 16, 1, "arrays must be 16-byte"), ("gated_ffn", 15, -1, "the workspace must be"),
                                              ("gated_ffn_bwd", 16, 5, "arrays must be 16-byte"), ("gated_ffn_bwd", 16, -1, "the workspace must be")])
def test_misaligned_gated_arrays_are_refused(op, d, arg, message):
    text = ("from __graft_entry__ import load_package\npkg = load_package()\nB = pkg.blob\ns = pkg.Session(device=0)\n"
            "k = s.kernel(B.%s('a', 2, %d, 8))\nn = %d\np = [s.alloc(4096) for _ in range(n)]\n"
            "p[%d] += 8\ns.launch(k, p)\n" % (op, d, 7 if op.endswith("bwd") else 3 + d % 2, arg))
    r = subprocess.run([sys.executable, "-c", text], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert r.returncode == -6 and message in r.stdout, r.stdout + r.stderr


# ------------------------------------------------------------------------------------------- rotary
def _rotate(x, positions, freqs, interleaved, inverse, factor):
    n = len(freqs)
    t = positions.double()[:, None] * torch.tensor(freqs, dtype=torch.float64)[None] * (-1 if inverse else 1)
    c, s = t.cos()[:, None], t.sin()[:, None]
    y = x.double().clone()
    a, b = ((x[..., 0:2 * n:2], x[..., 1:2 * n:2]) if interleaved else (x[..., :n], x[..., n:2 * n]))
    a, b = a.double(), b.double()
    if interleaved:
        y[..., 0:2 * n:2], y[..., 1:2 * n:2] = (a * c - b * s) * factor, (a * s + b * c) * factor
    else:
        y[..., :n], y[..., n:2 * n] = (a * c - b * s) * factor, (a * s + b * c) * factor
    return y


def _rotary_tolerance(x, want, n, kind, interleaved, factor):
    size = torch.zeros_like(want)
    if interleaved:
        pair = x[..., 0:2 * n:2].double().abs() + x[..., 1:2 * n:2].double().abs()
        size[..., 0:2 * n:2], size[..., 1:2 * n:2] = pair, pair
    else:
        pair = x[..., :n].double().abs() + x[..., n:2 * n].double().abs()
        size[..., :n], size[..., n:2 * n] = pair, pair
    # the reduced angle is off by 1e-7, sine and cosine by 1.2e-7, two products and a sum by 2^-24 each
    return HALF_STEP[kind] * want.abs() + 5e-7 * factor * size + (2.0 ** -25 if kind == "f16" else 0.0)


@pytest.mark.parametrize("interleaved", [False, True], ids=["halves", "interleaved"])
@pytest.mark.parametrize("inverse", [False, True], ids=["", "inverse"])
@pytest.mark.parametrize("case", [(1, 1, 2, 2, "f32"), (7, 3, 64, 64, "bf16"), (300, 2, 128, 64, "f16"), (5, 40, 80, 20, "bf16"),
                                  (33, 5, 96, 24, "f32"), (2, 9, 256, 256, "f16"), (600, 1, 66, 6, "bf16"),
                                  (3, 2, 511, 18, "f16"), (2000, 3, 16, 8, "f32"), (40, 7, 512, 256, "bf16")],
                         ids=lambda c: "-".join(str(x) for x in c))
def test_rotary(pkg, sess, case, interleaved, inverse):
    tokens, heads, d, rot, kind = case
    B = pkg.blob
    freqs = B.rotary_frequencies(rot, factor=4.0, original_length=4096)
    x = _rand((tokens, heads, d), kind, 5)
    pos = torch.randint(0, 2 ** 31 - 1 if tokens == 7 else 1000000, (tokens,), generator=torch.Generator().manual_seed(6), dtype=torch.int32)
    if tokens > 2:
        pos[0], pos[1] = 0, -3
    y = Output(sess, x.numel(), kind)
    dx, dp = sess.upload(_bits(x)), sess.upload(pos.numpy())
    desc = B.rotary("r", tokens, heads, d, freqs, _dt(pkg, kind), interleaved, inverse, factor=1.25)
    _launch(sess, desc, [dx, dp, y.ptr])
    got = y.get((tokens, heads, d))
    want = _rotate(x, pos, freqs, interleaved, inverse, 1.25)
    assert ((got.double() - want).abs() <= _rotary_tolerance(x, want, rot // 2, kind, interleaved, 1.25)).all()
    assert torch.equal(got[..., rot:], x[..., rot:])
    _launch(sess, desc, [dx, dp, dx])   # in place: the same bits
    back = sess.download(dx, tuple(x.shape), np.uint32 if kind == "f32" else np.uint16)
    assert np.array_equal(back.view(np.int32 if kind == "f32" else np.int16), _bits(got))


@pytest.mark.parametrize("interleaved", [False, True], ids=["halves", "interleaved"])
@pytest.mark.parametrize("step", [1, 2, 8])
def test_rotary_strides_and_alignment(pkg, sess, step, interleaved):
    """Heads inside a wider row, starting on any element."""
    tokens, heads, d, held = 20, 3, 64, 3 * 72 + step
    x = _rand((tokens * held + 16,), "f16", 8)
    pos = torch.arange(tokens, dtype=torch.int32)
    y = Output(sess, tokens * held, "f16")
    freqs = pkg.blob.rotary_frequencies(32)
    _launch(sess, pkg.blob.rotary("r", tokens, heads, d, freqs, pkg.blob.F16, interleaved, x_strides=(held, 72), y_strides=(held, 72)),
            [sess.upload(_bits(x)) + 2 * step, sess.upload(pos.numpy()), y.ptr])
    xs = x[step:step + tokens * held].reshape(tokens, held)[:, :3 * 72].reshape(tokens, 3, 72)[..., :d]
    got = y.get((tokens, held))
    assert (got[:, 3 * 72:].contiguous().view(torch.int16) == SENTINEL).all()
    got = got[:, :3 * 72].reshape(tokens, 3, 72)
    assert (got[..., d:].contiguous().view(torch.int16) == SENTINEL).all()
    want = _rotate(xs, pos, freqs, interleaved, False, 1.0)
    assert ((got[..., :d].double() - want).abs() <= _rotary_tolerance(xs, want, 16, "f16", interleaved, 1.0)).all()


# ------------------------------------------------------------------------------------- a block of them
def test_a_block_forward_and_backward(pkg, sess):
    """Rotated queries and keys of a packed projection -> causal attention -> gated product, and back: the gradients
    of the packed projection and of the feed-forward weights against autograd in 64 bits of the same chain.  Every
    hand-over rounds to bf16 (half a step 2^-8 each, six of them one after the other on the longest way), so results
    are compared in the 2-norm: 6 * 2^-8 / sqrt(3) (the mean square of a rounding) is 1.4e-2; 2e-2 is allowed."""
    n, hq, hkv, d, f = 260, 4, 2, 64, 200
    B, width, dm = pkg.blob, hq + 2 * hkv, hq * d
    qkv, w = _rand((n, width, d), "bf16", 1), _rand((dm, 2 * f), "bf16", 2, dm ** -0.5)
    dh = _rand((n, f), "bf16", 3)
    freqs = B.rotary_frequencies(d)
    pos = torch.arange(n, dtype=torch.int32)
    base, dpos = sess.upload(_bits(qkv)), sess.upload(pos.numpy())
    row = width * d
    at = [0, 2 * hq * d, 2 * (hq + hkv) * d]
    inside = {x: (n * row, d, row) for x in ("q", "k", "v")}
    turned = ("r", n, hq + hkv, d, freqs)
    _launch(sess, B.rotary(*turned, x_strides=(row, d), y_strides=(row, d)), [base, dpos, base])
    dims = (1, hq, hkv, n, n, d)
    o, lse = Output(sess, n * dm, "bf16"), Output(sess, hq * n, "f32")
    _launch(sess, B.attention("a", *dims, causal=True, layout="tokens", strides=inside), [base + x for x in at] + [o.ptr, lse.ptr])
    h, gu = Output(sess, n * f, "bf16"), Output(sess, n * 2 * f, "bf16")
    dw_in = sess.upload(_bits(w))
    _launch(sess, B.gated_ffn("g", n, dm, f, save_gu=True), [o.ptr, dw_in, h.ptr, gu.ptr])
    do, dw = Output(sess, n * dm, "bf16"), Output(sess, dm * 2 * f, "bf16")
    _launch(sess, B.gated_ffn_bwd("gb", n, dm, f), [o.ptr, dw_in, gu.ptr, sess.upload(_bits(dh)), do.ptr, dw.ptr])
    grads = Output(sess, n * row, "bf16")
    more = dict(inside, **{"d" + x: inside[x] for x in inside})
    _launch(sess, B.attention_bwd("ab", *dims, causal=True, layout="tokens", strides=more),
            [base + x for x in at] + [o.ptr, do.ptr, lse.ptr] + [grads.ptr + x for x in at])
    _launch(sess, B.rotary(*turned, inverse=True, x_strides=(row, d), y_strides=(row, d)), [grads.ptr, dpos, grads.ptr])

    x, wt = qkv.double().requires_grad_(True), w.double().requires_grad_(True)
    t = pos.double()[:, None] * torch.tensor(freqs, dtype=torch.float64)[None]
    z = torch.polar(torch.ones_like(t), t)[:, None]
    qk = torch.complex(x[:, :hq + hkv, :d // 2], x[:, :hq + hkv, d // 2:]) * z
    qk = torch.cat([qk.real, qk.imag], -1).transpose(0, 1)
    k, v = (y.repeat_interleave(hq // hkv, 0) for y in (qk[hq:], x[:, hq + hkv:].transpose(0, 1)))
    s = qk[:hq] @ k.transpose(1, 2) * d ** -0.5
    s = s.masked_fill(torch.ones(n, n, dtype=torch.bool).triu(1), -math.inf)
    attn = (s.softmax(2) @ v).transpose(0, 1).reshape(n, dm)
    y = attn @ wt
    out = torch.nn.functional.silu(y[:, :f]) * y[:, f:]
    gx, gw = torch.autograd.grad(out, (x, wt), dh.double())
    for name, got, want in (("h", h.get((n, f)), out), ("dw", dw.get((dm, 2 * f)), gw), ("dqkv", grads.get((n, width, d)), gx)):
        off = ((got.double() - want).norm() / want.norm()).item()
        assert off <= 2e-2, (name, off)


def test_captured_block_replays_on_new_inputs(pkg):
    """The launches captured into a CUDA graph and replayed give the bits of direct launches, on inputs that changed."""
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream), pkg.Session(device=0, adopt_stream=stream.cuda_stream) as sess:
        B, dims = pkg.blob, (2, 4, 2, 150, 150, 64)
        new = lambda *shape: torch.randn(shape, device="cuda").to(torch.bfloat16)  # noqa: E731
        q, do = new(2, 4, 150, 64), new(2, 4, 150, 64)
        k, v = new(2, 2, 150, 64), new(2, 2, 150, 64)
        lens = torch.tensor([150, 70], dtype=torch.int32, device="cuda")
        o, lse = torch.empty_like(q), torch.empty((2, 4, 150), device="cuda")
        dq, dk, dv = (torch.empty_like(t) for t in (q, k, v))
        x, w, dh = new(70, 64), new(64, 272), new(70, 136)
        h, gu, dx, dw = (torch.empty_like(t) for t in (dh, torch.empty(70, 272), x, w))
        gu = gu.cuda().to(torch.bfloat16)
        calls = [(B.attention("a", *dims, causal=True, key_lens=True), [q, k, v, o, lse, lens]),
                 (B.attention_bwd("b", *dims, causal=True, key_lens=True), [q, k, v, o, do, lse, dq, dk, dv, lens]),
                 (B.gated_ffn("g", 70, 64, 136, save_gu=True), [x, w, h, gu]),
                 (B.gated_ffn_bwd("gb", 70, 64, 136), [x, w, gu, dh, dx, dw])]
        # one query on a long cache (shares of the keys, joined), its gradients (shares in a cluster), few rows
        dims1 = (1, 4, 1, 1, 5000, 128)
        q1, do1, k1, v1 = new(1, 4, 1, 128), new(1, 4, 1, 128), new(1, 1, 5000, 128), new(1, 1, 5000, 128)
        o1, lse1, dq1, dk1, dv1 = torch.empty_like(q1), torch.empty((1, 4, 1), device="cuda"), torch.empty_like(q1), torch.empty_like(k1), torch.empty_like(k1)
        x1, w1, h1 = new(3, 1024), new(1024, 256), new(3, 128)
        calls += [(B.attention("a1", *dims1), [q1, k1, v1, o1, lse1]),
                  (B.attention_bwd("b1", *dims1), [q1, k1, v1, o1, do1, lse1, dq1, dk1, dv1]),
                  (B.gated_ffn("g1", 3, 1024, 128), [x1, w1, h1])]
        outs = [o, lse, dq, dk, dv, h, gu, dx, dw, o1, lse1, dq1, dk1, dv1, h1]
        launches, keep = [], []
        for desc, args in calls:
            kernel = sess.kernel(desc)
            need = sess.workspace_bytes(kernel)
            if need:
                args = args + [torch.empty(need, dtype=torch.uint8, device="cuda")]
            keep.append(args)
            launches.append(sess.bind(kernel, [t.data_ptr() for t in args]))
        for run in launches:
            run()
        stream.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            for run in launches:
                run()
        for t in (q, k, v, do, x, w, dh, q1, do1, k1, v1, x1, w1):
            t.copy_(new(*t.shape))
        lens.copy_(torch.tensor([0, 149], dtype=torch.int32))
        for run in launches:
            run()
        stream.synchronize()
        want = [t.clone() for t in outs]
        for t in outs:
            t.zero_()
        graph.replay()
        stream.synchronize()
        sess.wait()
        for a, b in zip(outs, want):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


def test_session_on_the_default_stream(pkg):
    """Handle 1 is the legacy default stream: launches are in order with torch's work on it."""
    with pkg.Session(device=0, adopt_stream=1) as sess:
        x = torch.randn(4096, 8, 64, device="cuda")
        pos = torch.arange(4096, dtype=torch.int32, device="cuda")
        y = torch.empty_like(x)
        freqs = pkg.blob.rotary_frequencies(64)
        run = sess.bind(sess.kernel(pkg.blob.rotary("r", 4096, 8, 64, freqs, pkg.blob.F32)), [x.data_ptr(), pos.data_ptr(), y.data_ptr()])
        for _ in range(5):
            x.mul_(1.5)
            run()
            y.add_(1.0)
        got = y.cpu()
        want = _rotate(x.cpu(), pos.cpu(), freqs, False, False, 1.0) + 1.0
        assert (got.double() - want).abs().max() <= 1e-5 * want.abs().max()
