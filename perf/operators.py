"""Cases of the transformer-block operators: attention forward with its row statistics, attention backward, the gated
feed-forward product (forward and backward) and rotary positions.

`run` computes a case either in elementary torch operations in 32 bits (own = False) or through the framework's kernels
(own = True: the blob builders, a kernel handle per case and a bound launch, as a program that repeats a step keeps them).

Conventions shared by both:
  attention   key j is visible to query i of batch b when j < key_lens[b] (all keys without lengths) and, when causal,
              j <= i + n_kv - n_q.  A row that sees no key has O = 0, LSE = -inf and gradients 0.
  gated       W is [d_in, 2 * d_ff]: the gate's columns, then the up projection's.  H = silu(X Wg) * (X Wu).
  rotary      pair (a, b) at angle t = position * frequency -> (a cos t - b sin t, a sin t + b cos t) * scale.
"""
import math

import torch

own = False

_TYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}


# ---------------------------------------------------------------------------------------------- cases
def _attention(kind, batch, q_heads, kv_heads, n_q, n_kv, d_head, dtype, causal, lens, layout):
    return {"op": kind, "batch": batch, "q_heads": q_heads, "kv_heads": kv_heads, "n_q": n_q, "n_kv": n_kv,
            "d_head": d_head, "dtype": dtype, "causal": causal, "lens": lens, "layout": layout}


def _gated(kind, tokens, d_in, d_ff, dtype, save):
    return {"op": kind, "tokens": tokens, "d_in": d_in, "d_ff": d_ff, "dtype": dtype, "save": save}


def _rotary(tokens, heads, held, d_head, rot, dtype, interleaved, inverse, far, factor):
    return {"op": "rotary", "tokens": tokens, "heads": heads, "held": held, "d_head": d_head, "rot": rot,
            "dtype": dtype, "interleaved": interleaved, "inverse": inverse, "far": far, "factor": factor}


def listed():
    return [
        # one long sequence of a training or prompt pass, four query heads to a key head
        dict(_attention("attention", 1, 32, 8, 8192, 8192, 128, "bf16", True, False, "tokens"), name="attention_long_causal"),
        # a padded batch of an encoder, odd length, one sequence of it empty
        dict(_attention("attention", 8, 12, 12, 500, 500, 64, "f16", False, True, "heads"), name="attention_padded"),
        # one new token for each of sixteen sequences against their caches, a free slot among them
        dict(_attention("attention", 16, 32, 8, 1, 8000, 128, "bf16", True, True, "heads"), name="attention_one_token"),
        # the backward pass of a causal layer with shared key heads
        dict(_attention("attention_bwd", 1, 32, 8, 4096, 4096, 128, "bf16", True, False, "tokens"), name="backward_long_causal"),
        # the backward pass of a padded batch, every query sees every key of its sequence
        dict(_attention("attention_bwd", 4, 16, 16, 1000, 1000, 64, "f16", False, True, "heads"), name="backward_padded"),
        # a short chunk that continues a sequence: fewer queries than keys, latency counts
        dict(_attention("attention_bwd", 2, 8, 2, 100, 130, 64, "bf16", True, False, "tokens"), name="backward_short"),
        # one token through the two projections: the weights' bytes are the time
        dict(_gated("gated", 1, 4096, 11264, "bf16", False), name="gated_one_token"),
        # a prompt or a training batch, with what its backward pass needs kept
        dict(_gated("gated", 4000, 4096, 11264, "bf16", True), name="gated_batch"),
        # the backward pass of a training batch
        dict(_gated("gated_bwd", 4096, 4096, 11264, "bf16", True), name="gated_backward"),
        # the same of a small layer on a ragged batch
        dict(_gated("gated_bwd", 300, 1000, 2720, "f16", True), name="gated_backward_small"),
        # queries and keys of a packed projection (the values behind them stay out of it)
        dict(_rotary(8192, 40, 48, 128, 128, "bf16", False, False, 131072, 8.0), name="rotary_batch"),
        # one token of each sequence, half of each head rotated, far positions
        dict(_rotary(24, 40, 40, 128, 64, "f16", True, False, 1000000, 1.0), name="rotary_one_token"),
    ]


def _log_int(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    kind = rng.choice(["attention", "attention", "attention_bwd", "attention_bwd", "gated", "gated_bwd", "rotary"])
    if kind.startswith("attention"):
        while True:
            kv_heads = _log_int(rng, 1, 16)
            group = rng.choice([1, 1, 2, 3, 4, 8])
            batch = _log_int(rng, 1, 16)
            # the gradients of a softmax over one key are zero: two keys and more are worth comparing
            n_kv = _log_int(rng, 8 if kind == "attention_bwd" else 1, 8192)
            shape = rng.choice(["same", "same", "same", "one", "chunk", "cross"])
            n_q = {"same": n_kv, "one": 1, "chunk": _log_int(rng, 1, n_kv), "cross": _log_int(rng, 1, 2048)}[shape]
            case = _attention(kind, batch, kv_heads * group, kv_heads, n_q, n_kv, rng.choice([64, 128]),
                              rng.choice(["f16", "bf16"]), rng.random() < 0.6, rng.random() < 0.4,
                              rng.choice(["heads", "tokens"]))
            scores = batch * kv_heads * group * n_q * n_kv
            if scores <= 32 * 4096 * 4096 and batch * kv_heads * n_kv <= 16 * 8 * 8192:
                return case
    if kind.startswith("gated"):
        d_in, d_ff = 8 * _log_int(rng, 8, 512), 8 * _log_int(rng, 8, 1408)
        if rng.random() < 0.15:   # extents that are no multiple of eight
            d_in, d_ff = d_in // 4 + 1, d_ff // 4 + 3
            return _gated(kind, _log_int(rng, 1, 300), d_in, d_ff, rng.choice(["f16", "bf16"]), kind == "gated_bwd")
        return _gated(kind, _log_int(rng, 1, 4096), d_in, d_ff, rng.choice(["f16", "bf16"]),
                      kind == "gated_bwd" or rng.random() < 0.5)
    d_head = rng.choice([64, 80, 96, 128, 256])
    heads = _log_int(rng, 1, 40)
    return _rotary(_log_int(rng, 1, 8192), heads, heads + rng.choice([0, 0, 1, 8]), d_head,
                   rng.choice([d_head, d_head, d_head // 2, d_head // 4]), rng.choice(["f16", "bf16", "f32"]),
                   rng.random() < 0.5, rng.random() < 0.5, rng.choice([4096, 131072, 1000000]), rng.choice([1.0, 4.0, 32.0]))


# --------------------------------------------------------------------------------------------- inputs
def _tensor(g, shape, dtype, std=1.0):
    return (torch.randn(shape, generator=g, device="cuda") * std).to(_TYPES[dtype])


def _frequencies(case):
    """Per pair of dimensions; for long contexts the slow ones are divided by `factor`, the fast ones stay, and those
    between are blended by how many turns they make over 8192 positions."""
    n = case["rot"] // 2
    out = []
    for i in range(n):
        f = 10000.0 ** (-2.0 * i / case["rot"])
        turns = 8192 * f / (2.0 * math.pi)
        blend = min(1.0, max(0.0, (turns - 1.0) / (4.0 - 1.0)))
        out.append(blend * f + (1.0 - blend) * f / case["factor"])
    return out


def _shape(case, heads, rows):
    b, d = case["batch"], case["d_head"]
    return (b, heads, rows, d) if case["layout"] == "heads" else (b, rows, heads, d)


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    s = {"case": case}
    if case["op"].startswith("attention"):
        q, kv = _shape(case, case["q_heads"], case["n_q"]), _shape(case, case["kv_heads"], case["n_kv"])
        s["q"], s["k"], s["v"] = (_tensor(g, x, case["dtype"]) for x in (q, kv, kv))
        s["lens"] = None
        if case["lens"]:  # the last quarter of a sequence may be padding; the first sequence of a batch is empty
            n = case["n_kv"]
            s["lens"] = (n - torch.randint(0, n // 4 + 1, (case["batch"],), generator=g, device="cuda")).to(torch.int32)
            if case["batch"] > 1:
                s["lens"][0] = 0
        if case["op"] == "attention_bwd":
            s["do"] = _tensor(g, q, case["dtype"])
            s["o"], s["lse"] = _plain_attention(s)
    elif case["op"].startswith("gated"):
        m, d, f = case["tokens"], case["d_in"], case["d_ff"]
        s["x"] = _tensor(g, (m, d), case["dtype"])
        s["w"] = _tensor(g, (d, 2 * f), case["dtype"], d ** -0.5)
        if case["op"] == "gated_bwd":
            s["gu"] = (s["x"].float() @ s["w"].float()).to(_TYPES[case["dtype"]])
            s["dh"] = _tensor(g, (m, f), case["dtype"])
    else:
        s["x"] = _tensor(g, (case["tokens"], case["held"], case["d_head"]), case["dtype"])
        s["positions"] = torch.randint(0, case["far"], (case["tokens"],), generator=g, device="cuda", dtype=torch.int32)
        s["frequencies"] = _frequencies(case)
        s["f64"] = torch.tensor(s["frequencies"], dtype=torch.float64, device="cuda")
    if own:
        _bind(s)
    return s


# -------------------------------------------------------------------------------- the framework's calls
_sessions = {}


def _framework():
    from __graft_entry__ import load_package
    pkg = load_package()
    # 1: the handle of the legacy default stream, which every device has
    at = torch.cuda.current_device(), torch.cuda.current_stream().cuda_stream or 1
    if at not in _sessions:
        _sessions[at] = pkg.Session(device=at[0], adopt_stream=at[1])
    return pkg.blob, _sessions[at]


def _bind(s):
    """The kernel handle of the case, its output and workspace buffers, and the bound launch."""
    case = s["case"]
    B, session = _framework()
    t = {"f16": B.F16, "bf16": B.BF16, "f32": B.F32}[case["dtype"]]
    if case["op"].startswith("attention"):
        make = B.attention if case["op"] == "attention" else B.attention_bwd
        desc = make(case["op"], case["batch"], case["q_heads"], case["kv_heads"], case["n_q"], case["n_kv"],
                    case["d_head"], dtype=t, causal=case["causal"], key_lens=case["lens"], layout=case["layout"])
        if case["op"] == "attention":
            o = torch.empty_like(s["q"])
            lse = torch.empty((case["batch"], case["q_heads"], case["n_q"]), dtype=torch.float32, device="cuda")
            args, s["out"] = [s["q"], s["k"], s["v"], o, lse], [o, lse]
        else:
            s["out"] = [torch.empty_like(s[n]) for n in ("q", "k", "v")]
            args = [s["q"], s["k"], s["v"], s["o"], s["do"], s["lse"]] + s["out"]
        if s["lens"] is not None:
            args.append(s["lens"])
    elif case["op"] == "gated":
        m, f = case["tokens"], case["d_ff"]
        desc = B.gated_ffn("gated", m, case["d_in"], f, dtype=t, save_gu=case["save"])
        s["out"] = [s["x"].new_empty((m, f))] + ([s["x"].new_empty((m, 2 * f))] if case["save"] else [])
        args = [s["x"], s["w"]] + s["out"]
    elif case["op"] == "gated_bwd":
        desc = B.gated_ffn_bwd("gated_bwd", case["tokens"], case["d_in"], case["d_ff"], dtype=t)
        s["out"] = [torch.empty_like(s["x"]), torch.empty_like(s["w"])]
        args = [s["x"], s["w"], s["gu"], s["dh"]] + s["out"]
    else:
        shape = (case["tokens"], case["heads"], case["d_head"])
        desc = B.rotary("rotary", *shape, s["frequencies"], dtype=t, interleaved=case["interleaved"],
                        inverse=case["inverse"], x_strides=(case["held"] * case["d_head"], case["d_head"]))
        s["out"] = [s["x"].new_empty(shape)]
        args = [s["x"], s["positions"]] + s["out"]
    kernel = session.kernel(desc)
    need = session.workspace_bytes(kernel)
    if need:
        s["workspace"] = torch.empty(need, dtype=torch.uint8, device="cuda")
        args.append(s["workspace"])
    s["args"] = args
    s["launch"] = session.bind(kernel, [a.data_ptr() for a in args])


def run(s):
    if own:
        s["launch"]()
        return s["out"]
    return _plain(s)


# ------------------------------------------------------------------------------------------ plain form
def _heads_first(x, case):
    return (x if case["layout"] == "heads" else x.transpose(1, 2)).float()


def _as_laid_out(x, case):
    return x if case["layout"] == "heads" else x.transpose(1, 2).contiguous()


def _visible(s, device):
    """[batch or 1, 1, n_q, n_kv] truth values, or None when every query sees every key."""
    case = s["case"]
    n_q, n_kv = case["n_q"], case["n_kv"]
    key = torch.arange(n_kv, device=device)
    seen = None
    if case["causal"]:
        seen = (key[None, :] <= torch.arange(n_q, device=device)[:, None] + (n_kv - n_q))[None, None]
    if s["lens"] is not None:
        inside = (key[None, :] < s["lens"][:, None])[:, None, None, :]
        seen = inside if seen is None else seen & inside
    return seen


def _scores(s):
    case = s["case"]
    group = case["q_heads"] // case["kv_heads"]
    q = _heads_first(s["q"], case)
    k, v = (_heads_first(s[n], case).repeat_interleave(group, 1) for n in ("k", "v"))
    x = torch.matmul(q, k.transpose(2, 3)) * case["d_head"] ** -0.5
    seen = _visible(s, x.device)
    return q, k, v, x if seen is None else x.masked_fill_(~seen, -math.inf)


def _plain_attention(s):
    _, _, v, x = _scores(s)
    top = x.amax(3, keepdim=True)
    e = torch.exp(x - torch.where(top == -math.inf, torch.zeros_like(top), top))
    total = e.sum(3, keepdim=True)
    o = torch.matmul(e, v) / torch.where(total == 0, torch.ones_like(total), total)
    lse = (top + torch.log(total)).squeeze(3)
    return _as_laid_out(o.to(s["q"].dtype), s["case"]), lse


def _plain_attention_bwd(s):
    case = s["case"]
    q, k, v, x = _scores(s)
    lse = s["lse"][..., None]
    p = torch.exp(x - torch.where(lse == -math.inf, torch.zeros_like(lse), lse))
    do, o = _heads_first(s["do"], case), _heads_first(s["o"], case)
    per_kv = (case["batch"], case["kv_heads"], -1, case["n_kv"], case["d_head"])
    dv = torch.matmul(p.transpose(2, 3), do).view(per_kv).sum(2)
    ds = p * (torch.matmul(do, v.transpose(2, 3)) - (do * o).sum(3, keepdim=True)) * case["d_head"] ** -0.5
    dq = torch.matmul(ds, k)
    dk = torch.matmul(ds.transpose(2, 3), q).view(per_kv).sum(2)
    return [_as_laid_out(t.to(s["q"].dtype), case) for t in (dq, dk, dv)]


def _plain_gated(s):
    case, t = s["case"], s["x"].dtype
    gu = s["x"].float() @ s["w"].float()
    g, u = gu[:, :case["d_ff"]], gu[:, case["d_ff"]:]
    h = (g / (1.0 + torch.exp(-g)) * u).to(t)
    return [h, gu.to(t)] if case["save"] else [h]


def _plain_gated_bwd(s):
    f, t = s["case"]["d_ff"], s["x"].dtype
    g, u, dh = s["gu"][:, :f].float(), s["gu"][:, f:].float(), s["dh"].float()
    sig = 1.0 / (1.0 + torch.exp(-g))
    dgu = torch.cat([dh * u * sig * (1.0 + g * (1.0 - sig)), dh * g * sig], 1)
    return [(dgu @ s["w"].float().t()).to(t), (s["x"].float().t() @ dgu).to(t)]


def _plain_rotary(s):
    case = s["case"]
    n, x = case["rot"] // 2, s["x"][:, :case["heads"]].float()
    angle = s["positions"].double()[:, None] * s["f64"][None, :]
    if case["inverse"]:
        angle = -angle
    cos, sin = torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]
    out = x.clone()
    if case["interleaved"]:
        a, b = x[..., 0:2 * n:2], x[..., 1:2 * n:2]
        out[..., 0:2 * n:2], out[..., 1:2 * n:2] = a * cos - b * sin, a * sin + b * cos
    else:
        a, b = x[..., :n], x[..., n:2 * n]
        out[..., :n], out[..., n:2 * n] = a * cos - b * sin, a * sin + b * cos
    return [out.to(s["x"].dtype)]


def _plain(s):
    form = {"attention": _plain_attention, "attention_bwd": _plain_attention_bwd, "gated": _plain_gated,
            "gated_bwd": _plain_gated_bwd, "rotary": _plain_rotary}[s["case"]["op"]]
    return list(form(s))


# ------------------------------------------------------------------------------------ exact, in 64 bits
def exact(case, seed):
    global own
    keep, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = keep
    if case["op"].startswith("attention"):
        tokens = case["layout"] == "tokens"
        group, d, n_q, n_kv = case["q_heads"] // case["kv_heads"], case["d_head"], case["n_q"], case["n_kv"]
        ins = {n: (s[n].transpose(1, 2) if tokens else s[n]) for n in ("q", "k", "v", "do") if n in s}
        back = "do" in ins
        outs = [torch.zeros(ins[n].shape, dtype=torch.float64, device="cuda") for n in (("q", "k", "v") if back else ("q",))]
        lse = torch.empty((case["batch"], case["q_heads"], n_q), dtype=torch.float64, device="cuda")
        late = torch.arange(n_kv, device="cuda")[None] > torch.arange(n_q, device="cuda")[:, None] + (n_kv - n_q)
        for b in range(case["batch"]):
            length = n_kv if s["lens"] is None else int(s["lens"][b])
            for h in range(case["q_heads"]):
                if length == 0:
                    lse[b, h] = -math.inf
                    continue
                q, k, v = ins["q"][b, h].double(), ins["k"][b, h // group, :length].double(), ins["v"][b, h // group, :length].double()
                leaves = [t.requires_grad_(back) for t in (q, k, v)]
                x = q @ k.t() / math.sqrt(d)
                if case["causal"]:
                    x = x.masked_fill(late[:, :length], -math.inf)
                some = (x.detach() > -math.inf).any(1)
                o = torch.softmax(x[some], 1) @ v
                if back:
                    got = torch.autograd.grad(o, leaves, ins["do"][b, h].double()[some])
                    outs[0][b, h] = got[0]
                    outs[1][b, h // group, :length] += got[1]
                    outs[2][b, h // group, :length] += got[2]
                else:
                    outs[0][b, h][some] = o
                    lse[b, h] = torch.logsumexp(x, 1)
        outs = [t.transpose(1, 2).contiguous() if tokens else t for t in outs]
        return outs if back else outs + [lse]
    if case["op"].startswith("gated"):
        f = case["d_ff"]
        x, w = s["x"].double(), s["w"].double()
        if case["op"] == "gated":
            gu = x @ w
            h = torch.nn.functional.silu(gu[:, :f]) * gu[:, f:]
            return [h, gu] if case["save"] else [h]
        gu = s["gu"].double().requires_grad_(True)
        h = torch.nn.functional.silu(gu[:, :f]) * gu[:, f:]
        dgu, = torch.autograd.grad(h, gu, s["dh"].double())
        return [dgu @ w.t(), x.t() @ dgu]
    n = case["rot"] // 2
    x = s["x"][:, :case["heads"]].double()
    turn = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"),
                       torch.outer(s["positions"].double(), s["f64"]) * (-1 if case["inverse"] else 1))[:, None]
    r, rest = x[..., :2 * n], x[..., 2 * n:]
    if case["interleaved"]:
        z = torch.view_as_complex(r.reshape(*r.shape[:2], n, 2).contiguous()) * turn
        r = torch.view_as_real(z).reshape(r.shape)
    else:
        z = torch.complex(r[..., :n].contiguous(), r[..., n:].contiguous()) * turn
        r = torch.cat([z.real, z.imag], -1)
    return [torch.cat([r, rest], -1)]


# ---------------------------------------------------------------------------------------------- work
def work(case):
    e = 4 if case["dtype"] == "f32" else 2
    if case["op"].startswith("attention"):
        b, hq, hkv, n_q, n_kv, d = (case[n] for n in ("batch", "q_heads", "kv_heads", "n_q", "n_kv", "d_head"))
        share = 1.0  # of the keys that are there: lengths lose an eighth on average, and the first sequence
        if case["lens"]:
            share = 0.875 * ((b - 1) / b if b > 1 else 1.0)
        off = n_kv - n_q
        pairs = sum(min(n_kv, max(0, i + off + 1)) for i in range(n_q)) if case["causal"] else n_q * n_kv
        rows, keys = b * hq * n_q * d * e, b * hkv * n_kv * d * e * share
        stats = b * hq * n_q * 4
        if case["op"] == "attention":
            return {"bytes": 2 * rows + 2 * keys + stats, "flops": 4.0 * b * hq * pairs * d * share}
        return {"bytes": 4 * rows + 4 * keys + stats, "flops": 10.0 * b * hq * pairs * d * share}
    if case["op"].startswith("gated"):
        m, d, f = case["tokens"], case["d_in"], case["d_ff"]
        if case["op"] == "gated":
            return {"bytes": e * (m * d + 2 * d * f + m * f * (3 if case["save"] else 1)), "flops": 4.0 * m * d * f}
        return {"bytes": e * (2 * m * d + 4 * d * f + 3 * m * f), "flops": 8.0 * m * d * f}
    n = case["tokens"] * case["heads"]
    return {"bytes": 2 * n * case["d_head"] * e + 4 * case["tokens"], "flops": 3.0 * n * case["rot"]}
