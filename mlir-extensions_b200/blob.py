"""Kernel-descriptor blobs (include/imex_b200_blob.h) built from Python.

A blob is what the front end attaches to a gpu.module in place of the
reference's serialised SPIR-V (lib/Transforms/SerializeSPIRV.cpp:64-69) and
what gpuModuleLoad receives."""
import ctypes as C
import math
import struct

MAGIC = 0x0030303242584D49
VERSION = 1
NAME_MAX = 64

OP_GEMM, OP_SOFTMAX, OP_REDUCE_ROWS, OP_REDUCE_LEADING, OP_REDUCE_ALL = 1, 2, 3, 4, 5
OP_TRANSPOSE2D, OP_TRANSPOSE3D, OP_ELTWISE, OP_FILL_UNIFORM, OP_FILL_NORMAL = 6, 7, 8, 9, 10
OP_EXPR, OP_ATTENTION_FWD, OP_LOOPNEST = 11, 12, 13
OP_ATTENTION, OP_ATTENTION_BWD, OP_GATED_FFN, OP_GATED_FFN_BWD, OP_ROTARY = 14, 15, 16, 17, 18
F32, BF16, F16, I32 = 1, 2, 3, 4
EPI_NONE, EPI_RELU, EPI_SILU = 0, 1, 2
FLAG_ACCUMULATE, FLAG_BIAS, FLAG_SOFTMAX_NEG_INF, FLAG_TRANS_A, FLAG_TRANS_B = 1, 2, 4, 8, 16
FLAG_REDUCE_LEADING = 32
FLAG_CAUSAL, FLAG_KEY_LENS, FLAG_SAVE_GU, FLAG_INTERLEAVED, FLAG_INVERSE = 64, 128, 256, 512, 1024

DTYPE_BYTES = {F32: 4, I32: 4, BF16: 2, F16: 2}
_DESC = struct.Struct("<64s6I6q2f")  # ImexKernelDesc, 144 bytes
_HEADER = struct.Struct("<QII")      # ImexBlobHeader, 16 bytes
assert _DESC.size == 144 and _HEADER.size == 16


class KernelDesc:
    def __init__(self, name, op, in_dtype=F32, out_dtype=F32, epilogue=EPI_NONE, flags=0,
                 dims=(), fparams=(0.0, 0.0), sm_margin=0):
        if len(name.encode()) >= NAME_MAX:
            raise ValueError("kernel name too long")
        if len(dims) > 6:
            raise ValueError("at most 6 dims")
        self.name, self.op = name, op
        self.in_dtype, self.out_dtype = in_dtype, out_dtype
        self.epilogue, self.flags = epilogue, flags
        self.sm_margin = int(sm_margin)
        self.dims = tuple(int(d) for d in dims) + (0,) * (6 - len(dims))
        self.fparams = tuple(float(f) for f in fparams)
        self.payload = b""  # the kernel's text (OP_LOOPNEST) or a shape struct; placed behind the table by pack_blob

    def pack(self):
        return _DESC.pack(self.name.encode(), self.op, self.in_dtype, self.out_dtype,
                          self.epilogue, self.flags, self.sm_margin, *self.dims, *self.fparams)

    def key(self):
        """Equal for descriptors of the same kernel (where in a blob the payload lies is not part of it)."""
        dims = self.dims[:1] + (0, 0) + tuple(self.dims[3:]) if self.payload else self.dims
        return _DESC.pack(self.name.encode(), self.op, self.in_dtype, self.out_dtype, self.epilogue, self.flags,
                          self.sm_margin, *dims, *self.fparams), bytes(self.payload)


def pack_blob(descs):
    """bytes of a blob holding `descs` (list of KernelDesc): header, descriptor table, then
    the payloads (kernel text, shape structs: addressed by offset and length in dims[1],
    dims[2])."""
    table_end = _HEADER.size + len(descs) * _DESC.size
    payload = b""
    for d in descs:
        if d.payload:
            d.dims = (d.dims[0], table_end + len(payload), len(d.payload)) + tuple(d.dims[3:])
            payload += d.payload
    return _HEADER.pack(MAGIC, VERSION, len(descs)) + b"".join(d.pack() for d in descs) + payload


def unpack_blob(data):
    magic, version, n = _HEADER.unpack_from(data, 0)
    if magic != MAGIC:
        raise ValueError("bad blob magic")
    out = []
    for i in range(n):
        f = _DESC.unpack_from(data, _HEADER.size + i * _DESC.size)
        out.append(KernelDesc(f[0].split(b"\0")[0].decode(), f[1], f[2], f[3], f[4], f[5],
                              f[7:13], f[13:15], sm_margin=f[6]))
    return version, out


def gemm(name, M, N, K, in_dtype=BF16, epilogue=EPI_NONE, accumulate=False, bias=False,
         lda=0, ldb=0, ldc=0, sm_margin=0, trans_a=False, trans_b=False, out_dtype=F32):
    """lda/ldb/ldc: row pitches of the arrays as stored, in elements (0 = dense);
    sm_margin: SMs the persistent kernel leaves free (for a collective running
    beside it); trans_a: A is stored [K,M]; trans_b: B is stored [N,K]; out_dtype
    BF16/F16: f32 accumulation, one rounding at the end."""
    flags = ((FLAG_ACCUMULATE if accumulate else 0) | (FLAG_BIAS if bias else 0)
             | (FLAG_TRANS_A if trans_a else 0) | (FLAG_TRANS_B if trans_b else 0))
    return KernelDesc(name, OP_GEMM, in_dtype, out_dtype, epilogue, flags, (M, N, K, lda, ldb, ldc),
                      sm_margin=sm_margin)


# postfix code of OP_EXPR (ImexExprCode)
X_END, X_IN, X_ROWV, X_COLV, X_C0, X_C1, X_ZERO, X_ONE = 0, 1, 5, 9, 13, 14, 15, 16
X_UNARY = {"neg": 32, "abs": 33, "log": 34, "exp": 35, "sqrt": 36, "rsqrt": 37, "tanh": 38, "relu": 39}
X_BINARY = {"add": 64, "sub": 65, "mul": 66, "div": 67, "max": 68, "min": 69}
EXPR_MAX_CODE = 32


def assemble_expr(text):
    """Postfix text -> code bytes.  Tokens: in0..in3 (full tensors), row0..row3 (row
    vectors [cols]), col0..col3 (column vectors [rows]), c0, c1 (fparams), zero, one,
    and the operation names of X_UNARY / X_BINARY.  "in0 log in1 abs add in0 sub" is
    (log(x0) + |x1|) - x0."""
    code = []
    for tok in text.split():
        if tok[:-1] in ("in", "row", "col") and tok[-1].isdigit() and int(tok[-1]) < 4:
            code.append({"in": X_IN, "row": X_ROWV, "col": X_COLV}[tok[:-1]] + int(tok[-1]))
        elif tok in ("c0", "c1", "zero", "one"):
            code.append({"c0": X_C0, "c1": X_C1, "zero": X_ZERO, "one": X_ONE}[tok])
        elif tok in X_UNARY:
            code.append(X_UNARY[tok])
        elif tok in X_BINARY:
            code.append(X_BINARY[tok])
        else:
            raise ValueError("unknown token %r in expression" % tok)
    if not 0 < len(code) <= EXPR_MAX_CODE:
        raise ValueError("expression programs hold 1..%d operations" % EXPR_MAX_CODE)
    return bytes(code)


def expr(name, rows, cols, program, dtype=F32, out_dtype=None, reduce_leading=False,
         accumulate=False, consts=(0.0, 0.0)):
    """Fused elementwise chain: pointers = the inputs in order, then Y.  `program` is
    postfix text (assemble_expr) or code bytes."""
    code = assemble_expr(program) if isinstance(program, str) else bytes(program)
    words = struct.unpack("<4q", code.ljust(EXPR_MAX_CODE, b"\0"))
    flags = (FLAG_REDUCE_LEADING if reduce_leading else 0) | (FLAG_ACCUMULATE if accumulate else 0)
    return KernelDesc(name, OP_EXPR, dtype, dtype if out_dtype is None else out_dtype, 0, flags,
                      (rows, cols) + words, fparams=consts)


def loopnest(name, source, threads, n_pointers):
    """A loop-nest kernel given as CUDA C++ text: one `extern "C" __global__ void
    imex_loopnest(pointers...)` written against the runtime's loop-nest prelude (element-type
    helpers, IMX_THREAD_INDEX); compiled for sm_100a at first launch and run over `threads`
    points.  Pointers = the kernel's arguments in order."""
    d = KernelDesc(name, OP_LOOPNEST, 0, 0, 0, 0, (threads, 0, 0, n_pointers))
    d.payload = source.encode() if isinstance(source, str) else bytes(source)
    return d


def attention_fwd(name, heads, n_ctx, d_head=64, dtype=F16, sm_scale=0.5):
    """Pointers Q, K, V, O: [heads * n_ctx, d_head] arrays of dtype, heads one after the other."""
    return KernelDesc(name, OP_ATTENTION_FWD, dtype, dtype, 0, 0, (heads, n_ctx, d_head),
                      fparams=(sm_scale, 0.0))


def _rows_overlap(width, steps):
    """Whether rows of `width` elements repeated by (stride, extent) pairs share elements."""
    for step, extent in sorted((s, n) for s, n in steps if n > 1):
        if step < width:
            return True
        width += step * (extent - 1)
    return False


# array order of ImexAttentionShape.strides
_ATTENTION_ARRAYS = ("q", "k", "v", "o", "do", "dq", "dk", "dv")


def _attention(op, name, batch, q_heads, kv_heads, n_q, n_kv, d_head, dtype, sm_scale, causal, key_lens, layout, strides):
    batch, q_heads, kv_heads, n_q, n_kv, d_head = (int(v) for v in (batch, q_heads, kv_heads, n_q, n_kv, d_head))
    if min(batch, q_heads, kv_heads, n_q, n_kv) < 1:
        raise ValueError("attention: batch, heads and lengths are at least 1 (key_lens may be 0)")
    if q_heads % kv_heads:
        raise ValueError("attention: q_heads must be a multiple of kv_heads")
    if d_head not in (64, 128):
        raise ValueError("attention: d_head is 64 or 128")
    if dtype not in (F16, BF16):
        raise ValueError("attention: the element type is F16 or BF16")
    if layout not in ("heads", "tokens"):
        raise ValueError('attention: layout is "heads" ([batch, heads, rows, d]) or "tokens" ([batch, rows, heads, d])')
    sm_scale = d_head ** -0.5 if sm_scale is None else float(sm_scale)
    if not 0 < sm_scale <= 1e30:
        raise ValueError("attention: sm_scale must be positive and at most 1e30")
    strides = dict(strides or {})
    table = []
    for a in _ATTENTION_ARRAYS:
        heads, rows = (kv_heads, n_kv) if a in ("k", "v", "dk", "dv") else (q_heads, n_q)
        if a in strides:
            s = tuple(int(v) for v in strides.pop(a))
            if len(s) != 3 or any(v % 8 for v in s) or min(s) < 0:
                raise ValueError("attention: the strides of %r are (batch, head, row) in elements, multiples of 8" % a)
            if any(step == 0 and n > 1 for step, n in zip(s, (batch, heads, rows))):
                raise ValueError("attention: a stride of %r is zero" % a)
            if a in ("o", "dq", "dk", "dv") and _rows_overlap(d_head, zip(s, (batch, heads, rows))):
                raise ValueError("attention: the rows of the output %r overlap" % a)
        elif layout == "heads":
            s = (heads * rows * d_head, rows * d_head, d_head)
        else:
            s = (rows * heads * d_head, d_head, heads * d_head)
        table += s
    if strides:
        raise ValueError("attention: strides of unknown arrays %s" % sorted(strides))
    d = KernelDesc(name, op, dtype, dtype, 0, (FLAG_CAUSAL if causal else 0) | (FLAG_KEY_LENS if key_lens else 0),
                   (), fparams=(sm_scale, 0.0))
    d.payload = struct.pack("<30q", batch, q_heads, kv_heads, n_q, n_kv, d_head, *table)
    return d


def attention(name, batch, q_heads, kv_heads, n_q, n_kv, d_head, dtype=BF16, sm_scale=None, causal=False,
              key_lens=False, layout="heads", strides=None):
    """Attention forward with row statistics.  Pointers Q, K, V, O, LSE (f32 [batch, q_heads, n_q]), then
    key_lens (int32 [batch]) when asked for, then the workspace when Session.workspace_bytes says so.

    Key j is visible to query i of batch b when j < key_lens[b] and, when causal, j <= i + n_kv - n_q
    (the last query sees every key: the diagonal belongs to n_kv, not to key_lens[b], so that causal with key_lens
    fits prompts that start at position 0 and single new tokens, not chunks behind caches of different
    lengths).  O = softmax(sm_scale Q K^T) V over the visible keys, LSE = log of
    the sum of exponentials; a row that sees no key gets O = 0 and LSE = -inf.  Keys and values at and
    behind key_lens[b] may hold anything, NaN included; elsewhere a NaN or infinite score makes the rows that see
    it NaN, LSE included (and under the causal mask a non-finite V of a later key of the same tile reaches earlier
    queries as 0 * inf).  P is rounded to the element type in between; sums stay in 32 bits.
    q_heads / kv_heads query heads share a key head.  sm_scale: 1 / sqrt(d_head) unless given.
    layout: "heads" for [batch, heads, rows, d] arrays, "tokens" for [batch, rows, heads, d];
    strides: {"q" | "k" | "v" | "o": (batch, head, row)} in elements overrides it per array.  O may be Q (with the
    same strides) and otherwise shares no element with an input."""
    return _attention(OP_ATTENTION, name, batch, q_heads, kv_heads, n_q, n_kv, d_head, dtype, sm_scale, causal,
                      key_lens, layout, strides)


def attention_bwd(name, batch, q_heads, kv_heads, n_q, n_kv, d_head, dtype=BF16, sm_scale=None, causal=False,
                  key_lens=False, layout="heads", strides=None):
    """The gradients of `attention` for dO, with the probabilities recomputed from LSE.  Pointers Q, K, V,
    O, dO, LSE, dQ, dK, dV, then key_lens and the workspace as in `attention`.  Gradients of shared key
    heads are summed over their query heads; masked keys and rows that see no key get zeros.  P and
    dS = P (dO V^T - rowsum(dO O)) are rounded to the element type in between, so with F16 |dS| has to stay
    below 65504, and what of it is below 2^-14 loses bits (scale the loss).  The result does not change from run to run (no atomics).  strides also takes "do", "dq", "dk", "dv".
    The gradients share no element with Q, K, V, dO or one another."""
    return _attention(OP_ATTENTION_BWD, name, batch, q_heads, kv_heads, n_q, n_kv, d_head, dtype, sm_scale, causal,
                      key_lens, layout, strides)


def _gated(op, name, tokens, d_in, d_ff, dtype, act, flags, ldx, ldw, ldh):
    if min(tokens, d_in, d_ff) < 1:
        raise ValueError("gated_ffn: extents are at least 1")
    if dtype not in (F16, BF16):
        raise ValueError("gated_ffn: the element type is F16 or BF16")
    if act not in (EPI_NONE, EPI_RELU, EPI_SILU):
        raise ValueError("gated_ffn: the activation is EPI_NONE, EPI_RELU or EPI_SILU")
    for pitch, width in ((ldx, d_in), (ldw, 2 * d_ff), (ldh, d_ff)):
        if pitch and pitch < width:
            raise ValueError("gated_ffn: row pitch smaller than the row")
    return KernelDesc(name, op, dtype, dtype, act, flags, (tokens, d_in, d_ff, ldx, ldw, ldh))


def gated_ffn(name, tokens, d_in, d_ff, dtype=BF16, act=EPI_SILU, save_gu=False, ldx=0, ldw=0, ldh=0):
    """H = act(X Wg) * (X Wu).  Pointers X [tokens, d_in], W [d_in, 2 * d_ff] (the gate's columns, then
    the up projection's), H [tokens, d_ff], and with save_gu GU [tokens, 2 * d_ff] = X W for the backward
    pass, then the workspace when Session.workspace_bytes says so (extents or pitches that are not multiples
    of 8).  f32 accumulation; H and GU are rounded once.  ldx / ldw / ldh: row pitches in elements (0 = dense;
    GU is dense).  Arrays start on 16-byte boundaries unless the extents need the workspace.  H and GU share no element
    with X, W or one another."""
    return _gated(OP_GATED_FFN, name, tokens, d_in, d_ff, dtype, act, FLAG_SAVE_GU if save_gu else 0, ldx, ldw, ldh)


def gated_ffn_bwd(name, tokens, d_in, d_ff, dtype=BF16, act=EPI_SILU, ldx=0, ldw=0, ldh=0):
    """The gradients of `gated_ffn` for dH.  Pointers X, W, GU (as the forward pass kept it), dH, dX, dW,
    workspace (Session.workspace_bytes).  [dG dU] is rounded to the element type in between, so with F16 |dG| and
    |dU| have to stay below 65504, and what of them is below 2^-14 loses bits (scale the loss).  relu's slope at
    0 is 0.  dX has X's shape and pitch, dW those of W, dH those of H.  dX and dW share no element with X, W or one
    another."""
    return _gated(OP_GATED_FFN_BWD, name, tokens, d_in, d_ff, dtype, act, 0, ldx, ldw, ldh)


ROTARY_MAX_PAIRS = 128


def rotary_frequencies(rot_dims, base=10000.0, factor=1.0, original_length=None, slow_turns=1.0, fast_turns=4.0):
    """base^(-2i / rot_dims) for every pair.  factor > 1 stretches the range of positions by it: all
    frequencies are divided by it (original_length None), or only those of pairs that make fewer than
    slow_turns turns over original_length positions; pairs with more than fast_turns keep theirs and the
    ones between are blended linearly."""
    out = []
    for i in range(rot_dims // 2):
        f = float(base) ** (-2.0 * i / rot_dims)
        keep = 0.0
        if original_length is not None:
            turns = original_length * f / (2.0 * math.pi)
            keep = min(1.0, max(0.0, (turns - slow_turns) / (fast_turns - slow_turns)))
        out.append(keep * f + (1.0 - keep) * f / factor)
    return out


def rotary(name, tokens, heads, d_head, frequencies, dtype=BF16, interleaved=False, inverse=False, factor=1.0,
           x_strides=None, y_strides=None):
    """Rotary positions.  Pointers X [tokens, heads, d_head], positions (int32 [tokens]), Y.  The first
    2 * len(frequencies) dimensions of every head are turned in pairs by position * frequency (angles are
    reduced in 64 bits, so far positions keep their precision) and multiplied by `factor`; the others are
    copied.  Pairs are (i, i + n) of the n frequencies, or (2i, 2i + 1) when interleaved.  inverse turns
    the other way: the gradient.  Y may be X (with the same strides) and otherwise
    shares no element with it.  x_strides / y_strides: (token, head) in elements, for heads inside a packed projection."""
    freqs = [float(f) for f in frequencies]
    if min(tokens, heads, d_head) < 1:
        raise ValueError("rotary: extents are at least 1")
    if d_head > 512:
        raise ValueError("rotary: d_head is at most 512")
    if not 1 <= len(freqs) <= ROTARY_MAX_PAIRS or 2 * len(freqs) > d_head:
        raise ValueError("rotary: 1..%d frequencies, two dimensions of the head each" % ROTARY_MAX_PAIRS)
    if not all(math.isfinite(f) for f in freqs) or not math.isfinite(factor):
        raise ValueError("rotary: frequencies and factor must be finite")
    if dtype not in (F32, F16, BF16):
        raise ValueError("rotary: the element type is F32, F16 or BF16")
    xs, ys = (tuple(int(v) for v in (s or (heads * d_head, d_head))) for s in (x_strides, y_strides))
    if any(len(s) != 2 or min(s) < 0 for s in (xs, ys)):
        raise ValueError("rotary: strides are (token, head) in elements")
    if _rows_overlap(d_head, zip(ys, (tokens, heads))):
        raise ValueError("rotary: the rows of Y overlap")
    d = KernelDesc(name, OP_ROTARY, dtype, dtype, 0, (FLAG_INTERLEAVED if interleaved else 0) | (FLAG_INVERSE if inverse else 0),
                   (), fparams=(factor, 0.0))
    turns = [f / (2.0 * math.pi) for f in freqs] + [0.0] * (ROTARY_MAX_PAIRS - len(freqs))
    d.payload = struct.pack("<8q%dd" % ROTARY_MAX_PAIRS, tokens, heads, d_head, 2 * len(freqs), *xs, *ys, *turns)
    return d


def softmax(name, rows, cols, neg_inf_init=False, dtype=F32):
    """dtype F16 / BF16: every operation of the chain rounds to the element type."""
    return KernelDesc(name, OP_SOFTMAX, dtype, dtype, 0, FLAG_SOFTMAX_NEG_INF if neg_inf_init else 0,
                      (rows, cols))


def reduce_rows(name, rows, cols, accumulate=False):
    return KernelDesc(name, OP_REDUCE_ROWS, F32, F32, 0, FLAG_ACCUMULATE if accumulate else 0,
                      (rows, cols))


def reduce_leading(name, lead, inner, accumulate=False):
    return KernelDesc(name, OP_REDUCE_LEADING, F32, F32, 0, FLAG_ACCUMULATE if accumulate else 0,
                      (lead, inner))


def reduce_all(name, n, accumulate=False):
    return KernelDesc(name, OP_REDUCE_ALL, F32, F32, 0, FLAG_ACCUMULATE if accumulate else 0, (n,))


def transpose2d(name, rows, cols, dtype=F32):
    return KernelDesc(name, OP_TRANSPOSE2D, dtype, dtype, 0, 0, (rows, cols))


def transpose3d(name, dims, perm, dtype=F32):
    return KernelDesc(name, OP_TRANSPOSE3D, dtype, dtype, 0, 0, tuple(dims) + tuple(perm))


def eltwise(name, n, epilogue):
    return KernelDesc(name, OP_ELTWISE, F32, F32, epilogue, 0, (n,))


def convert(name, n, in_dtype, out_dtype):
    """arith.extf / arith.truncf between f32 and bf16 / f16."""
    return KernelDesc(name, OP_ELTWISE, in_dtype, out_dtype, EPI_NONE, 0, (n,))


def fill_uniform(name, n, dtype, seed, lo, hi, first=0):
    return KernelDesc(name, OP_FILL_UNIFORM, dtype, dtype, 0, 0, (n, seed, first), (lo, hi))


def fill_normal(name, n, dtype, seed, mean, stddev, first=0):
    return KernelDesc(name, OP_FILL_NORMAL, dtype, dtype, 0, 0, (n, seed, first), (mean, stddev))


_KEEP = []


class Blob:
    """Owns the bytes at a fixed address for the life of the process.

    gpuModuleLoad caches parsed modules by blob ADDRESS until exit (in the
    reference the blob is a global constant of the compiled host module), so a
    blob must never be freed and its address reused for other contents."""

    def __init__(self, descs):
        _KEEP.append(self)
        self.descs = list(descs)
        data = pack_blob(self.descs)
        self.buffer = C.create_string_buffer(data, len(data))
        self.size = len(data)

    @property
    def address(self):
        return C.addressof(self.buffer)
