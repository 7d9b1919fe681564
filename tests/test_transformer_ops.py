"""Descriptors and refusals of the attention, gated feed-forward and rotary operators (no GPU)."""
import ctypes as C
import os
import struct
import subprocess
import sys

import pytest

from __graft_entry__ import ROOT, load_package

pkg = load_package()
B, rt = pkg.blob, pkg.runtime


def _kernel(desc):
    blob = B.Blob([desc])
    return rt.gpuKernelGet(None, rt.gpuModuleLoad(None, blob.address, blob.size), desc.name.encode())


def test_attention_descriptor():
    d = B.attention("a", 2, 8, 2, 100, 130, 64, dtype=B.F16, causal=True, key_lens=True, layout="tokens")
    assert d.op == B.OP_ATTENTION and d.flags == B.FLAG_CAUSAL | B.FLAG_KEY_LENS and d.fparams[0] == 0.125
    words = struct.unpack("<30q", d.payload)
    assert words[:6] == (2, 8, 2, 100, 130, 64)
    assert words[6:9] == (100 * 8 * 64, 64, 8 * 64) and words[9:12] == (130 * 2 * 64, 64, 2 * 64)
    d = B.attention_bwd("a", 1, 4, 4, 10, 10, 128, sm_scale=0.5, strides={"dk": (0, 128, 512), "q": (8, 16, 24)})
    words = struct.unpack("<30q", d.payload)
    assert words[6:9] == (8, 16, 24) and words[24:27] == (0, 128, 512) and words[27:30] == (5120, 1280, 128)


@pytest.mark.parametrize("change,message", [
    ({"batch": 0}, "at least 1"), ({"n_q": 0}, "at least 1"), ({"n_kv": -1}, "at least 1"), ({"q_heads": 3}, "multiple"),
    ({"d_head": 96}, "64 or 128"), ({"dtype": 1}, "F16 or BF16"), ({"layout": "rows"}, "layout"),
    ({"sm_scale": 0.0}, "positive"), ({"sm_scale": -1.0}, "positive"), ({"sm_scale": float("nan")}, "positive"),
    ({"strides": {"q": (1, 2)}}, "multiples of 8"), ({"strides": {"q": (64, 64, 68)}}, "multiples of 8"),
    ({"strides": {"x": (64, 64, 64)}}, "unknown"), ({"strides": {"k": (0, 64, 128)}}, "zero"), ({"sm_scale": 1e31}, "positive"), ({"strides": {"o": (640, 64, 8)}}, "overlap")])
def test_attention_refusals(change, message):
    args = dict(batch=2, q_heads=4, kv_heads=2, n_q=10, n_kv=10, d_head=64)
    args.update(change)
    with pytest.raises(ValueError, match=message):
        B.attention("a", **args)


def test_gated_descriptor_and_refusals():
    d = B.gated_ffn("g", 3, 16, 32, dtype=B.F16, act=B.EPI_RELU, save_gu=True, ldx=24)
    assert d.op == B.OP_GATED_FFN and d.epilogue == B.EPI_RELU and d.flags == B.FLAG_SAVE_GU
    assert d.dims == (3, 16, 32, 24, 0, 0)
    assert B.gated_ffn_bwd("g", 3, 16, 32).op == B.OP_GATED_FFN_BWD
    for bad in (dict(tokens=0), dict(d_ff=0), dict(dtype=B.F32), dict(act=7), dict(ldw=63), dict(ldh=31)):
        args = dict(tokens=3, d_in=16, d_ff=32)
        args.update(bad)
        with pytest.raises(ValueError):
            B.gated_ffn("g", **args)


def test_rotary_descriptor_and_refusals():
    d = B.rotary("r", 5, 2, 64, [1.0, 0.5], dtype=B.F32, interleaved=True, inverse=True, factor=2.0, x_strides=(200, 70))
    assert d.op == B.OP_ROTARY and d.flags == B.FLAG_INTERLEAVED | B.FLAG_INVERSE and d.fparams[0] == 2.0
    assert struct.unpack("<8q", d.payload[:64]) == (5, 2, 64, 4, 200, 70, 128, 64)
    for bad in (dict(tokens=0), dict(frequencies=[]), dict(frequencies=[1.0] * 33), dict(frequencies=[float("inf")]),
                dict(dtype=B.I32), dict(y_strides=(200, 63)), dict(y_strides=(100, 64)), dict(x_strides=(1, 2, 3)),
                dict(x_strides=(-64, 64)), dict(d_head=513)):
        args = dict(tokens=5, heads=2, d_head=64, frequencies=[1.0])
        args.update(bad)
        with pytest.raises(ValueError):
            B.rotary("r", **args)


def test_rotary_frequencies():
    f = B.rotary_frequencies(64)
    assert len(f) == 32 and f[0] == 1.0 and f[-1] == pytest.approx(10000.0 ** (-62 / 64))
    assert B.rotary_frequencies(64, factor=4.0) == pytest.approx([x / 4 for x in f])
    g = B.rotary_frequencies(64, factor=4.0, original_length=4096)
    turns = [4096 * x / 6.283185307179586 for x in f]
    for x, y, t in zip(f, g, turns):
        assert y == pytest.approx(x if t >= 4 else x / 4 if t <= 1 else x / 4 + (t - 1) / 3 * x * 0.75)


def test_workspace_bytes():
    assert rt.imexKernelWorkspaceBytes(_kernel(B.softmax("s", 4, 8))) == 0
    assert rt.imexKernelWorkspaceBytes(_kernel(B.attention_bwd("a", 3, 4, 2, 50, 60, 64))) >= 3 * 4 * 50 * 4
    assert rt.imexKernelWorkspaceBytes(_kernel(B.gated_ffn_bwd("g", 30, 64, 72))) >= 30 * 2 * 72 * 2
    # the gated product wants one only for extents or pitches that are not multiples of eight: its padded operands
    assert rt.imexKernelWorkspaceBytes(_kernel(B.gated_ffn("g", 30, 64, 72))) == 0
    for args in (dict(d_in=63, d_ff=72), dict(d_in=64, d_ff=71), dict(d_in=64, d_ff=72, ldx=65), dict(d_in=64, d_ff=72, ldw=145)):
        d_in = (args["d_in"] + 7) // 8 * 8
        assert rt.imexKernelWorkspaceBytes(_kernel(B.gated_ffn("g", 30, **args))) >= (30 * d_in + args["d_in"] * 2 * 72) * 2


@pytest.mark.parametrize("patch,message", [
    ("d.payload = d.payload[:-8]", "no shape payload"),
    ("d.payload = b''", "no shape payload|outside the blob"),
    ("d.in_dtype = d.out_dtype = B.F32", "element type"),
    ("d.out_dtype = B.F16", "keeps its element type"),
    ("d.fparams = (-1.0, 0.0)", "sm_scale"),
    ("d.payload = struct.pack('<q', 0) + d.payload[8:]", "at least 1"),
    ("d.payload = d.payload[:40] + struct.pack('<q', 80) + d.payload[48:]", "64 or 128"),
    ("d.payload = d.payload[:64] + struct.pack('<q', 63) + d.payload[72:]", "multiples of 8")])
def test_malformed_attention_blobs_follow_the_error_convention(patch, message):
    """A descriptor the builder would not make: one line on stdout, then abort()."""
    text = ("import struct\nfrom __graft_entry__ import load_package\npkg = load_package()\nB, rt = pkg.blob, pkg.runtime\n"
            "d = B.attention_bwd('a', 2, 2, 1, 8, 8, 64)\n%s\nblob = B.Blob([d])\n"
            "k = rt.gpuKernelGet(None, rt.gpuModuleLoad(None, blob.address, blob.size), b'a')\n"
            "rt.imexKernelWorkspaceBytes(k)\n" % patch)
    r = subprocess.run([sys.executable, "-c", text], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert r.returncode == -6
    import re
    assert re.search("An exception was thrown: .*(%s)" % message, r.stdout), r.stdout


def test_the_structs_match_the_header(tmp_path):
    """Sizes of the payload structs as the C compiler sees them."""
    src = tmp_path / "t.c"
    src.write_text('#include "imex_b200_blob.h"\n#include <stdio.h>\nint main(void) { printf("%zu %zu\\n", '
                   "sizeof(ImexAttentionShape), sizeof(ImexRotaryShape)); return 0; }\n")
    exe = tmp_path / "t"
    subprocess.check_call(["/usr/bin/gcc", "-I" + os.path.join(ROOT, "include"), "-o", str(exe), str(src)])
    a, r = (int(x) for x in subprocess.check_output([str(exe)], text=True).split())
    assert a == len(B.attention("a", 1, 1, 1, 1, 1, 64).payload)
    assert r == len(B.rotary("r", 1, 1, 64, [1.0]).payload)
    assert C.sizeof(C.c_double) == 8
