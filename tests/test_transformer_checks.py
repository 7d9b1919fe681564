"""Checks of the attention, gated feed-forward and rotary operators that need no GPU, beyond test_transformer_ops.py."""
import glob
import os
import subprocess
import sys

import pytest

from __graft_entry__ import ROOT, load_package

pkg = load_package()
B, rt = pkg.blob, pkg.runtime
KERNELS = os.path.join(ROOT, "mlir-extensions_b200", "csrc", "kernels")


def test_dynamic_shared_memory_is_asked_for_on_every_device():
    """The attribute belongs to a device: what asks for it once per process leaves the others with 48 KB.  One function
    keeps the record, a bit per device, and nothing else sets the attribute."""
    owners = []
    for path in glob.glob(os.path.join(KERNELS, "*.cu")) + glob.glob(os.path.join(KERNELS, "*.h")) + glob.glob(os.path.join(KERNELS, "*.cuh")):
        with open(path) as f:
            text = f.read()
        if "cudaFuncAttributeMaxDynamicSharedMemorySize" in text:
            owners.append(os.path.basename(path))
            assert "call_once" not in text, path
    assert owners == ["tcgen05_host.h"]


@pytest.mark.parametrize("make,patch,message", [
    # strides of dq, dk, dv and o are words 6 + 3 * (5, 6, 7, 3) of the payload: batch, head, row
    ("B.attention('a', 2, 2, 1, 8, 8, 64)", "put(17, 56)", "the rows of an output overlap"),
    ("B.attention('a', 2, 2, 1, 8, 8, 64)", "put(15, 512)", "the rows of an output overlap"),
    ("B.attention_bwd('a', 2, 2, 1, 8, 8, 64)", "put(23, 8)", "the rows of an output overlap"),
    ("B.attention_bwd('a', 2, 2, 1, 8, 8, 64)", "put(26, 32)", "the rows of an output overlap"),
    ("B.attention_bwd('a', 2, 2, 1, 8, 8, 64)", "put(27, 64)", "the rows of an output overlap"),
    ("B.attention_bwd('a', 2, 2, 1, 8, 8, 64)", "put(15, 512), put(17, 56)", None),   # O is only read
    ("B.attention('a', 1, 2, 2, 1, 8, 64, layout='tokens')", "put(15, 0), put(17, 0)", None),  # of extents of 1
    ("B.attention_bwd('a', 1, 1, 1, 1 << 30, 8, 64)", "put(21, 1 << 37), put(23, 1 << 37)", None),
    ("B.rotary('a', 5, 2, 64, [1.0])", "put(6, 100)", "the rows of Y overlap"),
    ("B.rotary('a', 5, 2, 64, [1.0])", "put(7, 63)", "the rows of Y overlap"),
    ("B.rotary('a', 5, 2, 64, [1.0])", "put(7, 0)", "the rows of Y overlap"),
    ("B.rotary('a', 5, 2, 64, [1.0])", "put(4, 0), put(5, 0)", None),                 # X may be broadcast
    ("B.rotary('a', 5, 2, 64, [1.0])", "put(6, 64), put(7, 320)", None),              # heads outside
    ("B.rotary('a', 5, 2, 64, [1.0])", "put(3, 5)", "rot_dims is even"),
    ("B.rotary('a', 5, 2, 64, [1.0])", "put(2, 513)", "512 dimensions"),
])
def test_problems_the_builders_refuse_are_refused_by_the_library(make, patch, message):
    """Descriptors of another program: the library makes the checks itself, before a launch."""
    text = ("import struct\nfrom __graft_entry__ import load_package\npkg = load_package()\nB, rt = pkg.blob, pkg.runtime\n"
            "d = %s\n"
            "def put(word, value):\n    d.payload = d.payload[:8 * word] + struct.pack('<q', value) + d.payload[8 * word + 8:]\n"
            "%s\nblob = B.Blob([d])\nk = rt.gpuKernelGet(None, rt.gpuModuleLoad(None, blob.address, blob.size), b'a')\n"
            "rt.imexKernelWorkspaceBytes(k)\n" % (make, patch))
    r = subprocess.run([sys.executable, "-c", text], cwd=ROOT, capture_output=True, text=True, timeout=300)
    if message is None:
        assert r.returncode == 0, r.stdout + r.stderr
    else:
        assert r.returncode == -6 and message in r.stdout, r.stdout + r.stderr


def test_equal_descriptors_share_a_kernel_handle():
    """In a session; descriptors that differ in anything have handles of their own."""
    s = object.__new__(pkg.Session)   # no stream: loading a module needs none
    s.stream, s._kernels = None, {}
    attention = lambda **kw: B.attention("a", 1, 2, 2, kw.pop("n_q", 8), 8, 64, **kw)  # noqa: E731
    desc = attention()
    first, kept = s.kernel(desc), len(B._KEEP)
    assert s.kernel(desc) == first and s.kernel(attention()) == first and len(B._KEEP) == kept
    others = [attention(n_q=9), attention(causal=True), attention(sm_scale=0.5), attention(dtype=B.F16),
              B.attention_bwd("a", 1, 2, 2, 8, 8, 64), B.gated_ffn("a", 3, 8, 8), B.gated_ffn("a", 4, 8, 8),
              B.rotary("a", 3, 1, 64, [1.0]), B.rotary("a", 3, 1, 64, [0.5]), B.gemm("a", 8, 8, 8, B.BF16), B.gemm("b", 8, 8, 8, B.BF16)]
    handles = [s.kernel(d) for d in others]
    assert len(set(handles + [first])) == len(others) + 1
    assert [s.kernel(d) for d in others] == handles
    assert rt.imexKernelWorkspaceBytes(handles[4]) > 0
