"""Checks of the attention, gated feed-forward and rotary operators that need no GPU, beyond test_transformer_ops.py."""
import glob
import os

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
