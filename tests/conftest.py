import os
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
PKG = os.path.join(ROOT, "xhy-flash-attention_amd")
for p in (ROOT, PKG):
    if p not in sys.path:
        sys.path.insert(0, p)
# the CPU emulator's kernels start from NaN registers and 0xff LDS bytes (tools/asm_emu.py): a read
# of state the kernel never wrote shows up as NaN, as it would on the GPU
os.environ.setdefault("FA_EMU_POISON", "1")


def pytest_configure(config):
    config.addinivalue_line("markers", "gpu: needs an MI355X (gfx950) GPU")


# Tests that stay off the GPU, with the reason.
SKIPPED = {
    "test_launch_gpu.py::test_graph_capture_varlen_fwd_bwd_bitwise":
        "its replay once faulted the GPU in the forward kernel (an address beyond the legal ones) and the cause "
        "is not known; the library refuses to capture such a launch (test_capture_refused_gpu.py)",
}


def pytest_collection_modifyitems(items):
    for item in items:
        for name, reason in SKIPPED.items():
            if item.nodeid.endswith(name):
                item.add_marker(pytest.mark.skip(reason=reason))
