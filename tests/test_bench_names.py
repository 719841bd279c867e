"""bench.py finds its kernel's counters by name: the library holds a kernel of that name."""
import subprocess

import bench
from irontimber_amd import _lib


def test_decode_kernel_is_in_the_library():
    names = subprocess.run(["nm", "-C", _lib.LIB_PATH], capture_output=True, text=True, check=True).stdout
    assert f"__device_stub__{bench.DECODE_KERNEL}(" in names
