"""A projection asked for where there is no GPU: an error code, whatever the size."""

import os
import subprocess
import sys

import pytest

from conftest import PKG_DIR

SCRIPT = """
import ctypes, sys
sys.path.insert(0, sys.argv[1])
from sgl_glm53_ascend_ops import abi
buf = (ctypes.c_uint8 * 4096)()
at = (ctypes.addressof(buf) + 255) // 256 * 256
a = abi.KdaLinearArgs(x=at, x_row_stride=64, weight=at, weight_row_stride=64, out=at, out_row_stride=int(sys.argv[3]),
                      num_tokens=int(sys.argv[2]), in_features=64, out_features=int(sys.argv[3]))
print(abi.lib().kda_linear_launch(ctypes.byref(a), None, 0, None))
"""


@pytest.mark.parametrize("T,N", [(1, 8), (64, 512), (65, 128), (8256, 4096)])
def test_launch_without_a_gpu_returns_an_error(T, N):
    """In a process that sees no device, so that nothing can be launched."""
    got = subprocess.run([sys.executable, "-c", SCRIPT, str(PKG_DIR), str(T), str(N)], capture_output=True, text=True,
                         env={**os.environ, "CUDA_VISIBLE_DEVICES": ""}, timeout=300)
    assert got.returncode == 0, f"ended by signal {-got.returncode}"
    assert int(got.stdout) == 5    # KDA_ERR_LAUNCH
