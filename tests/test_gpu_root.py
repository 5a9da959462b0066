"""The square root of the AdamW step (csrc/root.cuh) against CUDA's sqrtf and the rounded root in 64
bits, on every float it is used for.  The codes of 8-bit moments follow from it bit by bit."""
import ctypes
import os
import shutil
import subprocess

import pytest

pytestmark = pytest.mark.gpu

HERE = os.path.dirname(os.path.abspath(__file__))


def test_root_is_sqrtf_on_its_whole_range(tmp_path):
    from arboretum_b200 import build
    nvcc = shutil.which(build.NVCC) or "/usr/local/cuda/bin/nvcc"
    lib = str(tmp_path / "root_check.so")
    flags = [f for f in build.FLAGS if f not in ("-Xptxas", "-v")]
    subprocess.run([nvcc] + flags + ["-shared", "-I", build.CSRC, os.path.join(HERE, "root_check.cu"), "-o", lib], check=True)
    count = (ctypes.c_ulonglong * 2)()
    assert ctypes.CDLL(lib).check_roots(count) == 0
    assert count[0] == 0x7E800000 - 0x0D800000 + 1  # 2^-100 .. 2^126, and no others: negative ones, infinities, NaN
    assert count[1] == 0
