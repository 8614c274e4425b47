"""The reciprocals and roots that the ranking and the 8-bit moments are defined by: those of the CUDA library for
every float that they take."""
import os
import shutil
import subprocess

import pytest

from conftest import PKG_DIR, ROOT

gpu = pytest.mark.gpu


@gpu
def test_reciprocals_and_roots_are_the_librarys(tmp_path):
    nvcc = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    exe = str(tmp_path / "exact_rounding")
    subprocess.check_call([nvcc, "-gencode", "arch=compute_100a,code=sm_100a", "-O3", "-std=c++17", "--fmad=false", "-I", os.path.join(PKG_DIR, "csrc"),
                           "-I", os.path.join(ROOT, "include"), os.path.join(ROOT, "tests", "exact_rounding.cu"), "-o", exe])
    out = subprocess.run([exe], capture_output=True, text=True, timeout=120)
    assert out.returncode == 0 and out.stdout.split() == ["0", "0"], out.stdout + out.stderr
