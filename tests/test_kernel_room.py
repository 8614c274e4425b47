"""A kernel's shared-memory limit under two host threads, on the CPU against a runtime that holds one of
them up (kernel_room.cu, fake_runtime.cpp), and on the GPU with calls of different sizes at once."""
import os
import shutil
import subprocess
import threading

import pytest
import torch

from conftest import PKG_DIR, ROOT, import_package

import_package()
from eps_b200 import dense  # noqa: E402

gpu = pytest.mark.gpu


HERE = os.path.dirname(os.path.abspath(__file__))


def nvcc():
    return shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"


def test_a_smaller_request_does_not_lower_the_limit(tmp_path):
    exe, runtime = str(tmp_path / "kernel_room"), str(tmp_path / "fake_runtime.o")
    toolkit = os.path.dirname(os.path.dirname(os.path.realpath(nvcc())))
    subprocess.check_call(["g++", "-std=c++17", "-I", os.path.join(toolkit, "include"), "-c", os.path.join(HERE, "fake_runtime.cpp"), "-o", runtime])
    subprocess.check_call([nvcc(), "-gencode", "arch=compute_100a,code=sm_100a", "-std=c++17", "-cudart", "none", "-I", os.path.join(PKG_DIR, "csrc"),
                           "-I", os.path.join(ROOT, "include"), os.path.join(HERE, "kernel_room.cu"), runtime, "-o", exe, "-lpthread"])
    out = subprocess.run([exe], capture_output=True, text=True, timeout=60)
    assert out.returncode == 0, f"limits at the large launch and later: {out.stdout}"


@gpu
def test_calls_of_different_sizes_from_two_threads():
    """Products of few rows take shared memory by the inner size: both sizes at once, many times."""
    layers = [dense.QuantizedExperts.from_weights(torch.randn(64, k, device="cuda")) for k in (16000, 160)]
    xs = [torch.randn(8, layer.inner, device="cuda") for layer in layers]
    want = [layer.product(x) for layer, x in zip(layers, xs)]
    torch.cuda.synchronize()
    for dtype in (torch.float32, torch.bfloat16, torch.float16):
        start, failed = threading.Barrier(2), []

        def work(layer, x):
            try:
                start.wait()
                for n in (8, 4, 2, 1) * 20:
                    layer.product(x[:n].to(dtype))
                torch.cuda.current_stream().synchronize()
            except Exception as e:  # noqa: BLE001
                failed.append(e)
        threads = [threading.Thread(target=work, args=a) for a in zip(layers, xs)]
        for t in threads:
            t.start()
        for t in threads:
            t.join()
        assert not failed
    assert all(torch.equal(layer.product(x), w) for layer, x, w in zip(layers, xs, want))
