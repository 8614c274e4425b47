"""Tensors that a user made on one stream and gave to the dense operators on another: dropped there, their memory is not
handed out on the first before the call that uses them is through."""
import pytest
import torch

from conftest import import_package
from test_dense_streams import handed_out, place

import_package()
from eps_b200 import dense  # noqa: E402

gpu = pytest.mark.gpu


def norm(given):
    n = dense.GradientNorm(given)
    return lambda: n.clip(0.5)


def gradients(given):
    opt = dense.AdamW([torch.ones_like(g) for g in given], given)
    return opt.step


def parameters(given):
    opt = dense.AdamW(given, [torch.ones_like(g) for g in given])
    return opt.step


def rebound(given):
    opt = dense.AdamW([torch.ones_like(g) for g in given])
    opt.bind(given)                  # waits for the stream, so not in the call that is held up
    return opt.step


def scales(given):
    scale, bias = given
    layer = dense.QuantizedExperts(torch.ones(len(scale), 64, dtype=torch.int8, device="cuda"), scale, bias)
    x = torch.ones(4, 64, device="cuda")
    return lambda: layer.product(x)


@gpu
@pytest.mark.parametrize("make", [norm, gradients, parameters, rebound, scales])
def test_given_tensors_outlive_the_call_on_another_stream(make):
    make([torch.ones(70000, device="cuda"), torch.ones(70000, device="cuda")])()      # loads the kernels
    given = [torch.ones(70000, device="cuda"), torch.ones(70000, device="cuda")]
    old = place(*given)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    torch.cuda.synchronize()
    with torch.cuda.stream(s):
        call = make(given)                       # bound on the stream that calls
        torch.cuda._sleep(1_000_000_000)
        call()
        done = torch.cuda.Event()
        done.record()
    del call, given
    assert not handed_out(old, done)
    done.synchronize()
