"""What the dense operators hold between calls, dropped on one stream while a call on another still reads it:
its memory is not handed out before that call is through."""
import pytest
import torch

from conftest import import_package

import_package()
from eps_b200 import dense  # noqa: E402

gpu = pytest.mark.gpu


def held_up(call):
    """`call` on a stream of its own, behind a long wait; the event that ends it."""
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        torch.cuda._sleep(1_000_000_000)
        call()
        done = torch.cuda.Event()
        done.record()
    return done


def handed_out(tensors, done):
    """Whether new tensors of these sizes take the memory of the old ones, given as (address, bytes),
    before the event has come."""
    fresh = [torch.empty(n, dtype=torch.uint8, device="cuda") for _, n in tensors for _ in range(4)]
    places = {t.data_ptr() for t in fresh}
    assert not done.query()            # else nothing is shown
    return any(a in places for a, _ in tensors)


def place(*tensors):
    return [(t.data_ptr(), t.numel() * t.element_size()) for t in tensors]


@gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_a_plan_outlives_the_step_that_reads_it(bits):
    params = [torch.ones(40000, device="cuda"), torch.ones(70, device="cuda")]
    start = [p.clone() for p in params]
    grads = [torch.full_like(p, 0.5) for p in params]
    opt = dense.AdamW(params, grads, state_bits=bits, learning_rate=0.125, weight_decay=0.0)
    opt.step()                                     # loads the kernel
    torch.cuda.synchronize()
    old = place(opt._bound[1], *grads)
    done = held_up(opt.step)
    del grads
    opt.bind([torch.ones_like(p) for p in params])
    assert not handed_out(old, done)
    done.synchronize()
    torch.cuda.synchronize()
    for p, q in zip(params, start):                # both steps took the bound gradients
        assert bool(((q - p) - 0.25).abs().max() < 1e-3)


@gpu
def test_moments_outlive_the_step_that_reads_them():
    params = [torch.ones(40000, device="cuda")]
    opt = dense.AdamW(params, [torch.ones_like(params[0])], state_bits=8)
    opt.step()
    torch.cuda.synchronize()
    old = place(opt.first, opt.second, opt.first_scale, opt.second_scale)
    done = held_up(opt.step)
    del opt
    assert not handed_out(old, done)
    done.synchronize()


@gpu
def test_weights_outlive_the_product_that_reads_them():
    layer = dense.QuantizedExperts.from_weights(torch.randn(2000, 1000, device="cuda"))
    for n in (4, 300):
        x = torch.randn(n, 1000, device="cuda")
        layer.product(x)
    torch.cuda.synchronize()
    old = place(layer.weight, layer.scale)
    done = held_up(lambda: layer.product(x))
    del layer
    assert not handed_out(old, done)
    done.synchronize()
