"""AdamW in captured graphs: each replay is a step of its own, whatever is taken eagerly before, between
and after, with the rate that is set when it runs."""
import pytest
import torch

from conftest import import_package
from test_adamw import HYPER, tensors

import_package()
from eps_b200 import EpsError, INVALID_ARGUMENT, dense  # noqa: E402

gpu = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16
SIZES = (5000, 77, 256)


def pair(bits, master, dtype=F32):
    """Two optimizers of equal parameters that read the same gradients."""
    params, grads = tensors(1, SIZES, 0.1, dtype), tensors(2, SIZES, 1e-2, dtype)
    other = [p.clone() for p in params]
    how = dict(state_bits=bits, master=master, seed=9, **HYPER)
    return dense.AdamW(params, grads, **how), dense.AdamW(other, grads, **how), grads


def captured(opt, **more):
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step(**more)
    return graph


def equal(a, b):
    for p, q in zip(a.parameters, b.parameters):
        assert torch.equal(p, q)
    for name in ("first", "second", "first_scale", "second_scale", "master"):
        x, y = getattr(a, name), getattr(b, name)
        assert (x is None) == (y is None) and (x is None or torch.equal(x.view(torch.uint8), y.view(torch.uint8)))
    assert a.steps == b.steps


@gpu
@pytest.mark.parametrize("bits,master,dtype", [(32, False, F32), (8, False, F32), (8, True, BF16), (32, True, BF16)])
@pytest.mark.parametrize("before", [0, 3])
def test_each_replay_is_a_step(bits, master, dtype, before):
    a, b, grads = pair(bits, master, dtype)
    for _ in range(before):
        a.step()
        b.step()
    graph = captured(a)
    equal(a, b)                     # capturing takes no step
    for k in range(5):
        for g in grads:
            g.mul_(-0.7)
        graph.replay()
        b.step()
    equal(a, b)
    a.step()                        # eagerly behind the replays
    b.step()
    graph.replay()
    b.step()
    equal(a, b)


@gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_replays_follow_the_learning_rate_and_a_loaded_state(bits):
    a, b, _ = pair(bits, False)
    start = {k: v.clone() if torch.is_tensor(v) else v for k, v in a.state().items()}
    a.learning_rate = b.learning_rate = 4e-3
    graph = captured(a)
    for rate in (4e-3, 1e-3, 0.0, 5e-3):
        a.learning_rate = b.learning_rate = rate
        assert a.learning_rate == rate
        graph.replay()
        b.step()
        equal(a, b)
    for opt in (a, b):
        opt.load_state(**{**start, "steps": 40})
    assert a.steps == 40
    graph.replay()
    b.step()
    equal(a, b)


@gpu
def test_two_graphs_scale_and_skip():
    a, b, grads = pair(8, False)
    scale, skip = torch.tensor(0.5, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda")
    plain, scaled = captured(a), captured(a, gradient_scale=scale, skip=skip)
    for k in range(6):
        skip.fill_(k == 3)
        if k % 2:
            scaled.replay()
            b.step(gradient_scale=scale, skip=skip)
        else:
            plain.replay()
            b.step()
    equal(a, b)


@gpu
def test_a_graph_keeps_what_it_reads():
    """Buffers bound after a capture leave the captured step with its own."""
    a, b, grads = pair(32, False)
    graph = captured(a)
    first = [g.clone() for g in grads]
    a.bind([g * 2 for g in grads])
    del grads
    junk = [torch.full((1 << 12,), 255, dtype=torch.uint8, device="cuda") for _ in range(64)]
    graph.replay()
    b.step(first)
    equal(a, b)
    assert len(junk) == 64


@gpu
def test_rates_are_refused_before_they_are_used():
    a, _, _ = pair(32, False)
    captured(a)
    for rate in (-1.0, float("nan"), float("inf")):
        with pytest.raises(EpsError) as e:
            a.learning_rate = rate
        assert e.value.code == INVALID_ARGUMENT


def test_the_clock_is_laid_out_as_declared_and_needed(tmp_path):
    import ctypes as C
    import os
    import subprocess

    import eps_b200
    from conftest import ROOT
    from test_dense_abi import A, LIB, adamw, refused
    names = [f[0] for f in dense.AdamWClock._fields_]
    src = tmp_path / "s.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "eps_b200_dense.h"\nint main(void){printf("%zu", sizeof(EpsB200AdamWClock));'
                   + "".join(f'printf(" %zu", offsetof(EpsB200AdamWClock, {n}));' for n in names) + "return 0;}")
    subprocess.check_call(["gcc", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(tmp_path / "s")])
    got = [int(v) for v in subprocess.check_output([str(tmp_path / "s")]).split()]
    assert got == [C.sizeof(dense.AdamWClock)] + [getattr(dense.AdamWClock, n).offset for n in names]
    for clock in (None, A + 4):
        assert refused(LIB.eps_b200_adamw_counted, adamw(), A, 1, 1, clock, None) == eps_b200.INVALID_ARGUMENT
    assert refused(LIB.eps_b200_adamw_counted, adamw(step=0), A, 1, 1, A, None) == eps_b200.INVALID_ARGUMENT
