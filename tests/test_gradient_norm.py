"""The norm over many gradients against 64 bits: uneven tensors of mixed types and alignments, the whole range
of a float, clipping in place, what is not finite, and capture together with AdamW."""
import math

import pytest
import torch

import dense_reference as ref
from conftest import import_package

import_package()
from eps_b200 import EpsError, INVALID_ARGUMENT, dense  # noqa: E402

gpu = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
SMALL = (1, 3, 0, 255, 4097, 8200, 31)                        # a single cluster's work (up to 16 spans of 16 KB)
LARGE = (1, 700001, 5, 16384, 131073, 0, 1 << 20, 4095)        # more spans than that
# the sum of squares in groups of eight floats: a few units of 2^-24, half of that in the root; the result rounded once more
NORM = 8 * 2.0 ** -24


def tensors(seed, sizes, dtypes, scale=1.0, shift=0):
    g, out = torch.Generator(device="cuda").manual_seed(seed), []
    for i, n in enumerate(sizes):
        dtype = dtypes[i % len(dtypes)]
        room = torch.zeros(n + shift, dtype=dtype, device="cuda")
        room[shift:] = (torch.randn(n, generator=g, device="cuda") * scale).to(dtype)
        out.append(room[shift:])
    return out


def norm_of(gradients, kind):
    flat = torch.cat([g.double() for g in gradients])
    return float(torch.sqrt((flat * flat).sum()) if kind == "l2" else flat.abs().max())


def near(got, want):
    assert abs(float(got) - want) <= NORM * abs(want), (float(got), want)


@gpu
@pytest.mark.parametrize("sizes", [SMALL, LARGE])
@pytest.mark.parametrize("dtypes", [(F32,), (BF16,), (F16,), (F32, BF16, F16)])
@pytest.mark.parametrize("kind", ["l2", "max"])
@pytest.mark.parametrize("shift", [0, 1])
def test_measure_and_clip(sizes, dtypes, kind, shift):
    grads = tensors(1, sizes, dtypes, 1e-2, shift)
    before = [g.clone() for g in grads]
    n = dense.GradientNorm(grads, kind=kind)
    want = norm_of(grads, kind)
    r = n.measure()
    near(r.norm, want)
    assert float(r.scale) == 1.0 and int(r.skip) == 0
    near(n.measure(want / 3).scale, 1 / 3)
    assert float(n.measure(want * 3).scale) == 1.0
    u = torch.tensor(-0.125, device="cuda")
    r = n.measure(want / 16, gradient_scale=u)
    near(r.norm, want / 8)
    near(r.scale, -0.125 / 2)
    assert all(torch.equal(a, b) for a, b in zip(grads, before))
    r = n.clip(want / 16, gradient_scale=u)
    near(r.scale, -0.125 / 2)
    for a, b in zip(grads, before):      # the factor itself is tested above; each value takes it with one rounding
        assert torch.equal(a, (b.float() * r.scale).to(b.dtype))
    assert float(n.clip(0.0).scale) == 0.0 and not any(g.any() for g in grads)
    r = n.clip(0.0)                       # nothing is left to clip
    assert float(r.norm) == 0.0 and float(r.scale) == 1.0 and int(r.skip) == 0


@gpu
@pytest.mark.parametrize("sizes", [(5000,), (3000000,)])
@pytest.mark.parametrize("size", [1e-44, 1e-38, 1e-30, 1e-14, 1e14, 1e18, 1e30])
def test_whole_range_of_a_float(sizes, size):
    grads = tensors(2, sizes, (F32,), 1.0)
    grads = [g.double().mul(size).float() for g in grads]
    want = norm_of(grads, "l2")
    r = dense.GradientNorm(grads).measure(want / 2)
    got = float(r.norm)
    # a norm below the normal floats is rounded to their spacing
    assert abs(got - want) <= NORM * want + 2.0 ** -150
    near(r.scale, 0.5)


@gpu
def test_small_beside_large():
    grads = [torch.full((100000,), 1e-25, device="cuda"), torch.full((3,), 1e-22, device="cuda"), torch.zeros(70000, device="cuda")]
    near(dense.GradientNorm(grads).measure().norm, norm_of(grads, "l2"))


@gpu
@pytest.mark.parametrize("sizes", [SMALL, LARGE])
@pytest.mark.parametrize("kind", ["l2", "max"])
@pytest.mark.parametrize("value", [math.inf, -math.inf, math.nan])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_not_finite(sizes, kind, value, dtype):
    grads = tensors(3, sizes, (dtype,))
    grads[4][17] = value
    before = [g.clone() for g in grads]
    r = dense.GradientNorm(grads, kind=kind).clip(1.0)
    got = float(r.norm)
    assert math.isnan(got) if math.isnan(value) else got == math.inf
    assert int(r.skip) == 1 and float(r.scale) == 0.0
    for a, b in zip(grads, before):
        assert torch.equal(a.nan_to_num(7.0), b.nan_to_num(7.0))


@gpu
def test_scales_that_are_not_finite():
    grads = [torch.zeros(40, device="cuda")]
    n = dense.GradientNorm(grads)
    for u in (math.inf, math.nan):
        r = n.clip(1.0, gradient_scale=torch.tensor(u, device="cuda"))
        assert int(r.skip) == 1 and float(r.scale) == 0.0 and not grads[0].any()
    r = dense.GradientNorm([torch.full((4,), 3e38, device="cuda")]).measure(1.0)      # over the floats, though its terms are not
    assert float(r.norm) == math.inf and int(r.skip) == 1
    r = dense.GradientNorm([torch.full((4,), 3e38, device="cuda")]).measure(1.0, gradient_scale=torch.tensor(1e-3, device="cuda"))
    near(r.norm, norm_of([torch.full((4,), 3e38, device="cuda")], "l2") * float(torch.tensor(1e-3)))
    assert int(r.skip) == 0


@gpu
def test_neighbours_are_untouched_and_results_repeat():
    room = torch.randn(3000001, device="cuda")
    before = room.clone()
    parts = [room[1:5], room[7:900002], room[900003:3000000]]
    n = dense.GradientNorm(parts)
    first = [float(v) for v in n.measure(1.0)]
    assert all([float(v) for v in n.measure(1.0)] == first for _ in range(5))
    n.clip(1.0)
    for i in (0, 5, 6, 900002, 3000000):
        assert room[i] == before[i]
    near(n.measure().norm, 1.0)


@gpu
def test_elements_beyond_32_bits():
    g = torch.zeros((1 << 32) + 12345, dtype=BF16, device="cuda")
    for at, v in ((0, 3.0), (1 << 31, 4.0), (1 << 32, 12.0), (len(g) - 1, 84.0)):
        g[at] = v
    r = dense.GradientNorm([g]).clip(8.5)
    near(r.norm, math.sqrt(9 + 16 + 144 + 7056))
    near(r.scale, 0.1)
    assert [float(g[i]) for i in (0, 1 << 31, 1 << 32, -1)] == [float(torch.tensor(v * float(r.scale)).bfloat16()) for v in (3.0, 4.0, 12.0, 84.0)]


@gpu
def test_nothing_to_measure():
    r = dense.GradientNorm([torch.empty(0, device="cuda")]).clip(1.0)
    assert float(r.norm) == 0.0 and float(r.scale) == 1.0 and int(r.skip) == 0


@gpu
def test_refusals():
    x = torch.ones(64, device="cuda")
    bad = [lambda: dense.GradientNorm([]), lambda: dense.GradientNorm([x[:40], x[39:]]), lambda: dense.GradientNorm([x, x]),
           lambda: dense.GradientNorm([x[::2]]), lambda: dense.GradientNorm([x.double()]), lambda: dense.GradientNorm([x.cpu()]),
           lambda: dense.GradientNorm([x], kind="l1"), lambda: dense.GradientNorm([x]).measure(-1.0),
           lambda: dense.GradientNorm([x]).clip(math.nan), lambda: dense.GradientNorm([x]).clip(1.0, gradient_scale=x),
           lambda: dense.GradientNorm([x]).clip(None), lambda: dense.GradientNorm([x]).measure(1.0, gradient_scale=x[0].cpu())]
    for call in bad:
        with pytest.raises(EpsError) as e:
            call()
        assert e.value.code == INVALID_ARGUMENT
    dense.GradientNorm([x[:40], x[40:], x[:0], x[10:10]])      # side by side, or without elements


@gpu
@pytest.mark.parametrize("sizes", [(300, 9), (400000, 70)])
def test_clipped_steps_of_adamw_captured(sizes):
    """Measured, then stepped by the measure's factor, in a graph that is replayed: equal to steps with the factor by hand."""
    def make():
        return tensors(5, sizes, (F32,)), tensors(6, sizes, (F32,))
    params, grads = make()
    plain, kept = make()
    opt, n = dense.AdamW(params, grads), dense.GradientNorm(grads)
    other = dense.AdamW(plain, kept)

    def step():
        r = n.measure(0.5)
        opt.step(gradient_scale=r.scale, skip=r.skip)
        return r
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(s):
        step()
        torch.cuda.current_stream().synchronize()
        with torch.cuda.graph(graph, stream=s):
            r = step()
    torch.cuda.current_stream().wait_stream(s)
    other.step(gradient_scale=torch.tensor(0.5 / norm_of(kept, "l2"), device="cuda"))
    for k in range(3):
        for g, h in zip(grads, kept):
            g.mul_(-1.5)
            h.mul_(-1.5)
        if k == 1:
            grads[0][7] = math.inf
        graph.replay()
        if k == 1:
            assert int(r.skip) == 1
            grads[0][7] = kept[0][7]
            other.step(skip=torch.ones(1, dtype=torch.int32, device="cuda"))
        else:
            near(r.norm, norm_of(kept, "l2"))
            other.step(gradient_scale=torch.tensor(0.5 / norm_of(kept, "l2"), device="cuda"))
        for p, q in zip(params, plain):
            # the factors differ by NORM, which a step of 1e-3 hardly shows
            ref.close(p, q.double(), 1 + q.abs().double())


@gpu
def test_two_graphs_and_two_streams():
    """Calls keep no state between them: graphs of one object replay at once, beside a call on another stream."""
    grads = tensors(8, LARGE, (BF16,))
    n = dense.GradientNorm(grads)
    want = float(n.measure(1.0).norm)
    graphs, results, streams = [], [], [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    for s in streams[:2]:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            results.append(n.measure(1.0))
        graphs.append(g)
    for _ in range(20):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        with torch.cuda.stream(streams[2]):
            last = n.measure(1.0)
        torch.cuda.synchronize()
        assert [float(r.norm) for r in (*results, last)] == [want] * 3


@gpu
def test_buffers_outlive_the_call_that_reads_them():
    grads = [torch.ones(3000000, device="cuda")]
    n = dense.GradientNorm(grads)
    n.clip(1.0)
    torch.cuda.synchronize()
    old = [(t.data_ptr(), t.numel() * t.element_size()) for t in (n._bound[1], *grads)]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        torch.cuda._sleep(1_000_000_000)
        n.clip(0.5)
        done = torch.cuda.Event()
        done.record()
    del grads
    n.bind([torch.ones(5, device="cuda")])
    fresh = {torch.empty(b, dtype=torch.uint8, device="cuda").data_ptr() for _, b in old for _ in range(4)}
    assert not done.query()            # else nothing is shown
    assert not any(a in fresh for a, _ in old)
    done.synchronize()
