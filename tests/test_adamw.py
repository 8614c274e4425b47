"""AdamW against 64 bits: uneven tensors, types, master copies, 8-bit moments and their rounding."""
import math

import pytest
import torch

import dense_reference as ref
from conftest import import_package

import_package()
from eps_b200 import EpsError, INVALID_ARGUMENT, dense  # noqa: E402

gpu = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
SIZES = (1, 3, 255, 256, 257, 4095, 4096, 4097, 10000, 0, 5)
HYPER = dict(learning_rate=2e-3, beta1=0.9, beta2=0.98, epsilon=1e-8, weight_decay=0.05)


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def tensors(seed, sizes, scale=1.0, dtype=F32, shift=0):
    g = gen(seed)
    out = []
    for n in sizes:
        room = torch.zeros(n + shift, dtype=dtype, device="cuda")
        room[shift:] = (torch.randn(n, generator=g, device="cuda") * scale).to(dtype)
        out.append(room[shift:])
    return out


class Plain:
    """The step in 64 bits."""

    def __init__(self, values):
        self.p = [v.double().clone() for v in values]
        self.m = [torch.zeros_like(v) for v in self.p]
        self.v = [torch.zeros_like(v) for v in self.p]
        self.t = 0

    def step(self, grads, learning_rate, beta1, beta2, epsilon, weight_decay, scale=1.0):
        self.t += 1
        for i, g in enumerate(grads):
            g = g.double() * scale
            self.m[i] = beta1 * self.m[i] + (1 - beta1) * g
            self.v[i] = beta2 * self.v[i] + (1 - beta2) * g * g
            up = self.m[i] / (1 - beta1 ** self.t) / (torch.sqrt(self.v[i] / (1 - beta2 ** self.t)) + epsilon)
            self.p[i] = self.p[i] - learning_rate * (up + weight_decay * self.p[i])


def parts(flat, opt):
    return [flat[a:a + p.numel()] for p, a in zip(opt.parameters, opt.starts)]


@gpu
@pytest.mark.parametrize("dtype,grad,master", [(F32, F32, False), (BF16, BF16, True), (BF16, F32, True), (F16, F16, True), (F16, F32, False),
                                               (BF16, BF16, False)])
@pytest.mark.parametrize("shift", [0, 1])
def test_steps(dtype, grad, master, shift):
    params = tensors(1, SIZES, 0.1, dtype, shift)
    plain = Plain(params)
    opt = dense.AdamW(params, state_bits=32, master=master, **HYPER)
    assert opt.parameters[0].data_ptr() == params[0].data_ptr()
    for k in range(4):
        grads = tensors(10 + k, SIZES, 1e-2, grad, shift)
        before = [p.double().clone() for p in params]
        plain.step(grads, **HYPER)
        opt.step(grads)
        if dtype != F32 and not master:      # what a step starts from is the rounded parameter
            step = Plain(before)
            step.m, step.v, step.t = [m.clone() for m in plain.m], [v.clone() for v in plain.v], plain.t
            up = [m / (1 - 0.9 ** step.t) / (torch.sqrt(v / (1 - 0.98 ** step.t)) + 1e-8) for m, v in zip(plain.m, plain.v)]
            plain.p = [b - 2e-3 * (u + 0.05 * b) for b, u in zip(before, up)]
        size = lambda v: v.abs() + 0.02         # a value and its steps  # noqa: E731
        for have, want in zip(params, plain.p):
            ref.close(have, want, size(want))
        if master:
            for have, want in zip(parts(opt.master, opt), plain.p):
                ref.close(have, want, size(want))
        for have, want in zip(parts(opt.first, opt), plain.m):
            ref.close(have, want, 0.1)
        for have, want in zip(parts(opt.second, opt), plain.v):
            ref.close(have, want, want.abs())
    assert opt.steps == 4
    pad = torch.ones_like(opt.first, dtype=torch.bool)
    for p, a in zip(opt.parameters, opt.starts):
        pad[a:a + p.numel()] = False
    assert not opt.first[pad].any() and not opt.second[pad].any()


@gpu
def test_neighbours_are_untouched():
    room = torch.full((5000,), 7.0, device="cuda")
    part = room[1001:3333]
    opt = dense.AdamW([part], [torch.ones_like(part)], learning_rate=0.5)
    opt.step()
    assert bool((room[:1001] == 7).all()) and bool((room[3333:] == 7).all()) and bool((part < 7).all())


@gpu
def test_gradient_scale_skip_and_learning_rate():
    params, grads = tensors(1, (300, 9)), tensors(2, (300, 9))
    opt = dense.AdamW(params, grads, **HYPER)
    plain = Plain(params)
    before = [p.clone() for p in params]
    opt.step(skip=torch.ones(1, dtype=torch.int32, device="cuda"))
    assert all(torch.equal(a, b) for a, b in zip(params, before)) and not opt.first.any() and opt.steps == 1
    plain.t = 1
    opt.learning_rate = 1e-2
    opt.step(gradient_scale=torch.tensor(0.25, device="cuda"), skip=torch.zeros((), dtype=torch.int32, device="cuda"))
    plain.step(grads, **{**HYPER, "learning_rate": 1e-2}, scale=0.25)
    for have, want in zip(params, plain.p):
        ref.close(have, want, want.abs() + 0.05)
    opt.learning_rate = 0.0
    before = [p.clone() for p in params]
    opt.step()
    assert all(torch.equal(a, b) for a, b in zip(params, before))


@gpu
def test_bound_buffers_and_state():
    params, grads = tensors(1, (700, 40)), tensors(2, (700, 40))
    other = [p.clone() for p in params]
    a = dense.AdamW(params, grads, state_bits=8, **HYPER)
    a.step()
    b = dense.AdamW(other, grads, state_bits=8, **HYPER)
    for p, q in zip(params, other):
        q.copy_(p)
    b.load_state(**{k: v.clone() if torch.is_tensor(v) else v for k, v in a.state().items()})
    for g in grads:
        g.mul_(-0.5)           # the buffers are read at the step
    a.step()
    b.step([g.clone() for g in grads])
    assert all(torch.equal(p, q) for p, q in zip(params, other))
    assert all(torch.equal(x.view(torch.uint8), y.view(torch.uint8)) for x, y in ((a.first, b.first), (a.second, b.second)))


def decoded(codes, scale):
    return (codes.float().view(-1, 256) * scale[:, None]).view(-1).double()


@gpu
@pytest.mark.parametrize("dtype,master", [(F32, False), (BF16, True), (BF16, False), (F16, True)])
def test_8bit_step(dtype, master):
    """One step from given 8-bit moments: the parameters are those of the decoded moments, the new codes
    are neighbours of the new moments (m the nearest)."""
    params = tensors(1, SIZES, 0.1, dtype)
    opt = dense.AdamW(params, state_bits=8, master=master, seed=5, **HYPER)
    for k in range(3):
        grads = tensors(20 + k, SIZES, 1e-2, dtype)
        m0, r0 = decoded(opt.first, opt.first_scale), decoded(opt.second, opt.second_scale)
        plain = Plain(parts(opt.master, opt) if master else params)
        plain.m, plain.v, plain.t = parts(m0, opt), [r * r for r in parts(r0, opt)], k
        plain.step(grads, **HYPER)
        opt.step(grads)
        for have, want in zip(params, plain.p):
            ref.close(have, want, want.abs() + 0.02)
        for values, codes, scale in ((plain.m, opt.first, opt.first_scale), ([v.sqrt() for v in plain.v], opt.second, opt.second_scale)):
            flat = torch.zeros(codes.numel(), dtype=torch.float64, device="cuda")
            for x, a in zip(values, opt.starts):
                flat[a:a + x.numel()] = x
            top = flat.view(-1, 256).abs().amax(-1)
            ref.close(scale, top / 448, top / 448)
            got = decoded(codes, scale)
            unit = torch.maximum(2.0 ** (torch.floor(torch.log2(flat.abs().clamp(min=1e-30) / scale.double().clamp(min=1e-30).repeat_interleave(256))) - 3),
                                 torch.tensor(2.0 ** -9, device="cuda")) * scale.double().repeat_interleave(256)
            # half a unit or a whole one, and the float32 roundings of the moment's own two terms
            terms = torch.zeros_like(flat)
            for x, old, a, g in zip(values, parts(m0 if values is plain.m else r0, opt), opt.starts, grads):
                terms[a:a + x.numel()] = old.abs() + g.double().abs()
            bound = unit * (0.5 if values is plain.m else 1.0)
            assert bool(((got - flat).abs() <= bound * (1 + 1e-4) + 4 * 2.0 ** -24 * terms).all())
            assert bool((got[flat == 0] == 0).all())
        assert bool((decoded(opt.second, opt.second_scale)[torch.cat([torch.nn.functional.pad(v, (0, -v.numel() % 256)) for v in plain.v]) > 0] > 0).all())


def mixed(h):
    h = ((h ^ (h >> 16)) * 0x85EBCA6B) & 0xFFFFFFFF
    h = ((h ^ (h >> 13)) * 0xC2B2AE35) & 0xFFFFFFFF
    return h ^ (h >> 16)


@gpu
def test_8bit_codes_are_those_of_the_formula():
    """The codes and scales of several steps bit for bit, from a float32 restatement whose every operation
    is rounded by itself."""
    params = tensors(1, SIZES, 0.1)
    opt = dense.AdamW(params, state_bits=8, seed=77, **HYPER)
    n = opt.first.numel()
    m, r = torch.zeros(n, device="cuda"), torch.zeros(n, device="cuda")
    for k in range(5):
        grads = tensors(40 + k, SIZES, 1e-2)
        opt.step(grads)
        g = torch.zeros(n, device="cuda")
        for x, a in zip(grads, opt.starts):
            g[a:a + x.numel()] = x
        m = 0.9 * m + (1 - 0.9) * g
        root = torch.sqrt(0.98 * (r * r) + (1 - 0.98) * g * g)
        key = mixed(torch.tensor(77, device="cuda") ^ mixed(torch.tensor(k + 1, device="cuda")))
        h = mixed((torch.arange(n // 2, device="cuda") * 0x9E3779B1 + key) & 0xFFFFFFFF)
        u = torch.stack([h & 0xFFFF, h >> 16], -1).view(-1)
        out = []
        for v in (m, root):
            scale = v.view(-1, 256).abs().amax(-1) * torch.tensor(1 / 448, device="cuda")
            x = (v.view(-1, 256) * torch.where(scale == 0, 0.0, 1 / scale)[:, None]).view(-1)
            out.append((x, scale))
        (xm, sm), (xr, sr) = out
        coarse = ((xr.view(torch.int32) + (u.int() << 4)) & -0x100000).view(torch.float32)
        fine = torch.floor(xr * 512 + u.float() / 65536) / 512
        xr = torch.where(xr > 0, torch.where(xr < 2.0 ** -6, fine, coarse).clamp(2.0 ** -9, 448), xr)
        cm, cr = xm.clamp(-448, 448).to(torch.float8_e4m3fn), xr.to(torch.float8_e4m3fn)
        assert torch.equal(opt.first_scale, sm) and torch.equal(opt.second_scale, sr)
        assert torch.equal(opt.first.view(torch.uint8), cm.view(torch.uint8))
        assert torch.equal(opt.second.view(torch.uint8), cr.view(torch.uint8))
        m = (cm.float().view(-1, 256) * sm[:, None]).view(-1)
        r = (cr.float().view(-1, 256) * sr[:, None]).view(-1)


@gpu
def test_8bit_roots_are_right_on_average():
    """The same moments rounded at many places: their mean is the value, although a step moves it by far
    less than a unit; and a long run follows the 64-bit moments."""
    n = 1 << 20
    p, g = torch.zeros(n, device="cuda"), torch.zeros(n, device="cuda")
    opt = dense.AdamW([p], [g], state_bits=8, beta2=0.999, learning_rate=0.0, weight_decay=0.0)
    for value in (0.3, 0.00017):                # a normal value of e4m3, and one below its normal range
        g[:] = value
        g[::256] = 1.0                          # sets the scale
        opt.load_state(0, first=torch.zeros_like(opt.first), second=torch.zeros_like(opt.second),
                       first_scale=torch.zeros_like(opt.first_scale), second_scale=torch.zeros_like(opt.second_scale))
        opt.step()
        keep = torch.arange(n, device="cuda") % 256 != 0
        got = decoded(opt.second, opt.second_scale)[keep]
        want = math.sqrt(1 - 0.999) * value
        unit = max(2.0 ** (math.floor(math.log2(value * 448)) - 3), 2.0 ** -9) / 448 * math.sqrt(1 - 0.999)
        # the mean of a million roundings, each within a unit: five deviations of at most unit / 2, and 2^-16 of a unit
        assert abs(got.mean().item() - want) <= unit * (5 * 0.5 / math.sqrt(n) + 2.0 ** -16) + 1e-6 * want
    v = torch.zeros(n, dtype=torch.float64, device="cuda")
    opt.load_state(0, first=torch.zeros_like(opt.first), second=torch.zeros_like(opt.second),
                   first_scale=torch.zeros_like(opt.first_scale), second_scale=torch.zeros_like(opt.second_scale))
    r = gen(3)
    size = torch.exp(torch.randn(n, generator=r, device="cuda"))
    steps = 400
    for _ in range(steps):
        g.copy_(torch.randn(n, generator=r, device="cuda") * size)
        v = 0.999 * v + 0.001 * g.double() ** 2
        opt.step()
    got = decoded(opt.second, opt.second_scale) ** 2
    # each root carries a rounding of up to a unit (1/8) of variance at most (1/16)^2 a step, damped by
    # 0.999 a step: (1/256) * 400 in the worst case for one element, and none in the mean beyond that
    # variance's own square, which adds to v at most (1/256) a step and is what the bound below holds
    ratio = (got.mean() / v.mean()).item()
    assert 0.99 <= ratio <= 1.0 + steps / 256


@gpu
def test_8bit_learns_like_32bit():
    """Least squares by both, from the same start: the same loss to a tenth."""
    r = gen(7)
    a, b = torch.randn(512, 64, generator=r, device="cuda"), torch.randn(512, 32, generator=r, device="cuda")
    start, loss = torch.randn(64, 32, generator=r, device="cuda"), {}
    for bits in (32, 8):
        w = start.clone()
        g = torch.empty_like(w)
        opt = dense.AdamW([w], [g], state_bits=bits, learning_rate=1e-2, weight_decay=0.0)
        for _ in range(400):
            g.copy_(a.T @ (a @ w - b) / 512)
            opt.step()
        loss[bits] = ((a @ w - b) ** 2).mean().item()
    assert abs(loss[8] - loss[32]) <= 0.1 * loss[32]


@gpu
def test_zero_and_bad_gradients():
    for bits in (32, 8):
        p = [torch.ones(1000, device="cuda"), torch.ones(256, device="cuda")]
        g = [torch.zeros(1000, device="cuda"), torch.ones(256, device="cuda")]
        opt = dense.AdamW(p, g, state_bits=bits, weight_decay=0.0)
        opt.step()
        assert bool((p[0] == 1).all()) and bool((p[1] < 1).all())
        g[0][600] = math.nan
        opt.step()
        assert p[0][600].isnan() and int(p[0].isnan().sum()) == 1 and not p[1].isnan().any()
        g[0][600] = 0
        opt.step()
        # 8-bit moments share their scale: what is not a number spreads in its block of 256, not further
        assert int(p[0].isnan().sum()) == (1 if bits == 32 else 256) and not p[1].isnan().any()


@gpu
def test_stream_and_graph():
    params, grads = tensors(1, (5000, 77)), tensors(2, (5000, 77))
    other = [p.clone() for p in params]
    a, b = dense.AdamW(params, grads, **HYPER), dense.AdamW(other, grads, **HYPER)
    a.step()
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        copy = [torch.empty_like(g) for g in grads]
        torch.cuda._sleep(20_000_000)
        for c, g in zip(copy, grads):
            c.copy_(g)
        b.step(copy)
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(params, other))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        a.step()
    graph.replay()
    b.step(grads)
    assert all(torch.equal(p, q) for p, q in zip(params, other))


@gpu
def test_refusals():
    p, g = [torch.ones(8, 4, device="cuda")], [torch.ones(8, 4, device="cuda")]
    h = [p[0].to(BF16)]
    bad = [lambda: dense.AdamW([]), lambda: dense.AdamW([p[0].cpu()]), lambda: dense.AdamW([p[0].double()]), lambda: dense.AdamW([p[0].t()]),
           lambda: dense.AdamW([p[0], h[0]]), lambda: dense.AdamW(p, state_bits=16), lambda: dense.AdamW(p, master=True),
           lambda: dense.AdamW(p, []), lambda: dense.AdamW(p, [g[0].to(BF16)]), lambda: dense.AdamW(h, [g[0].to(F16)]), lambda: dense.AdamW(p, [g[0][:4]]),
           lambda: dense.AdamW(p, [g[0].cpu()]), lambda: dense.AdamW(p).step(), lambda: dense.AdamW(p, g, learning_rate=-1.0).step(),
           lambda: dense.AdamW(p, g, learning_rate=math.nan).step(), lambda: dense.AdamW(p, g, beta1=1.0).step(), lambda: dense.AdamW(p, g, beta2=-0.1).step(),
           lambda: dense.AdamW(p, g, epsilon=0.0).step(), lambda: dense.AdamW(p, g, weight_decay=-1.0).step(),
           lambda: dense.AdamW(p, g).step(gradient_scale=torch.ones(2, device="cuda")), lambda: dense.AdamW(p, g).step(skip=torch.zeros(1, device="cuda")),
           lambda: dense.AdamW(p, g).load_state(0, first=p[0]), lambda: dense.AdamW(p, g).load_state(0, first=p[0], second=p[0])]
    for call in bad:
        with pytest.raises(EpsError) as e:
            call()
        assert e.value.code == INVALID_ARGUMENT
    assert bool((p[0] == 1).all())
