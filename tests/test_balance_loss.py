"""The balance loss against 64 bits: widths, types, scores, padded batches and masked experts, its gradient against
the formula differentiated by torch and against differences, and its place beside the router."""
import math

import pytest
import torch

import dense_reference as ref
from conftest import import_package

import_package()
from eps_b200 import EpsError, INVALID_ARGUMENT, dense  # noqa: E402

gpu = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
SHAPES = [(1, 1, 1), (1, 8, 2), (3, 128, 6), (0, 16, 2), (77, 5, 3), (300, 96, 4), (1001, 250, 8), (513, 64, 32), (900, 12, 1), (40, 1024, 8),
          (700, 1023, 2), (5000, 16, 2), (2000, 256, 8), (300, 520, 3), (300, 261, 3), (9000, 33, 4)]
HOW = [("softmax", True), ("sigmoid", True), ("sigmoid", False)]


def inputs(T, E, k, dtype, seed=1, masked=False, padded=False):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(T, E, generator=g, device="cuda") * 2 + torch.randn(E, generator=g, device="cuda")
    if masked:
        x = x.masked_fill(torch.rand(T, E, generator=g, device="cuda") < 0.2, -math.inf)
        if T > 2:
            x[T // 2] = -math.inf
    chosen = torch.randint(0, E, (T, k), generator=g, device="cuda", dtype=torch.int32)
    chosen[torch.rand(T, k, generator=g, device="cuda") < 0.05] = -1
    chosen[torch.rand(T, k, generator=g, device="cuda") < 0.02] = E
    mask = torch.rand(T, generator=g, device="cuda") < 0.7 if padded else None
    x = x.to(dtype)
    if padded and T > 3:                # what padding holds is not looked at
        x[~mask] = math.nan
    return x, chosen, mask


def shares(x, score, normalise):
    """p in 64 bits, 0 for a row of -inf alone; differentiable."""
    dead = (x == -math.inf).all(-1, keepdim=True)
    live = torch.where(dead, 0.0, x)
    p = torch.softmax(live, -1) if score == "softmax" else torch.sigmoid(live)
    if score == "sigmoid" and normalise:
        p = p / p.sum(-1, keepdim=True)
    return torch.where(dead, 0.0, p)


def plain(x, chosen, mask, score, normalise, weight):
    """(loss, counts, mass, n), differentiable by x"""
    T, E = x.shape
    keep = torch.ones(T, dtype=torch.bool, device="cuda") if mask is None else mask
    k, n = chosen.shape[1], int(keep.sum())
    counts = [0] * E
    for row in chosen[keep].tolist():
        for e in row:
            if 0 <= e < E:
                counts[e] += 1
    counts = torch.tensor(counts, device="cuda")
    mass = shares(torch.where(keep[:, None], x, 0.0), score, normalise)[keep].sum(0)
    loss = weight * E / (k * n * n) * (counts * mass).sum() if n else 0 * mass.sum()
    return loss, counts, mass, n


@gpu
@pytest.mark.parametrize("T,E,k", SHAPES)
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("score,normalise", HOW)
@pytest.mark.parametrize("masked,padded", [(False, False), (True, True)])
def test_loss_and_gradient(T, E, k, dtype, score, normalise, masked, padded):
    x, chosen, mask = inputs(T, E, k, dtype, 1, masked, padded)
    how = dict(score=score, normalise=normalise, mask=mask, weight=0.25)
    got = dense.balance_loss(x, chosen, **how)
    xd = x.double().requires_grad_(True)
    loss, counts, mass, n = plain(xd, chosen, mask, score, normalise, 0.25)
    assert int(got.tokens) == n and torch.equal(got.counts.long(), counts)
    # a share is off by CHAIN at most, and so is their sum (a lane adds few rows)
    ref.close(got.mass, mass.detach(), mass.detach().max() if E else 0)
    ref.close(got.loss, loss.detach(), loss.detach().abs())
    again = dense.balance_loss(x, chosen, **how)
    assert all(torch.equal(a, b) for a, b in zip(got, again))

    # the counts' size in the gradient is what they differ from their mean by, where p adds up to 1
    dloss = torch.tensor(float(max(1, n)), device="cuda")
    want = torch.autograd.grad(loss, xd, dloss.double())[0].nan_to_num(0.0) if n else torch.zeros_like(xd)
    want = torch.where(mask[:, None], want, 0.0) if mask is not None else want
    have = dense.balance_loss_backward(x, got.counts, got.tokens, k, dloss=dloss, **how)
    c = 0.25 * E / (k * max(1, n))
    p = shares(torch.where(torch.isnan(xd), 0.0, xd), score, normalise).detach()
    d = (counts - k * n / E).abs().max() if score == "softmax" or normalise else counts.max()
    size = c * d * p
    ref.close(have, want, size)
    add = torch.randn(T, E, generator=torch.Generator(device="cuda").manual_seed(5), device="cuda").to(dtype)
    have = dense.balance_loss_backward(x, got.counts, got.tokens, k, dloss=dloss, add=add, **how)
    ref.close(have, want + add.double(), size + add.double().abs())


@gpu
@pytest.mark.parametrize("score,normalise", HOW)
def test_gradient_against_differences(score, normalise):
    """The kernel's own gradient against differences of the 64-bit loss."""
    x, chosen, mask = inputs(9, 7, 2, F32, 3, padded=True)
    x = torch.where(mask[:, None], x, 0.0)
    got = dense.balance_loss(x, chosen, score=score, normalise=normalise, mask=mask)
    have = dense.balance_loss_backward(x, got.counts, got.tokens, 2, score=score, normalise=normalise, mask=mask)
    step, want = 2.0 ** -10, torch.zeros(9, 7, dtype=torch.float64, device="cuda")
    for t in range(9):
        for e in range(7):
            up, down = x.double(), x.double()
            up[t, e] += step
            down[t, e] -= step
            want[t, e] = (plain(up, chosen, mask, score, normalise, 1.0)[0] - plain(down, chosen, mask, score, normalise, 1.0)[0]) / (2 * step)
    # a difference is off by step^2 / 6 of the third derivative, which is below the loss's size
    assert float((have.double() - want).abs().max()) <= step ** 2 / 6 * float(plain(x.double(), chosen, mask, score, normalise, 1.0)[0]) + ref.CHAIN


@gpu
def test_unbalanced_costs_more_and_one_expert():
    T, E, k = 640, 8, 1
    even = torch.arange(T, device="cuda", dtype=torch.int32).remainder(E)[:, None].contiguous()
    x = torch.zeros(T, E, device="cuda")
    assert float(dense.balance_loss(x, even).loss) == 1.0                  # equal shares, equal counts
    assert not dense.balance_loss_backward(x, *dense.balance_loss(x, even)[1::2], k).any()
    x[:, 3] = 100.0
    one = torch.full((T, 1), 3, device="cuda", dtype=torch.int32)
    assert float(dense.balance_loss(x, one).loss) == E


@gpu
def test_nothing_counts():
    x, chosen, _ = inputs(50, 16, 2, F32)
    none = torch.zeros(50, dtype=torch.bool, device="cuda")
    r = dense.balance_loss(x, chosen, mask=none)
    assert float(r.loss) == 0 and int(r.tokens) == 0 and not r.counts.any() and not r.mass.any()
    assert not dense.balance_loss_backward(x, r.counts, r.tokens, 2, mask=none).any()
    dead = torch.full((50, 16), -math.inf, device="cuda")
    for score, normalise in HOW:
        r = dense.balance_loss(dead, chosen, score=score, normalise=normalise)
        assert float(r.loss) == 0 and int(r.tokens) == 50 and not r.mass.any()
        assert not dense.balance_loss_backward(dead, r.counts, r.tokens, 2, score=score, normalise=normalise).any()


@gpu
@pytest.mark.parametrize("score,normalise", HOW)
def test_extreme_logits(score, normalise):
    """Lowest and largest values of the types, and rows that hold nothing else."""
    for dtype in (F32, BF16, F16):
        top = torch.finfo(dtype).max
        x = torch.tensor([[top, 0, -top, 3], [-top, -top, -top, -top], [top, top, top, top], [-90, -90, -91, -200], [60, 59, -60, 0]],
                         device="cuda").to(dtype)
        chosen = torch.tensor([[0, 1], [1, 2], [2, 3], [3, 0], [0, 1]], dtype=torch.int32, device="cuda")
        live = torch.ones(5, dtype=torch.bool, device="cuda")
        if score == "sigmoid":
            live[1] = live[3] = False             # scores below the floats count as 0: tested by themselves
        r = dense.balance_loss(x, chosen, score=score, normalise=normalise, mask=live)
        want = plain(x.double(), chosen, live, score, normalise, 1.0)
        ref.close(r.mass, want[2], want[2].max())
        g = dense.balance_loss_backward(x, r.counts, r.tokens, 2, score=score, normalise=normalise, mask=live)
        assert bool(torch.isfinite(g).all())
        if score == "sigmoid":
            low = ~live
            r = dense.balance_loss(x, chosen, score=score, normalise=normalise, mask=low)
            assert bool(torch.isfinite(r.mass).all()) and float(r.mass.max()) < (1e-30 if not normalise or dtype != F16 else 2)
            assert bool(torch.isfinite(dense.balance_loss_backward(x, r.counts, r.tokens, 2, score=score, normalise=normalise, mask=low)).all())


@gpu
def test_nan_stays_in_sight():
    x, chosen, _ = inputs(100, 16, 2, F32)
    x[7, 3] = math.nan
    for score, normalise in HOW:
        r = dense.balance_loss(x, chosen, score=score, normalise=normalise)
        assert math.isnan(float(r.loss)) and bool(torch.isnan(r.mass[3]))
        g = dense.balance_loss_backward(x, r.counts, r.tokens, 2, score=score, normalise=normalise)
        assert bool(torch.isnan(g[7, 3])) and bool(torch.isfinite(g[torch.arange(100, device="cuda") != 7]).all())


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_strides_and_leading_axes(dtype):
    x, chosen, _ = inputs(120, 24, 2, dtype)
    room = torch.full((120, 41), math.nan, dtype=dtype, device="cuda")
    for at in (0, 8, 1):
        part = room[:, at:at + 24]
        part.copy_(x)
        a, b = dense.balance_loss(part, chosen), dense.balance_loss(x, chosen)
        assert torch.equal(a.counts, b.counts)
        ref.close(a.mass, b.mass.double(), b.mass.max())
        ga = dense.balance_loss_backward(part, b.counts, b.tokens, 2, add=part)
        gb = dense.balance_loss_backward(x, b.counts, b.tokens, 2, add=x)
        assert ga.is_contiguous()
        ref.close(ga, gb.double(), 1 + gb.double().abs())
        part.fill_(math.nan)
    many = dense.balance_loss(x.view(4, 30, 24), chosen.view(4, 30, 2), mask=torch.ones(4, 30, dtype=torch.bool, device="cuda"))
    assert torch.equal(many.mass, dense.balance_loss(x, chosen, mask=torch.ones(120, dtype=torch.bool, device="cuda")).mass)
    assert dense.balance_loss_backward(x.view(4, 30, 24), many.counts, many.tokens, 2).shape == (4, 30, 24)


@gpu
def test_beside_the_router_and_over_ranks():
    """Two ranks' sums make the joint batch's gradient, added to that of the router's weights."""
    x, _, _ = inputs(800, 32, 4, F32, 9)
    r = dense.route(x, 4, score="sigmoid")
    whole = dense.balance_loss(x, r.experts, score="sigmoid", weight=0.1)
    assert torch.equal(whole.counts, torch.diff(r.offsets))
    dw = torch.randn(800, 4, generator=torch.Generator(device="cuda").manual_seed(2), device="cuda")
    first = dense.route_backward(x, r.experts, dw, score="sigmoid")
    joint = dense.balance_loss_backward(x, whole.counts, whole.tokens, 4, score="sigmoid", weight=0.1, add=first)
    parts = [dense.balance_loss(x[a:b], r.experts[a:b], score="sigmoid", weight=0.1) for a, b in ((0, 300), (300, 800))]
    counts, tokens = parts[0].counts + parts[1].counts, parts[0].tokens + parts[1].tokens
    assert torch.equal(counts, whole.counts) and int(tokens) == 800
    ref.close(parts[0].mass + parts[1].mass, whole.mass.double(), whole.mass.max())
    for a, b in ((0, 300), (300, 800)):
        g = dense.balance_loss_backward(x[a:b], counts, tokens, 4, score="sigmoid", weight=0.1, add=first[a:b])
        assert torch.equal(g, joint[a:b])


@gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_logits_beyond_32_bits(dtype):
    """Rows whose places pass 2^32 bytes; but a few are uniform, and add to each expert alike."""
    T, E = 2_300_000, 1000
    x = torch.zeros(T, E, dtype=dtype, device="cuda")
    chosen = torch.zeros(T, 1, dtype=torch.int32, device="cuda")
    odd = torch.tensor([5, T // 2, T - 2, T - 1], device="cuda")
    x[odd] = (torch.randn(4, E, generator=torch.Generator(device="cuda").manual_seed(1), device="cuda") * 3).to(dtype)
    r = dense.balance_loss(x, chosen)
    p = torch.softmax(x[odd].double(), -1)
    mass = p.sum(0) + (T - 4) / E
    assert int(r.tokens) == T and int(r.counts[0]) == T and not r.counts[1:].any()
    # a lane adds up to some 2000 rows' shares, each sum rounded to its half a unit
    ref.close(r.mass, mass, mass, rel=2000 * 2.0 ** -24)
    ref.close(r.loss, E / T * mass[0], mass[0], rel=2000 * 2.0 ** -24)
    g = dense.balance_loss_backward(x, r.counts, r.tokens, 1, dloss=torch.tensor(float(T), device="cuda"))
    d = torch.full((E,), -1.0, dtype=torch.float64, device="cuda")
    d[0] = E - 1.0
    want = p * (d - (p * d).sum(-1, keepdim=True))
    ref.close(g[odd], want, E * p)
    plain_row = (d - d.mean()) / E
    for a in (0, T // 2 + 1, T - 3):
        ref.close(g[a], plain_row, 1.0)


@gpu
def test_captured():
    x, chosen, mask = inputs(3000, 64, 4, BF16, 1, padded=True)
    want = dense.balance_loss(x, chosen, mask=mask)
    dwant = dense.balance_loss_backward(x, want.counts, want.tokens, 4, mask=mask)
    other, _, _ = inputs(3000, 64, 4, BF16, 2)
    graph = torch.cuda.CUDAGraph()
    held = other.clone()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        r = dense.balance_loss(held, chosen, mask=mask)
        g = dense.balance_loss_backward(held, r.counts, r.tokens, 4, mask=mask)
    held.copy_(x)
    graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(r, want)) and torch.equal(g, dwant)


@gpu
def test_refusals():
    x, chosen, _ = inputs(20, 16, 2, F32)
    ok = dense.balance_loss(x, chosen)
    bad = [lambda: dense.balance_loss(x.double(), chosen), lambda: dense.balance_loss(x, chosen.long()), lambda: dense.balance_loss(x, chosen[:10]),
           lambda: dense.balance_loss(x, chosen[:, :0]), lambda: dense.balance_loss(x, chosen, score="relu"),
           lambda: dense.balance_loss(x, chosen, mask=torch.ones(19, dtype=torch.bool, device="cuda")),
           lambda: dense.balance_loss(x, chosen, mask=torch.ones(20, device="cuda")), lambda: dense.balance_loss(x, chosen, weight=math.nan),
           lambda: dense.balance_loss(x.T, chosen), lambda: dense.balance_loss(x.cpu(), chosen),
           lambda: dense.balance_loss(torch.zeros(2, 1025, device="cuda"), chosen[:2]),
           lambda: dense.balance_loss(x, torch.zeros(20, 33, dtype=torch.int32, device="cuda")),
           lambda: dense.balance_loss_backward(x, ok.counts[:8], ok.tokens, 2), lambda: dense.balance_loss_backward(x, ok.mass, ok.tokens, 2),
           lambda: dense.balance_loss_backward(x, ok.counts, ok.tokens, 0), lambda: dense.balance_loss_backward(x, ok.counts, ok.tokens, 33),
           lambda: dense.balance_loss_backward(x, ok.counts, ok.tokens, 2, add=x.bfloat16()),
           lambda: dense.balance_loss_backward(x, ok.counts, ok.tokens, 2, add=x[:5]),
           lambda: dense.balance_loss_backward(x, ok.counts, ok.tokens, 2, dloss=ok.tokens)]
    for call in bad:
        with pytest.raises(EpsError) as e:
            call()
        assert e.value.code == INVALID_ARGUMENT
