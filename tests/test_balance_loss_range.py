"""Rows of sigmoids that are all next to nothing: their shares are those of the formula as far down as a float can tell a
score from 0, which is where the router's weights end: logits below -88.7 count as -inf."""
import math

import pytest
import torch

import dense_reference as ref
from conftest import import_package
from test_balance_loss import plain, shares

import_package()
from eps_b200 import dense  # noqa: E402

gpu = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
LEAST = 2.0 ** -149      # the smallest float: what a sum or product of scores may be off by below the normal ones
# half the spacing of each type's subnormal values, the rounding of a result there: the smallest normal value, 2^-126 or
# 2^-14, times half of the type's 2^-23, 2^-7 or 2^-10
HALF = {F32: 2.0 ** -150, BF16: 2.0 ** -134, F16: 2.0 ** -25}


def near(got, want, size, floor):
    """ref.close, with the rounding below the normal values and `floor` of the smallest floats."""
    want = want.double()
    limit = ref.UNIT[got.dtype] * want.abs() + ref.CHAIN * size + HALF[got.dtype] + floor * LEAST
    assert got.shape == want.shape and bool(((got.double() - want).abs() <= limit).all())


def rows(T, E, dtype, masked, seed=1):
    """Rows whose largest logits lie from -88.5 to -41, some among them ordinary; all multiples of 1/2, which each type holds."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    top = -41 - torch.rand(T, 1, generator=g, device="cuda") * 47.5
    top[torch.rand(T, 1, generator=g, device="cuda") < 0.3] = -88
    top[::5] = 1
    x = top - torch.rand(T, E, generator=g, device="cuda") * 12
    x[torch.arange(T, device="cuda"), torch.randint(0, E, (T,), generator=g, device="cuda")] = top[:, 0]
    x = (x * 2).round() / 2
    x = x.clamp(min=-96)
    if masked:
        out = torch.rand(T, E, generator=g, device="cuda") < 0.3
        x = x.masked_fill(out, -math.inf)
        x[T // 2] = -math.inf
    assert bool((x.to(dtype).float() == x).all())
    return x.to(dtype)


@gpu
@pytest.mark.parametrize("T,E,k", [(1, 1, 1), (3, 128, 6), (50, 5, 2), (300, 96, 4), (301, 250, 8), (900, 16, 1), (200, 261, 3), (1500, 256, 8), (60, 1023, 2),
                                   (40, 1024, 8), (2000, 33, 4)])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("normalise", [True, False])
@pytest.mark.parametrize("masked", [False, True])
def test_scores_next_to_nothing(T, E, k, dtype, normalise, masked):
    x = rows(T, E, dtype, masked)
    if T == 1:
        x.fill_(-88)
    mask = torch.rand(T, generator=torch.Generator(device="cuda").manual_seed(3), device="cuda") < 0.8
    chosen = torch.randint(0, E, (T, k), generator=torch.Generator(device="cuda").manual_seed(2), device="cuda", dtype=torch.int32)
    how = dict(score="sigmoid", normalise=normalise, mask=mask, weight=0.25)
    got = dense.balance_loss(x, chosen, **how)
    xd = x.double().masked_fill(x < -88.7, -math.inf).requires_grad_(True)
    loss, counts, mass, n = plain(xd, chosen, mask, "sigmoid", normalise, 0.25)
    assert int(got.tokens) == n and torch.equal(got.counts.long(), counts)
    near(got.mass, mass.detach(), mass.detach().max(), T)
    near(got.loss, loss.detach(), loss.detach().abs(), 0.25 * E * T)
    dloss = torch.tensor(float(max(1, n)), device="cuda")
    want = torch.autograd.grad(loss, xd, dloss.double())[0].nan_to_num(0.0) if n else torch.zeros_like(xd)
    want = torch.where(mask[:, None], want, 0.0)
    have = dense.balance_loss_backward(x, got.counts, got.tokens, k, dloss=dloss, **how)
    c = 0.25 * E / (k * max(1, n))
    d = (counts - k * n / E).abs().max() if normalise else counts.max()
    near(have, want, c * d * shares(xd, "sigmoid", normalise).detach(), 4 * (1 + c * d))


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("value", [-39.0, -41.0, -60.0, -87.0, -87.5, -88.0, -88.5, -89.0, -104.0, -200.0])
def test_equal_shares_as_the_router_has_them(value, dtype):
    """Equal logits have equal shares, as far as the router's renormalised weights have."""
    x = torch.full((70, 8), value, device="cuda").to(dtype)
    r = dense.route(x, 8, score="sigmoid", sort=False)
    got = dense.balance_loss(x, r.experts, score="sigmoid")
    weights = torch.zeros(70, 8, dtype=torch.float64, device="cuda").scatter_(1, r.experts.long(), r.weights.double())
    # a share is a score (an exponential and a reciprocal, a few units) by the reciprocal of their sum, added 70 times: within CHAIN
    want = torch.full((8,), 70 / 8 if value > -88.7 else 0.0, dtype=torch.float64, device="cuda")
    ref.close(got.mass, want, want)
    ref.close(got.mass, weights.sum(0), want)
    ref.close(got.loss, want[0] * 8 / 70, want[0] * 8 / 70)
    plain_mass = dense.balance_loss(x, r.experts, score="sigmoid", normalise=False).mass
    scores = dense.route(x, 8, score="sigmoid", renormalise=False, sort=False).weights
    near(plain_mass, torch.full((8,), float(scores.double()[0, 0] * 70), device="cuda"), plain_mass.max(), 140)
