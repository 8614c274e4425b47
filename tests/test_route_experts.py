"""Routing to experts against plain loops and 64-bit scores: ties, masked rows, NaN, groups, the sort
by expert and the gradient."""
import math

import pytest
import torch

import dense_reference as ref
from conftest import import_package

import_package()
from eps_b200 import EpsError, INVALID_ARGUMENT, dense  # noqa: E402

gpu = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def logits_of(seed, tokens, experts, dtype=F32):
    """Logits whose scores are far enough apart that rounding does not decide a rank: each row a
    permutation of evenly spaced values."""
    g = torch.Generator().manual_seed(seed)
    base = torch.linspace(-3.0, 3.0, experts) if experts > 1 else torch.zeros(1)
    rows = [base[torch.randperm(experts, generator=g)] for _ in range(tokens)]
    return (torch.stack(rows) if rows else torch.zeros(0, experts)).cuda().to(dtype)


def check_sort(r, experts):
    flat = r.experts.reshape(-1)
    order = torch.sort(flat, stable=True).indices
    assert torch.equal(r.order.long(), order)
    assert torch.equal(flat[r.order.long()], flat.sort(stable=True).values)
    back = torch.empty_like(order)
    back[order] = torch.arange(len(order), device="cuda")
    assert torch.equal(r.position.reshape(-1).long(), back)
    counts = torch.bincount(flat.long(), minlength=experts)
    assert torch.equal(r.offsets.long(), torch.cat([counts.new_zeros(1), counts.cumsum(0)]))


def weights_of(p, chosen, renormalise, scale):
    w = p.gather(1, chosen.long())
    if renormalise:
        total = w.sum(-1, keepdim=True)
        w = torch.where(total == 0, 0.0, w / torch.where(total == 0, 1.0, total))
    return w * scale


def check(logits, top_k, score="softmax", bias=None, groups=1, top_groups=1, renormalise=True, scale=1.0):
    r = dense.route(logits, top_k, score=score, bias=bias, groups=groups, top_groups=top_groups,
                    renormalise=renormalise, scale=scale)
    p = ref.scores(logits, score)
    key = p if bias is None else p + bias.double()
    want = torch.tensor(ref.ranked(key, groups, top_groups, top_k), dtype=torch.int32, device="cuda").view(-1, top_k)
    assert torch.equal(r.experts, want)
    ref.close(r.weights, weights_of(p, want, renormalise, scale), weights_of(p, want, renormalise, scale).abs())
    check_sort(r, logits.shape[1])
    return r


@gpu
@pytest.mark.parametrize("experts", [1, 4, 31, 32, 33, 64, 100, 128, 255, 256, 500, 1024])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_expert_counts(experts, score):
    for k in sorted({1, min(2, experts), min(8, experts), min(32, experts)}):
        check(logits_of(experts + k, 21, experts), k, score)


@gpu
@pytest.mark.parametrize("tokens", [0, 1, 15, 16, 17, 127, 128, 129, 1000, 4099])
def test_token_counts(tokens):
    check(logits_of(tokens, tokens, 24), 3)


@gpu
@pytest.mark.parametrize("experts,groups,top_groups,k", [(8, 8, 3, 3), (16, 4, 2, 5), (24, 3, 1, 8), (64, 8, 4, 6), (256, 8, 4, 8),
                                                         (96, 48, 20, 9), (1000, 40, 7, 12), (64, 8, 8, 4)])
def test_groups_with_bias(experts, groups, top_groups, k):
    bias = torch.linspace(-0.4, 0.4, experts, device="cuda")[torch.randperm(experts, generator=torch.Generator().manual_seed(1)).cuda()]
    for score in ("softmax", "sigmoid"):
        for renormalise in (True, False):
            # a row's scores plus the bias are sums of two spaced sets: ranks come from float32 sums, as here
            x = logits_of(3, 40, experts)
            r = dense.route(x, k, score=score, bias=bias, groups=groups, top_groups=top_groups, renormalise=renormalise, scale=2.5)
            p = scores32(x, score)
            want = torch.tensor(ref.ranked(p + bias, groups, top_groups, k), dtype=torch.int32, device="cuda")
            assert torch.equal(r.experts, want)
            w = weights_of(ref.scores(x, score), want, renormalise, 2.5)
            ref.close(r.weights, w, w.abs())
            check_sort(r, experts)


def scores32(x, score):
    x = x.float()
    if score == "sigmoid":
        return 1 / (1 + torch.exp(-x))
    e = torch.exp(x - x.max(-1, keepdim=True).values)
    return e / e.double().sum(-1, keepdim=True).float()


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_types_and_strides(dtype):
    x = logits_of(5, 50, 33, dtype)       # in 16 bits some neighbours are equal: the lower index comes first
    check(x, 4, "sigmoid")
    room = torch.zeros(50, 40, dtype=dtype, device="cuda")
    room[:, 3:36] = x
    check(room[:, 3:36], 4, "sigmoid")
    room = torch.zeros(50, 128, dtype=dtype, device="cuda")
    room[:, :64] = logits_of(6, 50, 64, dtype)
    check(room[:, :64], 4, "softmax")


@gpu
def test_ties_go_to_the_lower_index():
    x = torch.zeros(130, 40, device="cuda")
    r = check(x, 5)
    assert torch.equal(r.experts, torch.arange(5, dtype=torch.int32, device="cuda").expand(130, 5))
    x[:, 7], x[:, 30] = 1.0, 1.0
    assert check(x, 4, "sigmoid").experts[0].tolist() == [7, 30, 0, 1]
    r = check(torch.zeros(3, 40, device="cuda"), 6, groups=4, top_groups=2)
    assert r.experts[0].tolist() == [0, 1, 2, 3, 4, 5]


@gpu
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_masked_experts_and_rows(score):
    x = logits_of(7, 12, 20)
    x[:, 5:15] = -math.inf
    x[3] = -math.inf                     # nothing left: scores 0, weights 0, the lowest indices
    x[4, 1:] = -math.inf                 # less left than wanted
    r = check(x, 6, score)
    assert r.experts[3].tolist() == [0, 1, 2, 3, 4, 5] and not r.weights[3].any()
    x[:, :] = torch.finfo(F32).min       # the type's lowest value: equal logits
    r = check(x, 3, score)
    assert r.experts[0].tolist() == [0, 1, 2]


@gpu
def test_bad_values():
    nan, inf = math.nan, math.inf
    x = logits_of(8, 5, 10)
    clean = dense.route(x, 3, score="sigmoid")
    x[1, 4] = nan
    r = dense.route(x, 3, score="sigmoid", renormalise=False)
    assert 4 not in r.experts[1].tolist() and not r.weights.isnan().any()      # ranks last
    assert torch.equal(r.experts[0], clean.experts[0])
    r = dense.route(x, 10, score="sigmoid", renormalise=False)
    assert r.experts[1, 9] == 4 and r.weights[1, 9].isnan()
    r = dense.route(x, 3, score="softmax")                      # a NaN in a softmax is in all of the row
    assert r.experts[1].tolist() == [0, 1, 2] and r.weights[1].isnan().all() and not r.weights[2].isnan().any()
    x[1, 4] = inf
    assert dense.route(x, 3, score="softmax").weights[1].isnan().all()
    assert dense.route(x, 3, score="sigmoid").experts[1, 0] == 4
    bias = torch.zeros(10, device="cuda")
    bias[[0, 3]] = -inf                                        # experts taken out by their bias
    r = dense.route(x, 8, score="sigmoid", bias=bias)
    assert not ((r.experts == 0) | (r.experts == 3)).any()


@gpu
def test_large_batch_sorts():
    x = torch.randn(70001, 128, generator=torch.Generator(device="cuda").manual_seed(3), device="cuda")
    r = dense.route(x, 6, score="sigmoid")
    check_sort(r, 128)
    assert torch.equal(r.experts, torch.sort(scores32(x, "sigmoid"), dim=-1, descending=True, stable=True).indices[:, :6].int())
    skewed = x.clone()
    skewed[:, 5] += 100                                       # one expert takes every token
    check_sort(dense.route(skewed, 2), 128)
    plain = dense.route(x, 6, score="sigmoid", sort=False)
    assert plain.order is None and torch.equal(plain.experts, r.experts) and torch.equal(plain.weights, r.weights)


@gpu
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renormalise", [True, False])
@pytest.mark.parametrize("experts,k,dtype", [(1, 1, F32), (5, 5, F32), (32, 4, BF16), (100, 8, F32), (256, 8, F16), (1024, 32, F32)])
def test_gradient(score, renormalise, experts, k, dtype):
    x = logits_of(11, 45, experts, dtype)
    x[2, 0] = -math.inf
    chosen = dense.route(x, k, score=score).experts
    dw = torch.randn(45, k, generator=torch.Generator(device="cuda").manual_seed(2), device="cuda")
    got = dense.route_backward(x, chosen, dw, score=score, renormalise=renormalise, scale=1.5)
    assert got.dtype == dtype and got.shape == x.shape
    p = ref.scores(x, score)
    s, d = p.gather(1, chosen.long()), dw.double() * 1.5
    size = d.abs()
    if renormalise:
        total = s.sum(-1, keepdim=True)
        size = torch.where(total == 0, 0.0, (size + (size * s).sum(-1, keepdim=True) / total) / total)
        d = torch.where(total == 0, 0.0, (d - (d * s).sum(-1, keepdim=True) / total) / total)
    ds = torch.zeros_like(p).scatter_(1, chosen.long(), d)
    ss = torch.zeros_like(p).scatter_(1, chosen.long(), size)
    if score == "sigmoid":
        want, terms = ds * p * (1 - p), ss * p
    else:
        want, terms = p * (ds - (ds * p).sum(-1, keepdim=True)), p * (ss + (ss * p).sum(-1, keepdim=True))
    ref.close(got, want, terms)


@gpu
def test_gradient_against_differences():
    x = logits_of(13, 6, 12)
    dw = torch.randn(6, 4, generator=torch.Generator(device="cuda").manual_seed(2), device="cuda")
    direction = torch.randn(6, 12, generator=torch.Generator(device="cuda").manual_seed(4), device="cuda").double()
    for score in ("softmax", "sigmoid"):
        for renormalise in (True, False):
            chosen = dense.route(x, 4, score=score).experts
            got = dense.route_backward(x, chosen, dw, score=score, renormalise=renormalise)
            loss = lambda v: (weights_of(ref.scores(v, score), chosen, renormalise, 1.0) * dw).sum().item()  # noqa: E731
            step = 1e-6
            want = (loss(x.double() + step * direction) - loss(x.double() - step * direction)) / (2 * step)
            have = (got.double() * direction).sum().item()
            assert abs(want - have) <= 1e-5 * (got.double() * direction).abs().sum().item() + 1e-7


@gpu
def test_gradient_of_masked_rows_and_strange_entries():
    x = logits_of(15, 4, 8)
    x[1] = -math.inf
    chosen = dense.route(x, 2).experts
    dw = torch.ones(4, 2, device="cuda")
    assert not dense.route_backward(x, chosen, dw)[1].any()
    chosen[2] = torch.tensor([-1, 8], dtype=torch.int32)      # outside: skipped
    got = dense.route_backward(x, chosen, dw, renormalise=False)
    assert not got[2].any() and got[0].any()
    assert dense.route_backward(x[:0], chosen[:0], dw[:0]).shape == (0, 8)


@gpu
def test_stream_and_graph():
    x = logits_of(17, 600, 64)
    want = dense.route(x, 4)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        late = torch.empty_like(x)
        torch.cuda._sleep(20_000_000)
        late.copy_(x)
        got = dense.route(late, 4)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = dense.route(x, 4)
    x.copy_(x.flip(1))
    graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(got, dense.route(x, 4)))


@gpu
def test_refusals():
    x = logits_of(1, 4, 12)
    bad = [lambda: dense.route(x, 0), lambda: dense.route(x, 13), lambda: dense.route(x, 2, groups=5), lambda: dense.route(x, 2, groups=0),
           lambda: dense.route(x, 2, groups=4, top_groups=5), lambda: dense.route(x, 7, groups=4, top_groups=2),
           lambda: dense.route(x, 2, score="relu"), lambda: dense.route(x, 2, bias=torch.zeros(11, device="cuda")),
           lambda: dense.route(x, 2, bias=torch.zeros(12, device="cuda", dtype=BF16)), lambda: dense.route(x.cpu(), 2),
           lambda: dense.route(x.double(), 2), lambda: dense.route(x.t(), 2), lambda: dense.route(x, 2, scale=math.nan),
           lambda: dense.route(torch.zeros(2, 1025, device="cuda"), 2), lambda: dense.route(torch.zeros(2, 64, device="cuda"), 33),
           lambda: dense.route_backward(x, torch.zeros(4, 2, device="cuda"), torch.zeros(4, 2, device="cuda")),
           lambda: dense.route_backward(x, torch.zeros(3, 2, device="cuda", dtype=torch.int32), torch.zeros(3, 2, device="cuda"))]
    for call in bad:
        with pytest.raises(EpsError) as e:
            call()
        assert e.value.code == INVALID_ARGUMENT
