"""Masked logits (-inf) under a bias: they rank last whatever their bias, alone and in their groups."""
import math

import pytest
import torch

import dense_reference as ref
from conftest import import_package
from test_route_experts import check_sort, logits_of, scores32, weights_of

import_package()
from eps_b200 import dense  # noqa: E402

gpu = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def wanted(x, bias, score, groups, top_groups, k):
    """By plain loops: the key of a masked logit is the lowest."""
    key = (scores32(x, score) + bias).masked_fill(x == -math.inf, -math.inf)
    return torch.tensor(ref.ranked(key, groups, top_groups, k), dtype=torch.int32, device="cuda").view(-1, k)


@gpu
@pytest.mark.parametrize("score,high", [("softmax", 0.3), ("sigmoid", 0.9)])
def test_a_bias_does_not_bring_a_masked_expert_back(score, high):
    x = torch.tensor([[2.0, 1.0, -1.0, -math.inf]], device="cuda")
    bias = torch.tensor([0.0, 0.0, 0.0, high], device="cuda")
    r = dense.route(x, 3, score=score, bias=bias)
    assert r.experts.tolist() == [[0, 1, 2]] and bool((r.weights > 0).all())
    r = dense.route(x, 4, score=score, bias=bias)
    assert r.experts.tolist() == [[0, 1, 2, 3]] and r.weights[0, 3] == 0


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("experts,groups,top_groups,k", [(20, 1, 1, 6), (96, 1, 1, 4), (64, 8, 4, 6), (24, 3, 1, 8), (96, 48, 20, 9), (512, 8, 3, 12),
                                                         (1000, 40, 7, 12)])
def test_masked_experts_with_bias(experts, groups, top_groups, k, score, dtype):
    x = logits_of(experts + k, 40, experts, dtype)
    g = torch.Generator().manual_seed(5)
    bias = torch.linspace(-0.4, 0.4, experts)[torch.randperm(experts, generator=g)].cuda()
    x[(torch.rand(40, experts, generator=g) < 0.3).cuda()] = -math.inf
    x[3, : experts // groups] = -math.inf                      # a whole group of one row, with the largest bias
    bias[: experts // groups] += 1.0
    x[4] = -math.inf                                           # a whole row
    x[5, k:] = -math.inf                                       # about as many as wanted
    r = dense.route(x, k, score=score, bias=bias, groups=groups, top_groups=top_groups)
    want = wanted(x, bias, score, groups, top_groups, k)
    assert torch.equal(r.experts, want)
    w = weights_of(ref.scores(x, score), want, True, 1.0)
    ref.close(r.weights, w, w.abs())
    assert r.experts[4].tolist() == list(range(k)) and not r.weights[4].any()
    check_sort(r, experts)


@gpu
def test_only_minus_infinity_masks():
    """The lowest finite logit has a score of 0, and its bias still ranks it; +infinity is the best score."""
    x = torch.tensor([[1.0, torch.finfo(F32).min, 0.0, math.inf]], device="cuda")
    bias = torch.tensor([0.0, 2.0, 0.0, 0.0], device="cuda")
    assert dense.route(x, 3, score="sigmoid", bias=bias).experts.tolist() == [[1, 3, 0]]
