"""The block trained with a balance loss and clipped steps and served with adapters: its gradients are those of the same
model differentiated by torch, its steps those of the clipped gradients, and what it serves that of the formula."""
import importlib.util
import os

import pytest
import torch

import dense_reference as ref
from conftest import ROOT, import_package

import_package()
gpu = pytest.mark.gpu


def example():
    spec = importlib.util.spec_from_file_location("expert_block", os.path.join(ROOT, "examples", "expert_block.py"))
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m


def rand(seed, *shape):
    return torch.randn(*shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda")


def rms(v, w):
    return v / torch.sqrt((v * v).mean(-1, keepdim=True) + 1e-6) * w


@gpu
def test_example_runs():
    first, last, served = example().run(steps=5, batch=64, rows=50, balance_weight=0.01, max_norm=0.5)
    assert all(map(torch.isfinite, torch.tensor([first, last, served])))


@gpu
def test_gradients_and_clipped_step():
    from eps_b200 import dense
    weight = 0.3
    block = example().ExpertBlock(dense, 3, 8, experts=5, top_k=2, hidden=12, state_bits=32, balance_weight=weight, max_norm=0.1)
    x, ds = rand(3, 40, 24), rand(4, 40)
    score, kept = block.forward(x)
    dx = block.backward(ds, kept)
    p = {k: v.double().requires_grad_(True) for k, v in block.p.items()}
    xd = x.double().requires_grad_(True)
    z = rms(xd, p["pre"])
    chosen = kept[2].experts.long()
    all_scores = torch.sigmoid(z @ p["router"].T)
    s = all_scores.gather(1, chosen)
    w = s / s.sum(-1, keepdim=True)
    mid = torch.relu(torch.einsum("td,ehd->teh", z, p["up"]))
    each = torch.einsum("teh,edh->ted", mid, p["down"]).gather(1, chosen[..., None].expand(-1, -1, 24))
    h = xd + 0.5 * torch.sigmoid(z @ p["gate"].T) * rms((each * w[..., None]).sum(1), p["post"])
    want = rms(h, p["final"]) @ p["head"][0]
    counts = torch.bincount(chosen.reshape(-1), minlength=5)
    mass = (all_scores / all_scores.sum(-1, keepdim=True)).sum(0)
    balance = weight * 5 / (2 * 40 * 40) * (counts * mass).sum()
    assert torch.equal(block.balanced.counts.long(), counts)
    ref.close(block.balanced.loss, balance.detach())
    ((want * ds.double()).sum() + balance).backward()
    for name, g in [("x", xd.grad), *((k, v.grad) for k, v in p.items())]:
        have = dx if name == "x" else block.grads[name]
        # a chain of six products of up to 40 terms each: some ten times one operator's roundings
        ref.close(have, g, 10 * g.abs().max())
    # the step takes the gradients at a norm of 0.1, whatever they were
    before = {k: v.clone() for k, v in block.p.items()}
    norm = torch.sqrt(sum((g.double() ** 2).sum() for g in block.grads.values()))
    assert norm > 0.1
    block.step()
    for k, g in block.grads.items():
        g = g.double() * 0.1 / norm
        moved = before[k].double() * (1 - 3e-3 * 1e-4) - 3e-3 * g / (g.abs() + 1e-8)      # a first step: its moments are those of g
        # the factor is off by some units, which g / (|g| + epsilon) does not show
        ref.close(block.p[k], moved, 1 + moved.abs())
    block.grads["head"][0, 0] = float("nan")
    before = {k: v.clone() for k, v in block.p.items()}
    block.step()
    assert all(torch.equal(before[k], v) for k, v in block.p.items())


@gpu
def test_served_with_adapters():
    from eps_b200 import dense
    block = example().ExpertBlock(dense, 3, 8, experts=5, top_k=2, hidden=12)
    down, up = rand(1, 4, 3, 24), rand(2, 4, 24, 3)
    for rows in (30, 300):
        x = rand(3, rows, 24)
        ids = torch.randint(-1, 4, (rows,), generator=torch.Generator(device="cuda").manual_seed(5), device="cuda", dtype=torch.int32)
        adapted, plain = block.serve(dense.Adapters(down, up)), block.serve()
        got, base = adapted(x, ids), plain(x)
        none = ids < 0
        assert torch.equal(adapted(x), base)
        ref.close(got[none], base[none].double(), 10 * base.abs().max())
        # one adapter at a time, as a gate of its own
        gate = block.p["gate"].clone()
        for a in range(4):
            block.p["gate"].copy_(gate + up[a] @ down[a])
            want = block.serve()(x)[ids == a]
            # the same products and roundings but for the gate's, whose terms are some 24 * 3 times as large as a score's unit
            ref.close(got[ids == a], want.double(), 72 * 10 * want.abs().max())
        block.p["gate"].copy_(gate)
