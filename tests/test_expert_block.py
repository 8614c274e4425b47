"""The dense operators and the store together: the example trains, serves in 8 bits, and its gradients
are those of the same model differentiated by torch."""
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


@gpu
@pytest.mark.parametrize("bits", [8, 32])
def test_example_learns_and_serves(bits):
    first, last, served = example().run(steps=60, batch=512, rows=300, state_bits=bits)
    assert last < 0.9 * first
    # 8-bit products: each value is off by at most half of 1 / 127 of its row's largest, far below the loss
    assert abs(served - last) < 0.02


@gpu
def test_block_gradients_against_autograd():
    from eps_b200 import dense
    block = example().ExpertBlock(dense, 3, 8, experts=5, top_k=2, hidden=12)
    x = torch.randn(40, 24, generator=torch.Generator(device="cuda").manual_seed(3), device="cuda")
    ds = torch.randn(40, generator=torch.Generator(device="cuda").manual_seed(4), device="cuda")
    score, kept = block.forward(x)
    dx = block.backward(ds, kept)
    p = {k: v.double().requires_grad_(True) for k, v in block.p.items()}
    xd = x.double().requires_grad_(True)
    rms = lambda v, w: v / torch.sqrt((v * v).mean(-1, keepdim=True) + 1e-6) * w  # noqa: E731
    z = rms(xd, p["pre"])
    chosen = kept[2].experts.long()
    s = torch.sigmoid(z @ p["router"].T).gather(1, chosen)
    w = s / s.sum(-1, keepdim=True)
    mid = torch.relu(torch.einsum("td,ehd->teh", z, p["up"]))
    each = torch.einsum("teh,edh->ted", mid, p["down"]).gather(1, chosen[..., None].expand(-1, -1, 24))
    y = (each * w[..., None]).sum(1)
    h = xd + 0.5 * torch.sigmoid(z @ p["gate"].T) * rms(y, p["post"])
    want = rms(h, p["final"]) @ p["head"][0]
    ref.close(score, want.detach(), 10 * want.detach().abs().max())
    want.backward(ds.double())
    for name, g in [("x", xd.grad), *((k, v.grad) for k, v in p.items())]:
        have = dx if name == "x" else block.grads[name]
        # a chain of six products of up to 40 terms each: some ten times one operator's roundings
        ref.close(have, g, 10 * g.abs().max())
