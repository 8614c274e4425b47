"""A mixture-of-experts ranking model on the embedding store: trained, then served in 8 bits.

The store holds the sparse part (its rows pooled by the lookup, its gradients coalesced and
applied by the push); the dense operators hold the rest:

    pull -> block_norm -> route -> experts' products -> block_norm (gate, residual) -> score
    backward of the same -> push of the embeddings' gradients, AdamW on the dense weights

Serving reuses the trained weights: a read-only lookup, the same router, and the experts'
products in 8-bit integers (dense.QuantizedExperts) grouped by the router's offsets.

    python examples/expert_block.py [--steps N] [--state-bits 8|32]
"""
from __future__ import annotations

import argparse
import importlib
import math
import os
import sys

import numpy as np
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
PACKAGE = "distributed-recommendation-model-training-system_b200"


def load_package():
    """The package under the name eps_b200 (its folder's name is no Python identifier)."""
    if "eps_b200" not in sys.modules:
        sys.path.insert(0, ROOT)
        sys.modules["eps_b200"] = importlib.import_module(PACKAGE)
    return sys.modules["eps_b200"], importlib.import_module("eps_b200.dense")


class ExpertBlock:
    """One mixture-of-experts block over pooled embeddings, with its backward pass."""

    def __init__(self, dense, features: int, dimension: int, experts: int = 8, top_k: int = 2, hidden: int = 128,
                 state_bits: int = 8, learning_rate: float = 3e-3, seed: int = 1):
        self.dense, self.width, self.top_k, self.experts = dense, features * dimension, top_k, experts
        g = torch.Generator(device="cuda").manual_seed(seed)
        d = self.width

        def weight(*shape):
            return torch.randn(*shape, generator=g, device="cuda") / math.sqrt(shape[-1])
        self.p = {"pre": torch.ones(d, device="cuda"), "post": torch.ones(d, device="cuda"), "final": torch.ones(d, device="cuda"),
                  "router": weight(experts, d), "up": weight(experts, hidden, d), "down": weight(experts, d, hidden),
                  "gate": weight(d, d), "head": weight(1, d)}
        self.grads = {k: torch.zeros_like(v) for k, v in self.p.items()}
        self.balance = torch.zeros(experts, device="cuda")
        self.norm = dict(kind="rms", activation="sigmoid", scale=0.5, epsilon=1e-6)
        self.optimizer = dense.AdamW(list(self.p.values()), list(self.grads.values()), learning_rate=learning_rate,
                                     weight_decay=1e-4, state_bits=state_bits, seed=seed)

    def route(self, z):
        return self.dense.route(z @ self.p["router"].T, self.top_k, score="sigmoid", bias=self.balance)

    def forward(self, x):
        """Scores of x [batch, features * dimension], and what the backward pass needs."""
        p, n = self.p, self.norm
        _, z = self.dense.block_norm(x, pre_weight=p["pre"], kind=n["kind"], epsilon=n["epsilon"])
        r = self.route(z)
        ends = r.offsets.tolist()
        rows = z[r.order.long() // self.top_k]
        up = torch.cat([rows[a:b] @ w.T for a, b, w in zip(ends, ends[1:], p["up"])])
        mid = torch.relu(up)
        out = torch.cat([mid[a:b] @ w.T for a, b, w in zip(ends, ends[1:], p["down"])])
        each = out[r.position.long()]                       # [batch, top_k, width]
        y = (each * r.weights[..., None]).sum(1)
        gate = z @ p["gate"].T
        h, last = self.dense.block_norm(x, y, gate, post_weight=p["post"], pre_weight=p["final"], **n)
        return last @ p["head"][0], (x, z, r, ends, rows, up, mid, each, y, gate, h, last)

    def backward(self, dscore, kept):
        """Fills the gradients; returns that of x."""
        p, n, g = self.p, self.norm, self.grads
        x, z, r, ends, rows, up, mid, each, y, gate, h, last = kept
        torch.mv(last.T, dscore, out=g["head"][0])
        joint = self.dense.block_norm_backward(None, dscore[:, None] * p["head"], h, y, gate, post_weight=p["post"],
                                               pre_weight=p["final"], **n)
        g["post"].copy_(joint.post_weight)
        g["final"].copy_(joint.pre_weight)
        torch.mm(joint.gate.T, z, out=g["gate"])
        dz = joint.gate @ p["gate"]
        dweights = (each * joint.y[:, None]).sum(-1)
        dout = (joint.y[:, None] * r.weights[..., None]).reshape(-1, self.width)[r.order.long()]
        dmid = torch.empty_like(mid)
        drows = torch.empty_like(rows)
        for e, (a, b) in enumerate(zip(ends, ends[1:])):
            torch.mm(dout[a:b].T, mid[a:b], out=g["down"][e])
            torch.mm(dout[a:b], p["down"][e], out=dmid[a:b])
        dmid *= up > 0
        for e, (a, b) in enumerate(zip(ends, ends[1:])):
            torch.mm(dmid[a:b].T, rows[a:b], out=g["up"][e])
            torch.mm(dmid[a:b], p["up"][e], out=drows[a:b])
        dz += drows[r.position.long()].sum(1)
        dlogits = self.dense.route_backward(z @ p["router"].T, r.experts, dweights, score="sigmoid")
        torch.mm(dlogits.T, z, out=g["router"])
        dz += dlogits @ p["router"]
        first = self.dense.block_norm_backward(joint.x, dz, x, pre_weight=p["pre"], kind=n["kind"], epsilon=n["epsilon"])
        g["pre"].copy_(first.pre_weight)
        return first.x

    def rebalance(self, routing, rate: float = 1e-3):
        """Moves the ranking bias towards experts that got fewer tokens than their share."""
        counts = torch.diff(routing.offsets).float()
        self.balance += rate * torch.sign(counts.mean() - counts)

    def serve(self):
        """The scoring function with the experts' products in 8-bit integers."""
        dense, p, n = self.dense, self.p, self.norm
        up, down = dense.QuantizedExperts.from_weights(p["up"]), dense.QuantizedExperts.from_weights(p["down"])

        def score(x):
            _, z = dense.block_norm(x, pre_weight=p["pre"], kind=n["kind"], epsilon=n["epsilon"])
            r = self.route(z)
            mid = torch.relu(up.product(z, offsets=r.offsets, rows=r.order, rows_divisor=self.top_k))
            each = down.product(mid, offsets=r.offsets)[r.position.long()]
            y = (each * r.weights[..., None]).sum(1)
            _, last = dense.block_norm(x, y, z @ p["gate"].T, post_weight=p["post"], pre_weight=p["final"], **n)
            return last @ p["head"][0]
        return score


def run(steps: int = 150, batch: int = 1024, features: int = 4, dimension: int = 32, rows: int = 5000, state_bits: int = 8):
    """Trains on synthetic preferences; returns (first loss, last loss, loss served in 8 bits)."""
    eps, dense = load_package()
    rng = np.random.default_rng(3)
    taste = rng.normal(size=(features, rows)).astype(np.float32)       # what each id adds to a click's odds
    store = eps.ParameterStore(device=0, state_bytes=1 << 30)
    store.create_table(eps.TableDefinition(id=1, dimension=dimension, key_space=features * rows, learning_rate=0.02))
    block = ExpertBlock(dense, features, dimension, state_bits=state_bits)

    def draw():
        bags = rng.integers(1, 6, size=(features, batch))
        inputs, odds = [], np.zeros(batch, np.float32)
        for f in range(features):
            offsets = np.concatenate([[0], np.cumsum(bags[f])]).astype(np.int64)
            ids = rng.integers(0, rows, size=int(offsets[-1]))
            odds += np.add.reduceat(taste[f][ids], offsets[:-1]) / bags[f]
            inputs.append(eps.FeatureInput(1, f, eps.MEAN, torch.from_numpy(ids + f * rows).cuda(), torch.from_numpy(offsets).cuda()))
        return inputs, torch.from_numpy((odds > 0).astype(np.float32)).cuda()

    def loss_of(score, clicked):
        return torch.nn.functional.binary_cross_entropy_with_logits(score, clicked)

    losses = []
    for _ in range(steps):
        inputs, clicked = draw()
        stream = torch.cuda.current_stream()
        ticket, pooled = store.lookup(inputs, stream=stream)
        x = torch.cat(pooled, dim=1)
        score, kept = block.forward(x)
        losses.append(loss_of(score, clicked).item())
        dx = block.backward((torch.sigmoid(score) - clicked) / batch, kept)
        store.push(ticket, [d.contiguous() for d in dx.split(dimension, dim=1)], stream=stream)
        block.optimizer.step()
        block.rebalance(kept[2])

    served, plain = [], []
    scored = block.serve()
    for _ in range(8):
        inputs, clicked = draw()
        _, pooled = store.lookup(inputs, read_only=True, stream=torch.cuda.current_stream())
        x = torch.cat(pooled, dim=1)
        served.append(loss_of(scored(x), clicked).item())
        plain.append(loss_of(block.forward(x)[0], clicked).item())
    store.close()
    return losses[0], float(np.mean(plain)), float(np.mean(served))


if __name__ == "__main__":
    a = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    a.add_argument("--steps", type=int, default=150)
    a.add_argument("--state-bits", type=int, default=8, choices=(8, 32))
    a = a.parse_args()
    start, plain, served = run(steps=a.steps, state_bits=a.state_bits)
    print(f"loss {start:.4f} at the start, {plain:.4f} after {a.steps} steps, {served:.4f} served in 8 bits")
