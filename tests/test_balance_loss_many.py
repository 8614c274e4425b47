"""The balance loss's sums over many tokens are as exact as those over few, whatever the roundings of equal rows do."""
import pytest
import torch

import dense_reference as ref
from conftest import import_package

import_package()
from eps_b200 import dense  # noqa: E402

gpu = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16


@gpu
@pytest.mark.parametrize("T,E,dtype", [(1_200_000, 1000, BF16), (600_000, 1000, F32), (500_000, 1001, BF16), (900_000, 520, F32), (3_000_000, 96, BF16),
                                       (2_000_000, 33, F32), (6_000_000, 8, BF16), (9_000_000, 1, F32)])
@pytest.mark.parametrize("score,normalise", [("softmax", True), ("sigmoid", True), ("sigmoid", False)])
def test_equal_rows(T, E, dtype, score, normalise):
    """A share is within some ten units of 2^-24; equal shares, added 64 times, are off by 32 of them (each sum by one of its
    own size), by 3 over a warp's lanes and by 16 over a block's warps, the rest is added in double, and a block's sum is
    rounded once.  That is below CHAIN, whatever T."""
    row = torch.linspace(-2, 2, E).to(dtype)
    x = row.cuda().expand(T, E).contiguous()
    chosen = torch.zeros(T, 1, dtype=torch.int32, device="cuda")
    mask = torch.ones(T, dtype=torch.bool, device="cuda")
    mask[::7] = False
    p = torch.softmax(row.double(), -1) if score == "softmax" else torch.sigmoid(row.double())
    if normalise:
        p = p / p.sum()
    for m in (None, mask):
        n = T if m is None else int(mask.sum())
        got = dense.balance_loss(x, chosen, score=score, normalise=normalise, mask=m)
        want = (p * n).cuda()
        ref.close(got.mass, want, want)
        ref.close(got.loss, (E * p[0]).cuda(), E * p[0].cuda())
