"""A float block's gates in float precision over their whole range."""
import pytest
import torch

from conftest import import_package

import_package()
from eps_b200 import dense  # noqa: E402

gpu = pytest.mark.gpu
PLAIN = dict(post_norm=False, pre_norm=False)


@gpu
@pytest.mark.parametrize("row", [False, True])
@pytest.mark.parametrize("activation", ["sigmoid", "silu"])
@pytest.mark.parametrize("columns", [64, 33])
def test_gates_keep_float_precision(columns, activation, row):
    """h = act(gate) alone.  The power is good to 2^-22, what multiplies it to two roundings, the sum, the
    reciprocal (2^-23) and silu's product to one or two each: 12 roundings of 2^-24 hold them all."""
    rows = 4000
    g = torch.linspace(-86, 86, rows * (1 if row else columns), device="cuda").view(rows, -1)
    gate = g[:, 0].contiguous() if row else g
    x, y = torch.zeros(rows, columns, device="cuda"), torch.ones(rows, columns, device="cuda")
    h, _ = dense.block_norm(x, y, gate, activation=activation, **PLAIN)
    want = torch.sigmoid(g.double())
    want = (want * g.double() if activation == "silu" else want).expand(rows, columns)
    assert bool(((h.double() - want).abs() <= 12 * 2.0 ** -24 * want.abs()).all())
    if activation == "sigmoid" and not row:
        # the slope a - a^2 adds two roundings; above 0 it is a difference that cancels
        got = dense.block_norm_backward(y, None, h, y, gate, activation=activation, **PLAIN).gate[g < 0].double()
        want = (want * (1 - want))[g < 0]
        assert bool(((got - want).abs() <= 15 * 2.0 ** -24 * want).all())


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_gates_at_the_ends(dtype):
    """Open, closed and bad gates."""
    inf, nan = float("inf"), float("nan")
    g = torch.tensor([[inf, -inf, nan, 1e30, -1e30, 200.0, -200.0, 0.0]] * 3, device="cuda", dtype=dtype)
    x, y = torch.zeros(3, 8, device="cuda", dtype=dtype), torch.full((3, 8), 2.0, device="cuda", dtype=dtype)
    h = dense.block_norm(x, y, g, **PLAIN)[0][1].tolist()
    assert h[:2] == [2.0, 0.0] and h[2] != h[2] and h[3:] == [2.0, 0.0, 2.0, 0.0, 1.0]
    dg = dense.block_norm_backward(y, None, x, y, g, **PLAIN).gate[1]
    assert dg[2].isnan() and dg[7] == 1.0 and not dg[[0, 1, 3, 4, 5, 6]].any()
