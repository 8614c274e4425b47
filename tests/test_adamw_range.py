"""AdamW at the ends of its range: moments below float32's normal numbers, the smallest epsilons, and
tensors without elements."""
import pytest
import torch

from conftest import import_package

import_package()
from eps_b200 import dense  # noqa: E402

gpu = pytest.mark.gpu


@gpu
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("epsilon", [1e-25, 1e-37, 1e-42, 1e-60])
def test_small_gradients_under_a_small_epsilon(bits, epsilon):
    """The first step moves a parameter by the learning rate, however small the gradient."""
    rate, beta2, size = 0.25, 0.98, 1e-20
    g = torch.full((300,), size, device="cuda")
    g[::3] *= -1
    p = torch.zeros(300, device="cuda")
    dense.AdamW([p], [g], state_bits=bits, learning_rate=rate, beta2=beta2, epsilon=epsilon, weight_decay=0.0).step()
    # v = 0.02 g^2 = 2e-42 is subnormal: four roundings of 2^-150 on its way, half of that in the root, and
    # float32's roundings behind it (epsilon itself, against a root of 1.4e-21, is below 1e-3 in all cases)
    v = (1 - beta2) * size * size
    off = 4 * 2.0 ** -150 / v / 2 + 64 * 2.0 ** -24 + epsilon / size
    want = -rate * torch.sign(g.double())
    assert bool(((p.double() - want).abs() <= rate * off).all())


@gpu
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("epsilon", [1e-42, 1e-60])
def test_no_gradient_under_the_smallest_epsilons(bits, epsilon):
    p, g = torch.ones(300, device="cuda"), torch.zeros(300, device="cuda")
    dense.AdamW([p], [g], state_bits=bits, epsilon=epsilon, weight_decay=0.0).step()
    assert bool((p == 1).all())


@gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_nothing_to_update(bits):
    p = [torch.empty(0, device="cuda"), torch.empty(0, 4, device="cuda")]
    opt = dense.AdamW(p, [torch.empty_like(t) for t in p], state_bits=bits)
    opt.step()
    assert opt.steps == 1
