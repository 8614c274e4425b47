"""Addresses that a kernel could not read in the type of what lies there: C calls with them are refused before a GPU is
looked for."""
import pytest

from conftest import gpu_available, import_package
from test_more_dense_abi import A, LIB, balance, low_rank, norm, refused

eps = import_package()
GONE = (eps.UNAVAILABLE, eps.RUN_FAILED)


@pytest.mark.parametrize("change", [dict(gradient_scale=8 * A + 2), dict(gradient_scale=8 * A + 1), dict(result=8 * A + 2)])
def test_gradient_norm(change):
    assert refused(LIB.eps_b200_gradient_norm, norm(**change), None) == eps.INVALID_ARGUMENT


@pytest.mark.parametrize("kind,off", [(0, 2), (0, 1), (1, 1), (2, 1)])
def test_balance_loss_rows(kind, off):
    for change in (dict(logits=A + off), dict(logits=A + off, tokens=1)):
        a = balance(type=kind, **change)
        assert refused(LIB.eps_b200_balance_loss, a, A, A, A, A, A, None, 0, None) == eps.INVALID_ARGUMENT
        assert refused(LIB.eps_b200_balance_loss_backward, a, A, A, A, None, 0, 2 * A, 16, None) == eps.INVALID_ARGUMENT
    for add, out in ((3 * A + off, 2 * A), (3 * A, 2 * A + off), (None, 2 * A + off)):
        assert refused(LIB.eps_b200_balance_loss_backward, balance(type=kind), A, A, A, add, 16, out, 16, None) == eps.INVALID_ARGUMENT


def test_balance_loss_words():
    for i in range(5):
        args = [A] * 5
        args[i] = A + 2
        assert refused(LIB.eps_b200_balance_loss, balance(), *args, None, 0, None) == eps.INVALID_ARGUMENT
    for i in range(3):
        args = [A] * 3
        args[i] = A + 2
        assert refused(LIB.eps_b200_balance_loss_backward, balance(), *args, None, 0, 2 * A, 16, None) == eps.INVALID_ARGUMENT


@pytest.mark.parametrize("kind,off", [(0, 2), (0, 1), (1, 1), (2, 1)])
@pytest.mark.parametrize("which", ["x", "base", "out"])
@pytest.mark.parametrize("rows", [1, 4])
def test_adapter_rows(kind, off, which, rows):
    places = dict(x=A, base=2 * A, out=3 * A)
    assert refused(LIB.eps_b200_low_rank, low_rank(type=kind, rows=rows, **{**places, which: places[which] + off}), None) == eps.INVALID_ARGUMENT


@pytest.mark.parametrize("change", [dict(scale=A + 2), dict(ids=A + 2), dict(ids=A + 1)])
def test_adapter_words(change):
    assert refused(LIB.eps_b200_low_rank, low_rank(**change), None) == eps.INVALID_ARGUMENT


@pytest.mark.skipif(gpu_available(), reason="checks the no-GPU failure path")
def test_aligned_to_the_type_is_enough():
    assert refused(LIB.eps_b200_low_rank, low_rank(x=A + 2, base=2 * A + 2, out=3 * A + 2), None) in GONE
    assert refused(LIB.eps_b200_low_rank, low_rank(type=0, x=A + 4, base=2 * A + 4, out=3 * A + 4, scale=A + 4, ids=A + 4), None) in GONE
    assert refused(LIB.eps_b200_balance_loss, balance(type=1, logits=A + 2), A + 4, A + 4, A + 4, A + 4, A + 4, None, 0, None) in GONE
    assert refused(LIB.eps_b200_balance_loss_backward, balance(type=2, logits=A + 2), A, A, A, 3 * A + 2, 16, 2 * A + 2, 16, None) in GONE
    assert refused(LIB.eps_b200_gradient_norm, norm(gradient_scale=8 * A + 4, result=A + 4), None) in GONE
