"""Tensors of the newer dense operators' C calls that may not share memory: refused before a GPU is looked for."""
import pytest

from conftest import gpu_available, import_package
from test_more_dense_abi import A, LIB, norm, refused

eps = import_package()

WORK = 8 * 1000      # bytes of the workspace of 1000 blocks
NORM = dict(workspace=A + 4096, workspace_bytes=WORK)


@pytest.mark.parametrize("blocks", [3, 1000])
@pytest.mark.parametrize("change", [dict(gradient_scale=A), dict(gradient_scale=A + 4), dict(gradient_scale=A + 8), dict(gradient_scale=A + 2),
                                    dict(gradient_scale=A - 2)])
def test_a_norm_is_not_scaled_by_its_own_result(blocks, change):
    assert refused(LIB.eps_b200_gradient_norm, norm(blocks=blocks, **NORM, **change), None) == eps.INVALID_ARGUMENT


@pytest.mark.parametrize("change", [dict(gradient_scale=A + 4096), dict(gradient_scale=A + 4096 + WORK - 4)])
def test_a_norm_is_not_scaled_by_its_workspace(change):
    assert refused(LIB.eps_b200_gradient_norm, norm(**{**NORM, **change}), None) == eps.INVALID_ARGUMENT


@pytest.mark.skipif(gpu_available(), reason="checks the no-GPU failure path")
@pytest.mark.parametrize("change", [dict(gradient_scale=A + 12), dict(gradient_scale=A - 4), dict(gradient_scale=A + 4096 + WORK),
                                    dict(gradient_scale=A + 4096, blocks=3)])
def test_a_norm_takes_what_lies_beside(change):
    assert refused(LIB.eps_b200_gradient_norm, norm(**{**NORM, **change}), None) in (eps.UNAVAILABLE, eps.RUN_FAILED)
