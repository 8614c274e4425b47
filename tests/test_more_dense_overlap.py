"""Tensors of the newer dense operators' C calls that may not share memory: refused before a GPU is looked for."""
import pytest
import torch

from conftest import gpu_available, import_package
from test_more_dense_abi import A, LIB, balance, norm, refused

eps = import_package()
from eps_b200 import dense  # noqa: E402

gpu = pytest.mark.gpu
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


def gradient(out, out_stride=16, add=None, add_stride=16, **change):
    """logits [8, 16] of floats at A, each row 64 bytes of 128"""
    return refused(LIB.eps_b200_balance_loss_backward, balance(**{**dict(logits_stride=32), **change}), 64 * A, 64 * A, None, add, add_stride,
                   out, out_stride, None)


@pytest.mark.parametrize("out,how", [(A, dict()), (A, dict(out_stride=48)), (A + 4, dict(out_stride=32)), (A + 60, dict(out_stride=32)),
                                     (A - 4, dict(out_stride=32)), (A + 128 * 7 + 60, dict()), (A - 64 * 8 + 4, dict()),
                                     (A + 128 * 7, dict(out_stride=-32)), (A + 128 * 7 + 64, dict(out_stride=-16)),
                                     (A * 8, dict(add=A * 8, add_stride=0)), (A * 8, dict(add=A * 8 + 4)), (A * 8, dict(add=A * 8, add_stride=20)),
                                     (A * 8, dict(add=A * 8 - 8 * 64 + 4)), (A * 8, dict(out_stride=15)), (A * 8, dict(out_stride=0)),
                                     (A * 8, dict(out_stride=-15)), (A * 8, dict(add=A * 8 - 128, add_stride=(1 << 62) + 5))])
def test_a_gradient_is_not_written_where_others_are_read(out, how):
    assert gradient(out, **how) == eps.INVALID_ARGUMENT


@pytest.mark.skipif(gpu_available(), reason="checks the no-GPU failure path")
@pytest.mark.parametrize("out,how", [(A, dict(out_stride=32)), (A + 64, dict(out_stride=32)), (A - 64, dict(out_stride=32)), (A - 64 * 8, dict()),
                                     (A + 128 * 7 + 64, dict()), (A + 128 * 7 + 64, dict(out_stride=-32)), (A * 8, dict(add=A * 8)),
                                     (A * 8, dict(add=A)), (A * 8, dict(add=A, add_stride=0)), (A, dict(out_stride=0, tokens=1)),
                                     (A + 64, dict(out_stride=0, tokens=1)), (A * 8, dict(out_stride=-16)), (A * 8, dict(add=A * 8 + 64 * 8))])
def test_a_gradient_is_written_in_place_and_beside(out, how):
    assert gradient(out, **how) in (eps.UNAVAILABLE, eps.RUN_FAILED)


@gpu
@pytest.mark.parametrize("tokens,E", [(1, 8), (3, 128), (2000, 64), (700, 63), (5000, 12), (300, 1000)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("flip", [False, True])
def test_a_gradient_in_the_place_of_the_logits(tokens, E, dtype, flip):
    """Bit for bit that of a call with tensors apart, rows in either order."""
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(tokens, E, generator=g, device="cuda").to(dtype)
    add = torch.randn(tokens, E, generator=g, device="cuda").to(dtype)
    chosen = torch.randint(0, E, (tokens, 2), generator=g, device="cuda", dtype=torch.int32)
    mask = torch.rand(tokens, generator=g, device="cuda") < 0.7
    r = dense.balance_loss(x, chosen, mask=mask)
    want = dense.balance_loss_backward(x, r.counts, r.tokens, 2, mask=mask, add=add)
    if flip:
        x, add, want, mask = x.flip(0), add.flip(0), want.flip(0), mask.flip(0)
    at, stride = (x[-1].data_ptr(), -E) if flip else (x.data_ptr(), E)
    plus = add[-1].data_ptr() if flip else add.data_ptr()
    kept = mask.flip(0).contiguous() if flip else mask
    args = bytes(dense.BalanceLossArgs(device=0, type=dense._TYPES[dtype], score=0, normalise=1, experts=E, top_k=2, tokens=tokens, weight=1.0,
                                       logits=at, logits_stride=stride, mask=kept.data_ptr()))
    assert refused(LIB.eps_b200_balance_loss_backward, args, r.counts.data_ptr(), r.tokens.data_ptr(), None, plus, stride, at, stride,
                   torch.cuda.current_stream().cuda_stream) == 0
    assert torch.equal(x, want)
