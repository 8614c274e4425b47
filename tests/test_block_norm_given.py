"""block_norm where tensors are not given: what is wanted is written all the same, and what belongs to the
missing tensors leaves no trace.  One column with a gate for each row."""
import ctypes as C
import math

import pytest
import torch

import dense_reference as ref
from conftest import import_package
from test_block_norm import values

eps = import_package()
from eps_b200 import dense  # noqa: E402

gpu = pytest.mark.gpu


def backward(args, **gradients):
    st = eps.Status()
    given = {k: v.data_ptr() if torch.is_tensor(v) else v for k, v in gradients.items()}
    rc = dense._lib.eps_b200_block_norm_backward(bytes(args), bytes(dense.BlockNormGradientArgs(**given)),
                                                 torch.cuda.current_stream().cuda_stream, C.byref(st))
    return rc, st.message


@gpu
@pytest.mark.parametrize("columns", [40, 33, 2048])
@pytest.mark.parametrize("kind", [0, 1])
def test_wanted_gradients_are_written_where_nothing_comes_in(columns, kind):
    """Without dh and dz the gradients of the norm's weight and bias are zeros, whatever else is asked for."""
    rows = 7
    args = dense.BlockNorm(device=0, kind=kind, pre_norm=1, type=0, residual_type=0, parameter_type=0, columns=columns, rows=rows, epsilon=1e-5, scale=1.0)
    h = values(1, rows, columns)
    space = dense._lib.eps_b200_block_norm_workspace(rows, columns)
    workspace = torch.empty(space, dtype=torch.uint8, device="cuda")
    for more in ({}, {"h": h, "h_stride": columns}):
        w, b = (torch.full((columns,), 7.0, device="cuda") for _ in range(2))
        rc, message = backward(args, dpre_weight=w, dpre_bias=b, workspace=workspace, workspace_bytes=space, **more)
        assert rc == 0, message
        assert not w.any() and not b.any()
    rc, _ = backward(args, dpre_weight=w)
    assert rc == eps.INVALID_ARGUMENT              # sums need their workspace
    assert backward(args)[0] == 0                  # nothing comes in and nothing is asked for


@gpu
@pytest.mark.parametrize("columns", [48, 33, 1024])
@pytest.mark.parametrize("kind", ["rms", "layer"])
def test_what_belongs_to_missing_tensors_leaves_no_trace(columns, kind):
    x, y, g = values(1, 5, columns), values(2, 5, columns), values(3, 5, columns)
    bad = torch.ones(columns, device="cuda")
    bad[3], bad[4] = math.inf, math.nan
    # no block output: its scale and weights do not matter
    want = dense.block_norm(x, kind=kind)
    for more in (dict(scale=math.inf), dict(channel_scale=bad), dict(post_weight=bad, post_bias=bad), dict(activation="silu")):
        h, z = dense.block_norm(x, kind=kind, **more)
        assert h is x and torch.equal(z, want[1])
        got = dense.block_norm_backward(x, g, x, kind=kind, **more)
        assert torch.equal(got.x, dense.block_norm_backward(x, g, x, kind=kind).x)
    # no gradient by way of the norm after: its weight does not matter
    want = dense.block_norm_backward(g, None, x, y, g, kind=kind, pre_weight=torch.ones(columns, device="cuda"))
    got = dense.block_norm_backward(g, None, x, y, g, kind=kind, pre_weight=bad, pre_bias=bad)
    assert torch.equal(got.x, g) and torch.equal(got.y, want.y) and torch.equal(got.gate, want.gate)
    assert not got.pre_weight.any() and not got.pre_bias.any()
    # a norm that is left out, with weights
    h, z = dense.block_norm(x, y, post_norm=False, pre_norm=False, post_weight=bad, pre_weight=bad)
    assert z is None and torch.equal(h, x + y)


@gpu
def test_one_column_with_a_gate_for_each_row():
    x, y, g = values(1, 6, 1), values(2, 6, 1), values(3, 6)
    w = values(4, 1)
    how = dict(post_norm=False, pre_norm=False, channel_scale=w, scale=0.5)
    h, _ = dense.block_norm(x, y, g, **how)
    assert torch.equal(h, dense.block_norm(x, y, g[:, None], **how)[0])
    ref.close(h, x.double() + 0.5 * w.double() * torch.sigmoid(g.double())[:, None] * y.double(), x.abs() + y.abs())
    got, want = (dense.block_norm_backward(x, None, h, y, gate, **how) for gate in (g, g[:, None]))
    assert got.gate.shape == (6,) and torch.equal(got.gate, want.gate[:, 0]) and torch.equal(got.y, want.y)
