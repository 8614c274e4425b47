"""Calls of the newer dense operators that Python does not make but C may, and several at once."""
import ctypes as C

import pytest
import torch

import dense_reference as ref
from conftest import import_package

eps = import_package()
from eps_b200 import dense  # noqa: E402

gpu = pytest.mark.gpu
LIB = eps.load_library()


def ok(fn, *args):
    st = eps.Status()
    assert fn(*args, C.byref(st)) == 0, st.message


def stream():
    return torch.cuda.current_stream().cuda_stream


@gpu
@pytest.mark.parametrize("E,dtype", [(64, torch.bfloat16), (63, torch.bfloat16), (40, torch.float32), (256, torch.float32)])
def test_balance_gradient_in_the_place_of_add_and_with_strides(E, dtype):
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(3000, E, generator=g, device="cuda").to(dtype)
    add = torch.randn(3000, E, generator=g, device="cuda").to(dtype)
    chosen = torch.randint(0, E, (3000, 2), generator=g, device="cuda", dtype=torch.int32)
    dloss = torch.tensor(3000.0, device="cuda")
    r = dense.balance_loss(x, chosen)
    want = dense.balance_loss_backward(x, r.counts, r.tokens, 2, dloss=dloss, add=add)
    args = bytes(dense.BalanceLossArgs(device=0, type=dense._TYPES[dtype], score=0, normalise=1, experts=E, top_k=2, tokens=3000, weight=1.0,
                                       logits=x.data_ptr(), logits_stride=E))
    ptrs = (r.counts.data_ptr(), r.tokens.data_ptr(), dloss.data_ptr())
    wide = torch.full((3000, E + 9), 7.0, dtype=dtype, device="cuda")
    ok(LIB.eps_b200_balance_loss_backward, args, *ptrs, add.data_ptr(), E, wide.data_ptr() + 5 * wide.element_size(), E + 9, stream())
    # other packs, so other sums: the same but for some units
    ref.close(wide[:, 5:5 + E], want.double(), 1 + want.double().abs())
    assert bool((wide[:, :5] == 7).all()) and bool((wide[:, 5 + E:] == 7).all())
    ok(LIB.eps_b200_balance_loss_backward, args, *ptrs, add.data_ptr(), E, add.data_ptr(), E, stream())
    assert torch.equal(add, want)


@gpu
@pytest.mark.parametrize("rows", [7, 300])
def test_adapters_without_scales(rows):
    g = torch.Generator(device="cuda").manual_seed(1)
    down, up = torch.randn(3, 16, 64, generator=g, device="cuda"), torch.randn(3, 32, 16, generator=g, device="cuda")
    x, ids = torch.randn(rows, 64, generator=g, device="cuda"), torch.randint(-1, 3, (rows,), generator=g, device="cuda", dtype=torch.int32)
    want = dense.Adapters(down, up).product(x, ids)
    out = torch.full((rows, 32), 7.0, device="cuda")
    space = LIB.eps_b200_low_rank_workspace(rows, 3)
    room = torch.empty(max(1, space), dtype=torch.uint8, device="cuda")
    args = bytes(dense.LowRank(device=0, type=0, adapters=3, rank=16, inner=64, channels=32, rows=rows, down=down.data_ptr(), up=up.data_ptr(),
                               ids=ids.data_ptr(), x=x.data_ptr(), out=out.data_ptr(), x_stride=64, out_stride=32,
                               workspace=room.data_ptr(), workspace_bytes=space))
    ok(LIB.eps_b200_low_rank, args, stream())
    assert torch.equal(out, want)


@gpu
@pytest.mark.parametrize("tokens,rows", [(30, 20), (4000, 700)])
def test_graphs_and_streams_at_once(tokens, rows):
    """Calls keep nothing between them: two graphs of the same calls replay at once, beside calls on a third stream."""
    g = torch.Generator(device="cuda").manual_seed(1)
    logits = torch.randn(tokens, 96, generator=g, device="cuda")
    chosen = torch.randint(0, 96, (tokens, 4), generator=g, device="cuda", dtype=torch.int32)
    a = dense.Adapters(torch.randn(5, 16, 256, generator=g, device="cuda"), torch.randn(5, 128, 16, generator=g, device="cuda"))
    x, ids = torch.randn(rows, 256, generator=g, device="cuda"), torch.randint(-1, 5, (rows,), generator=g, device="cuda", dtype=torch.int32)

    def calls():
        r = dense.balance_loss(logits, chosen, score="sigmoid")
        return [*r, dense.balance_loss_backward(logits, r.counts, r.tokens, 4, score="sigmoid"), a.product(x, ids)]
    want = [t.clone() for t in calls()]
    torch.cuda.synchronize()
    graphs, results, streams = [], [], [torch.cuda.Stream() for _ in range(3)]
    for s in streams[:2]:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            results.append(calls())
        graphs.append(graph)
    for _ in range(20):
        for t in (t for r in results for t in r):
            t.zero_()
        torch.cuda.synchronize()
        for graph, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                graph.replay()
        with torch.cuda.stream(streams[2]):
            last = calls()
        torch.cuda.synchronize()
        for r in (*results, last):
            assert all(torch.equal(p, q) for p, q in zip(r, want))


@gpu
def test_only_the_rows_of_a_padded_batch_are_written():
    """Rows behind those of the call, in buffers that hold more."""
    g = torch.Generator(device="cuda").manual_seed(1)
    a = dense.Adapters(torch.randn(2, 8, 64, generator=g, device="cuda"), torch.randn(2, 64, 8, generator=g, device="cuda"))
    for rows, all_rows in ((5, 64), (130, 256)):
        x = torch.randn(all_rows, 64, generator=g, device="cuda")
        out = torch.full((all_rows, 64), 7.0, device="cuda")
        ids = torch.randint(0, 2, (all_rows,), generator=g, device="cuda", dtype=torch.int32)
        a.product(x[:rows], ids[:rows], out=out[:rows])
        assert bool((out[rows:] == 7).all()) and not bool((out[:rows] == 7).any())
