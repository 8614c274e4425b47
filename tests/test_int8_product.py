"""8-bit products against exact integer sums: ragged groups, odd sizes, gathered rows, both kernels, and
rows that cannot be quantized."""
import math

import pytest
import torch

import dense_reference as ref
from conftest import import_package

import_package()
from eps_b200 import EpsError, INVALID_ARGUMENT, dense  # noqa: E402

gpu = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def quantized(x):
    """(q, scale) by the definition, whose float32 roundings are part of it (127 / top is 127 * (1 / top)
    here as there)."""
    top = x.float().abs().amax(-1, keepdim=True)
    q = torch.round(x.float() * torch.where(top < 2.0 ** -120, 0.0, 127 * top.reciprocal()))
    return q, torch.where(top < 2.0 ** -120, 0.0, (top.double() / 127).float())


def offsets_of(sizes):
    return torch.tensor([0, *torch.tensor(sizes).cumsum(0).tolist()], dtype=torch.int32, device="cuda")


def check(sizes, channels, inner, dtype=F32, bias=False, rows=None, divisor=1, tokens=None, x=None, seed=1):
    experts, n = len(sizes), sum(sizes)
    g = gen(seed)
    if x is None:
        x = torch.randn(tokens if tokens is not None else n, inner, generator=g, device="cuda").to(dtype)
    w = torch.randint(-127, 128, (experts, channels, inner), generator=g, device="cuda", dtype=torch.int8)
    ws = torch.rand(experts, channels, generator=g, device="cuda") / 1000 + 1e-4
    b = torch.randn(experts, channels, generator=g, device="cuda") if bias else None
    layer = dense.QuantizedExperts(w, ws, b)
    out = layer.product(x, offsets=None if experts == 1 and seed % 2 else offsets_of(sizes), rows=rows, rows_divisor=divisor)
    assert out.dtype == x.dtype and out.shape == (n, channels)
    q, s = quantized(x)
    if rows is not None:
        q, s = q[rows.long() // divisor], s[rows.long() // divisor]
    at = 0
    for e, k in enumerate(sizes):
        total = q[at:at + k].double() @ w[e].double().T          # exact: below 2^53
        want = total * s[at:at + k].double() * ws[e].double()
        size = want.abs() + (0 if b is None else b[e].double().abs())
        want = want if b is None else want + b[e].double()
        ref.close(out[at:at + k], want, size)
        at += k
    return out


@gpu
@pytest.mark.parametrize("inner", [1, 15, 16, 17, 100, 128, 130, 1000, 4112])
@pytest.mark.parametrize("channels", [1, 7, 64, 129, 264])
def test_sizes(inner, channels):
    for n in (1, 3, 9, 40, 200):
        check([n], channels, inner, seed=n)


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_types_with_bias(dtype):
    check([5], 96, 256, dtype, bias=True)
    check([150], 96, 250, dtype, bias=True)
    check([700], 520, 384, dtype, bias=True)


@gpu
@pytest.mark.parametrize("sizes", [[0, 0, 7], [1, 0, 2, 0], [130, 0, 1, 64, 300, 0, 17, 128], [0, 0, 0], [3] * 40, [257, 511],
                                   [1] * 100 + [900], [5] * 300 + [0] * 20 + [70], [0] * 299 + [400]])
def test_ragged_groups(sizes):
    check(sizes, 136, 200, bias=True)
    check(sizes, 64, 64, BF16)


@gpu
def test_many_rows():
    check([3000], 1000, 520, BF16)
    check([1500, 2, 1300], 260, 1040, BF16, bias=True)


@gpu
def test_gathered_rows():
    rows = torch.randint(0, 60 * 4, (333,), generator=gen(3), device="cuda", dtype=torch.int32)
    check([100, 0, 233], 72, 144, BF16, rows=rows, divisor=4, tokens=60)
    check([333], 72, 144, F32, rows=rows // 4, tokens=60)
    check([2], 40, 48, rows=torch.tensor([1, 0], dtype=torch.int32, device="cuda"), tokens=2)


@gpu
def test_with_a_routing():
    """The experts' products of routed tokens, joined again with their weights."""
    x = torch.randn(90, 64, generator=gen(5), device="cuda")
    r = dense.route(torch.randn(90, 6, generator=gen(6), device="cuda"), 2)
    layer = dense.QuantizedExperts.from_weights(torch.randn(6, 48, 64, generator=gen(7), device="cuda"))
    out = layer.product(x, offsets=r.offsets, rows=r.order, rows_divisor=2)
    joined = (out[r.position.long()] * r.weights[..., None]).sum(1)
    q, s = quantized(x)
    w = layer.weight[..., :64].double() * layer.scale.double()[..., None]
    each = torch.einsum("tk,enk->ten", (q * s).double(), w)
    want = (each.gather(1, r.experts.long()[..., None].expand(-1, -1, 48)) * r.weights.double()[..., None]).sum(1)
    ref.close(joined, want, each.abs().amax(1) * 2)


@gpu
def test_strides_and_alignment():
    room = torch.randn(70, 300, generator=gen(8), device="cuda").to(BF16)
    for view in (room[:, 3:131], room[:, :128], room[::2, 8:136], room[:1, 1:129]):
        check([view.shape[0]], 80, 128, x=view)
    expanded = room[:1, :128].expand(20, 128)
    check([20], 16, 128, x=expanded)


@gpu
def test_sum_is_exact_at_its_largest():
    """All products of one sign over the longest inner size: just below 2^31."""
    x = torch.ones(2, 131072, device="cuda")
    w = torch.full((1, 3, 131072), 127, dtype=torch.int8, device="cuda")
    w[0, 1] = -127
    layer = dense.QuantizedExperts(w, torch.ones(1, 3, device="cuda"))
    out = layer.product(x)
    want = 127.0 * 127 * 131072 / 127
    assert torch.equal(out.double().cpu(), torch.tensor([[want, -want, want]] * 2, dtype=torch.float64))
    out = layer.product(x[:1].expand(300, 131072))
    assert bool((out.abs().double() == want).all())


@gpu
def test_quantize_rows():
    x = torch.randn(17, 100, generator=gen(9), device="cuda") * 3
    x[2] = 0
    x[3] = 1e-38
    x[4, 7], x[5, 8] = math.nan, -math.inf
    q, s = dense.quantize_rows(x)
    assert q.shape == (17, 112) and not q[:, 100:].any()
    wq, ws = quantized(x)
    fine = [0, 1, 2, 3, *range(6, 17)]
    assert torch.equal(q[fine, :100].float(), wq[fine]) and torch.equal(s[fine], ws[fine, 0])
    assert s[4].isnan() and s[5].isnan() and not q[3].any() and s[3] == 0
    assert int(q.abs().max()) == 127
    half = torch.tensor([[127.0, 0.5, 1.5, 2.5, -0.5, -1.5, 126.5]], device="cuda")     # ties go to even
    assert dense.quantize_rows(half)[0][0, :7].tolist() == [127, 0, 2, 2, 0, -2, 126]
    rows = torch.tensor([3, -1, 40, 0], dtype=torch.int32, device="cuda")              # outside x: NaN scales
    q, s = dense.quantize_rows(x, rows, 2)
    assert s[1].isnan() and s[2].isnan() and s[3] == ws[0, 0] and s[0] == ws[1, 0]


@gpu
@pytest.mark.parametrize("n", [0, 3, 60, 400])
def test_product_of_quantized_rows(n):
    """eps_b200_int8_product on rows that were quantized before gives what the one call gives."""
    import ctypes as C
    import eps_b200
    layer = dense.QuantizedExperts.from_weights(torch.randn(2, 200, 144, generator=gen(20), device="cuda"))
    x = torch.randn(n, 144, generator=gen(21), device="cuda")
    off = offsets_of([n // 3, n - n // 3])
    q, s = dense.quantize_rows(x)
    out = torch.empty(n, 200, device="cuda")
    args = bytes(dense.Int8Product(device=0, type=0, experts=2, channels=200, inner=144, rows_divisor=1, rows=n, weight=layer.weight.data_ptr(),
                                   weight_scale=layer.scale.data_ptr(), offsets=off.data_ptr(), out=out.data_ptr()))
    st = eps_b200.Status()
    assert dense._lib.eps_b200_int8_product(args, q.data_ptr(), s.data_ptr(), torch.cuda.current_stream().cuda_stream, C.byref(st)) == 0, st.message
    assert torch.equal(out, layer.product(x, offsets=off))


@gpu
def test_a_bad_row_stays_alone():
    for n in (6, 300):
        x = torch.randn(n, 96, generator=gen(10), device="cuda")
        layer = dense.QuantizedExperts.from_weights(torch.randn(40, 96, generator=gen(11), device="cuda"))
        clean = layer.product(x)
        x[1, 3] = math.nan
        x[4] = 0
        out = layer.product(x)
        assert out[1].isnan().all() and not out[4].any()
        keep = [i for i in range(n) if i not in (1, 4)]
        assert torch.equal(out[keep], clean[keep])


@gpu
def test_offsets_outside_are_clamped():
    """Offsets are read on the GPU; what they say wrongly may cost rows, never touch other memory."""
    layer = dense.QuantizedExperts.from_weights(torch.randn(3, 40, 32, generator=gen(12), device="cuda"))
    x = torch.randn(20, 32, generator=gen(13), device="cuda")
    want = layer.product(x, offsets=offsets_of([5, 5, 10]))
    got = layer.product(x, offsets=torch.tensor([-7, 5, 10, 1000], dtype=torch.int32, device="cuda"))
    assert torch.equal(got, want)
    got = layer.product(x, offsets=torch.tensor([0, 5, 2, 20], dtype=torch.int32, device="cuda"))     # the second run is empty
    assert torch.equal(got[:2], want[:2])


@gpu
def test_stream_and_graph():
    layer = dense.QuantizedExperts.from_weights(torch.randn(2, 264, 200, generator=gen(14), device="cuda").to(BF16))
    for n in (4, 400):
        x = torch.randn(n, 200, generator=gen(15), device="cuda").to(BF16)
        off = offsets_of([n // 2, n - n // 2])
        want = layer.product(x, offsets=off)
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            late = torch.empty_like(x)
            torch.cuda._sleep(20_000_000)
            late.copy_(x)
            got = layer.product(late, offsets=off)
        torch.cuda.synchronize()
        assert torch.equal(got, want)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = layer.product(x, offsets=off)
        x.mul_(-2)
        graph.replay()
        assert torch.equal(got, layer.product(x, offsets=off))


@gpu
def test_refusals():
    w, s = torch.ones(2, 8, 16, dtype=torch.int8, device="cuda"), torch.ones(2, 8, device="cuda")
    layer = dense.QuantizedExperts(w, s)
    x = torch.ones(4, 16, device="cuda")
    off = offsets_of([1, 3])
    bad = [lambda: dense.QuantizedExperts(w.float(), s), lambda: dense.QuantizedExperts(w, s[:1]), lambda: dense.QuantizedExperts(w, None),
           lambda: dense.QuantizedExperts(w, s.double()), lambda: dense.QuantizedExperts(w[:0], s[:0]), lambda: dense.QuantizedExperts(w, s, s[:1]),
           lambda: layer.product(x), lambda: layer.product(x[:, :15], off), lambda: layer.product(x, off[:2]), lambda: layer.product(x, off.long()),
           lambda: layer.product(x, off, rows=off.long()), lambda: layer.product(x, off, rows=off, rows_divisor=0),
           lambda: layer.product(x.cpu(), off), lambda: layer.product(x.double(), off), lambda: layer.product(x.t().expand(16, 4).t().t(), off),
           lambda: dense.quantize_rows(torch.ones(1, 131073, device="cuda")), lambda: dense.quantize_rows(torch.ones(3, 0, device="cuda"))]
    for call in bad:
        with pytest.raises(EpsError) as e:
            call()
        assert e.value.code == INVALID_ARGUMENT
