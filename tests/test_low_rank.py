"""Low-rank adapters against 64 bits: rows of one, few and many adapters, ranks, odd widths, strides, what is not
finite, results in place, and their place beside an 8-bit layer."""
import math

import pytest
import torch

import dense_reference as ref
from conftest import import_package

import_package()
from eps_b200 import EpsError, INVALID_ARGUMENT, dense  # noqa: E402

gpu = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
# rows, adapters, rank, inner, channels
SHAPES = [(1, 1, 1, 1, 1), (1, 3, 8, 64, 64), (5, 4, 16, 100, 72), (17, 2, 16, 33, 31), (64, 5, 12, 256, 264), (64, 1, 4, 40, 40),
          (63, 2, 128, 96, 80), (65, 4, 16, 128, 64), (130, 3, 32, 512, 320), (128, 90, 8, 64, 40), (127, 1, 16, 72, 64), (129, 5, 16, 72, 64), (300, 300, 7, 96, 50), (1000, 7, 64, 200, 136),
          (200, 3, 128, 160, 96), (401, 2, 100, 2050, 40), (2500, 1, 16, 64, 1000), (150, 9, 40, 7, 9), (9000, 40, 8, 72, 24), (70, 5, 3, 31, 33)]


def make(rows, n, rank, K, N, dtype, seed=1):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rand = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    x, base = rand(rows, K).to(dtype), rand(rows, N).to(dtype)
    down, up = (rand(n, rank, K) / math.sqrt(K)).to(dtype), (rand(n, N, rank) / math.sqrt(rank)).to(dtype)
    scale = torch.rand(n, generator=g, device="cuda") + 0.5
    ids = torch.randint(-1, n, (rows,), generator=g, device="cuda", dtype=torch.int32)
    return x, base, down, up, scale, ids


def plain(x, ids, base, down, up, scale):
    """(out, size of its terms, size of u's share)"""
    out = torch.zeros(len(x), up.shape[1], dtype=torch.float64, device="cuda") if base is None else base.double().clone()
    size, part = out.abs(), torch.zeros_like(out)
    for a in range(len(down)):
        m = (ids == a).nonzero()[:, 0]
        d, w, s = down[a].double(), up[a].double(), 1.0 if scale is None else scale[a].double()
        u = x[m].double() @ d.T
        out[m] += s * (u @ w.T)
        part[m] = s * (u.abs() @ w.T.abs())
        size[m] += s * (x[m].double().abs() @ d.T.abs() @ w.T.abs())
    return out, size, part


def close(got, want, K, rank):
    """Within the rounding to got's type; a unit of 2^-23 of the terms for each matrix instruction in a row (its sums are
    cut off) and 32 more for joining; 2^-17 of u for its second 16-bit part (two roundings of 2^-9)."""
    value, size, part = want
    units = -(-K // 16) + -(-rank // 16) + 32
    limit = ref.UNIT[got.dtype] * value.abs() + units * 2.0 ** -23 * size + (0 if got.dtype == F32 else 2.0 ** -17) * part
    if got.dtype == F16:
        limit = limit + 2.0 ** -25
    off = (got.double() - value).abs()
    assert got.shape == value.shape and bool((off <= limit).all()), f"{(off / limit).max().item():.3g} of the limit"


@gpu
@pytest.mark.parametrize("rows,n,rank,K,N", SHAPES)
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_product(rows, n, rank, K, N, dtype):
    x, base, down, up, scale, ids = make(rows, n, rank, K, N, dtype)
    if rows > 3:
        ids[3] = n
        ids[2] = -7
    a = dense.Adapters(down, up, scale)
    want = plain(x, ids, base, down, up, scale)
    got = a.product(x, ids, base)
    close(got, want, K, rank)
    none = (ids < 0) | (ids >= n)
    assert torch.equal(got[none], base[none])
    assert torch.equal(got, a.product(x, ids, base))
    alone = a.product(x, ids)
    close(alone, plain(x, ids, None, down, up, scale), K, rank)
    assert not alone[none].any()
    place = base.clone()
    assert a.product(x, ids, place, out=place) is place
    assert torch.equal(place, got)
    close(dense.Adapters(down, up).product(x, ids, base), plain(x, ids, base, down, up, None), K, rank)


@gpu
@pytest.mark.parametrize("rows", [40, 200, 700])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_a_row_does_not_depend_on_the_others(rows, dtype):
    """Whatever the other rows hold and ask for, and wherever a row stands."""
    x, base, down, up, scale, ids = make(rows, 5, 16, 256, 128, dtype)
    a = dense.Adapters(down, up, scale)
    want = a.product(x, ids, base)
    p = torch.randperm(rows, generator=torch.Generator().manual_seed(3)).cuda()
    assert torch.equal(a.product(x[p], ids[p], base[p]), want[p])
    y, b = x.clone(), base.clone()
    y[1::2] = math.inf
    b[1::2] = math.nan
    got = a.product(y, ids, b)
    assert torch.equal(got[0::2], want[0::2])
    assert bool(torch.isnan(got[1::2]).all())


@gpu
@pytest.mark.parametrize("rows", [9, 100, 400])
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_what_is_not_finite(rows, dtype):
    """An infinity of x in a row: as the formula has it in 16 bits, NaN at the latest in float; padded ranks and
    inner places add nothing."""
    x, base, down, up, scale, ids = make(rows, 2, 5, 40, 24, dtype)
    ids.fill_(1)
    x[4, 7] = math.inf
    got = dense.Adapters(down, up, scale).product(x, ids, base)
    rest = torch.arange(rows, device="cuda") != 4
    assert bool(torch.isfinite(got[rest]).all()) and not bool(torch.isfinite(got[4]).any())
    if dtype != F32:
        want = plain(x, ids, base, down, up, scale)[0][4]
        assert torch.equal(torch.isnan(got[4]), torch.isnan(want)) and torch.equal(got[4].double().nan_to_num(0.0), want.nan_to_num(0.0))
    ids[4] = -1                          # a row without an adapter is its base, whatever x holds
    assert torch.equal(dense.Adapters(down, up, scale).product(x, ids, base)[4], base[4])
    base[3, 2], base[2, 1] = math.nan, -math.inf
    ids[3] = -1
    got = dense.Adapters(down, up, scale).product(x, ids, base)
    assert bool(torch.isnan(got[3, 2])) and got[2, 1] == -math.inf and int(torch.isfinite(got).logical_not().sum()) == 2


@gpu
@pytest.mark.parametrize("size", [2.0 ** -20, 1.0, 2.0 ** 12])
def test_float16_sums_beyond_its_range(size):
    """down x may leave float16's range on either side, as long as the result does not."""
    x, base, down, up, scale, ids = make(300, 3, 16, 512, 64, F16)
    down = (down.float() * size * 8).half()
    x = (x.float() * 256 * min(1.0, size * 16)).half()
    up = (up.float() / 64).half()
    scale = scale / size / 256 / min(1.0, size * 16)
    ids.clamp_(min=0)
    u = torch.einsum("tk,trk->tr", x.double(), down[ids.long()].double()).abs()
    assert size != 2.0 ** 12 or float(u.max()) > 65504
    a = dense.Adapters(down, up, scale)
    for part in (slice(0, 300), slice(0, 90), slice(0, 30)):
        close(a.product(x[part], ids[part], base[part]), plain(x[part], ids[part], base[part], down, up, scale), 512, 16)


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows", [33, 500])
@pytest.mark.parametrize("at", [0, 8, 3])
def test_strides(dtype, rows, at):
    x, base, down, up, scale, ids = make(rows, 4, 16, 64, 48, dtype)
    a = dense.Adapters(down, up, scale)
    want = a.product(x, ids, base)
    near = lambda got: close(got, plain(x, ids, base, down, up, scale), 64, 16)  # noqa: E731
    wide = torch.full((rows, 64 + 48 + 48 + 16), 7.0, dtype=dtype, device="cuda")
    xs, bs, os = wide[:, at:at + 64], wide[:, at + 64:at + 112], wide[:, at + 112:at + 160]
    xs.copy_(x)
    bs.copy_(base)
    got = a.product(xs, ids, bs, out=os)            # columns of one tensor
    assert got is os
    near(got)
    assert torch.equal(xs, x) and torch.equal(bs, base)
    assert bool((wide[:, :at] == 7).all()) and bool((wide[:, at + 160:] == 7).all())
    near(a.product(xs, ids, bs, out=bs))
    assert bool((wide[:, at + 160:] == 7).all()) and torch.equal(xs, x)
    row = base[:1].expand(rows, 48)                  # one row for all: a bias
    close(a.product(x, ids, row), plain(x, ids, row, down, up, scale), 64, 16)
    same = x[:1].expand(rows, 64)
    close(a.product(same, ids, base), plain(same, ids, base, down, up, scale), 64, 16)
    many = a.product(x[:30].view(5, 6, 64), ids[:30].view(5, 6), base[:30].view(5, 6, 48))
    assert many.shape == (5, 6, 48)
    close(many.view(30, 48), plain(x[:30], ids[:30], base[:30], down, up, scale), 64, 16)
    assert torch.equal(a.product(x, ids, base), want)


@gpu
def test_loading():
    x, base, down, up, scale, ids = make(200, 4, 16, 64, 48, BF16)
    a = dense.Adapters(down, up, scale)
    _, _, d, w, _, _ = make(1, 1, 6, 64, 48, BF16, 9)
    assert a.load(2, d[0], w[0], 0.5) is a
    down[2], up[2], scale[2] = 0, 0, 0.5
    down[2, :6], up[2, :, :6] = d[0], w[0]
    close(a.product(x, ids, base), plain(x, ids, base, down, up, scale), 64, 16)
    x, base, down, up, scale, ids = make(200, 4, 16, 64, 48, BF16)      # the tensors that it was made from are its own no more
    a = dense.Adapters(down, up, scale)
    want = a.product(x, ids, base)
    down.zero_()
    scale.zero_()
    assert torch.equal(a.product(x, ids, base), want)


@gpu
def test_no_rows():
    _, _, down, up, scale, _ = make(1, 4, 16, 64, 48, BF16)
    a = dense.Adapters(down, up, scale)
    out = a.product(torch.empty(0, 64, dtype=BF16, device="cuda"), torch.empty(0, dtype=torch.int32, device="cuda"))
    assert out.shape == (0, 48)


@gpu
def test_rows_beyond_32_bits():
    """Rows whose places pass 2^32 bytes, in x, base and out."""
    g = torch.Generator(device="cuda").manual_seed(1)
    T, K, N = 540000, 4096, 4096
    down, up = torch.randn(3, 8, K, generator=g, device="cuda").bfloat16() / 64, torch.randn(3, N, 8, generator=g, device="cuda").bfloat16()
    x, base = torch.zeros(T, K, dtype=BF16, device="cuda"), torch.zeros(T, N, dtype=BF16, device="cuda")
    rows = torch.cat([torch.arange(40, device="cuda"), torch.randint(0, T, (200,), generator=g, device="cuda"), torch.arange(T - 40, T, device="cuda")]).unique()
    x[rows] = torch.randn(len(rows), K, generator=g, device="cuda").bfloat16()
    base[rows] = torch.randn(len(rows), N, generator=g, device="cuda").bfloat16()
    ids = (torch.arange(T, device="cuda") % 4).int() - 1
    a = dense.Adapters(down, up)
    assert a.product(x, ids, base, out=base) is base
    small = torch.zeros(len(rows), N, dtype=BF16, device="cuda")
    want = plain(x[rows], ids[rows], small, down, up, None)
    g = torch.Generator(device="cuda").manual_seed(1)
    torch.randn(3, 8, K, generator=g, device="cuda"), torch.randn(3, N, 8, generator=g, device="cuda")
    torch.randint(0, T, (200,), generator=g, device="cuda"), torch.randn(len(rows), K, generator=g, device="cuda")
    start = torch.randn(len(rows), N, generator=g, device="cuda").bfloat16()
    close(base[rows], (want[0] + start.double(), want[1] + start.double().abs(), want[2]), K, 8)
    base[rows] = 0
    for part in base.split(1 << 16):
        assert not part.any()


@gpu
def test_many_adapters():
    g = torch.Generator(device="cuda").manual_seed(1)
    n = 16384
    down, up = torch.randn(n, 2, 8, generator=g, device="cuda"), torch.randn(n, 8, 2, generator=g, device="cuda")
    x = torch.randn(3000, 8, generator=g, device="cuda")
    ids = torch.randint(0, n, (3000,), generator=g, device="cuda", dtype=torch.int32)
    ids[5], ids[6] = n - 1, 0
    got = dense.Adapters(down, up).product(x, ids)
    i = ids.long()
    u = torch.einsum("tk,trk->tr", x.double(), down[i].double())
    want = torch.einsum("tr,tnr->tn", u, up[i].double())
    size = torch.einsum("tr,tnr->tn", torch.einsum("tk,trk->tr", x.double().abs(), down[i].double().abs()), up[i].double().abs())
    close(got, (want, size, size), 8, 2)


@gpu
@pytest.mark.parametrize("rows", [20, 700])
def test_captured_and_beside_an_8_bit_layer(rows):
    """A served layer: the shared product in 8 bits, adapters added in place, in a graph replayed for other requests."""
    x, _, down, up, scale, ids = make(rows, 6, 16, 128, 96, BF16)
    layer = dense.QuantizedExperts.from_weights(torch.randn(96, 128, device="cuda"))
    a = dense.Adapters(down, up, scale)

    def serve(x, ids):
        out = layer.product(x)
        return a.product(x, ids, out, out=out)
    want = serve(x, ids)
    base = layer.product(x)
    close(want, plain(x, ids, base, down, up, scale), 128, 16)
    held, asked = torch.zeros_like(x), torch.full_like(ids, -1)
    graph = torch.cuda.CUDAGraph()
    serve(held, asked)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        out = serve(held, asked)
    graph.replay()
    assert not out.any()
    held.copy_(x)
    asked.copy_(ids)
    graph.replay()
    assert torch.equal(out, want)


@gpu
def test_streams():
    """Calls on several streams at once, and adapters dropped while a call reads them."""
    x, base, down, up, scale, ids = make(500, 6, 16, 512, 256, BF16)
    a = dense.Adapters(down, up, scale)
    want = a.product(x, ids, base)
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(4)], []
    for s in streams * 4:
        with torch.cuda.stream(s):
            got.append(a.product(x, ids, base))
    torch.cuda.synchronize()
    assert all(torch.equal(g, want) for g in got)
    old = [(t.data_ptr(), t.numel() * t.element_size()) for t in (a.down, a.up, a.scale)]
    with torch.cuda.stream(streams[0]):
        torch.cuda._sleep(1_000_000_000)
        last = a.product(x, ids, base)
        done = torch.cuda.Event()
        done.record()
    del a
    fresh = {torch.empty(b, dtype=torch.uint8, device="cuda").data_ptr() for _, b in old for _ in range(4)}
    assert not done.query()            # else nothing is shown
    assert not any(p in fresh for p, _ in old)
    done.synchronize()
    assert torch.equal(last, want)


@gpu
def test_refusals():
    x, base, down, up, scale, ids = make(10, 4, 8, 32, 32, F32)
    a = dense.Adapters(down, up, scale)
    wide = torch.zeros(10, 80, device="cuda")
    bad = [lambda: dense.Adapters(down[0], up[0]), lambda: dense.Adapters(down, up[:3]), lambda: dense.Adapters(down, up[..., :4]),
           lambda: dense.Adapters(down, up.half()), lambda: dense.Adapters(down.double(), up.double()), lambda: dense.Adapters(down, up, scale[:2]),
           lambda: dense.Adapters(down.cpu(), up), lambda: dense.Adapters(torch.zeros(1, 129, 4, device="cuda"), torch.zeros(1, 4, 129, device="cuda")),
           lambda: dense.Adapters(torch.zeros(16385, 1, 1, device="cuda"), torch.zeros(16385, 1, 1, device="cuda")),
           lambda: a.product(x[:, :31], ids), lambda: a.product(x.half(), ids), lambda: a.product(x, ids[:9]), lambda: a.product(x, ids.long()),
           lambda: a.product(x, ids, base[:9]), lambda: a.product(x, ids, base.half()), lambda: a.product(x, ids, base, out=x),
           lambda: a.product(x, ids, base, out=base[:, :31]), lambda: a.product(x, ids, base, out=torch.zeros(1, 32, device="cuda").expand(10, 32)),
           lambda: a.product(wide[:, :32], ids, out=wide[:, 31:63]), lambda: a.product(x, ids, wide[:, :32], out=wide[:, 16:48]),
           lambda: a.product(x, ids, base[:1].expand(10, 32), out=base), lambda: a.load(4, down[0], up[0]), lambda: a.load(-1, down[0], up[0]),
           lambda: a.load(0, down[0, :, :31], up[0]), lambda: a.load(0, down[0].half(), up[0]), lambda: a.load(0, down[0], up[0, :, :7]),
           lambda: a.product(x.cpu(), ids), lambda: a.product(x, ids.cpu())]
    for i, call in enumerate(bad):
        with pytest.raises(EpsError) as e:
            call()
        assert e.value.code == INVALID_ARGUMENT, i
