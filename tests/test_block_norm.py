"""block_norm and its gradients against a 64-bit restatement: widths from one column to the most,
rows from none, odd strides and alignments, every gate, and the parts that may be left out."""
import itertools

import pytest
import torch

import dense_reference as ref
from conftest import import_package

import_package()
from eps_b200 import EpsError, INVALID_ARGUMENT, dense  # noqa: E402

gpu = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
EPS = 1e-5


def values(seed, *shape, scale=1.0, dtype=F32):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)


def strided(t, pad, shift):
    """t with `pad` columns between its rows, beginning `shift` elements off an aligned address."""
    rows, columns = t.shape
    room = torch.zeros(rows * (columns + pad) + shift, dtype=t.dtype, device=t.device)
    v = room[shift:].view(rows, columns + pad)[:, :columns]
    v.copy_(t)
    return v


def parameters(columns, which, dtype=F32):
    names = ("post_weight", "post_bias", "channel_scale", "pre_weight", "pre_bias")
    return {n: (values(50 + i, columns, scale=0.3) + (0 if "bias" in n else 1)).to(dtype) if n in which else None
            for i, n in enumerate(names)}


ALL = ("post_weight", "post_bias", "channel_scale", "pre_weight", "pre_bias")


def check(rows, columns, dtype=F32, residual=None, kind="rms", gate="element", activation="sigmoid", which=ALL,
          param_dtype=F32, post_norm=True, pre_norm=True, with_y=True, pad=0, shift=0, dh=True, dz=True, scale=0.7):
    residual = residual or dtype
    if not post_norm:
        which = [w for w in which if not w.startswith("post")]
    if not pre_norm:
        which = [w for w in which if not w.startswith("pre")]
    if not with_y:
        which = [w for w in which if w.startswith("pre")]
    p = parameters(columns, which, param_dtype)
    place = (lambda t: strided(t, pad, shift)) if pad or shift else (lambda t: t)
    x = place(values(1, rows, columns, scale=2.0, dtype=residual))
    y = place(values(2, rows, columns, dtype=dtype)) if with_y else None
    g = None
    if with_y and gate != "none":
        g = place(values(3, rows, columns, dtype=dtype)) if gate == "element" else values(3, rows, dtype=dtype)
    how = dict(scale=scale, kind=kind, activation=activation, epsilon=EPS, post_norm=post_norm, pre_norm=pre_norm)
    h, z = dense.block_norm(x, y, g, **p, **how)
    plain = (p, scale, kind, activation, EPS, post_norm, pre_norm)
    wh, wz, size = ref.block_norm(x, y, g, *plain)
    assert h.dtype == residual
    ref.close(h, wh, size)
    if pre_norm:
        assert z.dtype == dtype
        r = ref.norm(wh, kind, EPS)[1]
        row = (size * r).amax(-1, keepdim=True) if rows else 0
        w = 1 if p["pre_weight"] is None else p["pre_weight"].double().abs()
        b = 0 if p["pre_bias"] is None else p["pre_bias"].double().abs()
        ref.close(z, wz, row * w + b)
    else:
        assert z is None
    gh = place(values(4, rows, columns, scale=1e-2, dtype=residual)) if dh else None
    gz = place(values(5, rows, columns, scale=1e-2, dtype=dtype)) if dz and pre_norm else None
    got = dense.block_norm_backward(gh, gz, h, y, g, **p, **how)
    want = ref.block_norm_backward(gh, gz, h, y, g, *plain)
    for name in got._fields:
        t = getattr(got, name)
        given = {"x": True, "y": with_y, "gate": g is not None, **{n: n in which for n in ALL}}[name]
        assert (t is not None) == given, name
        if t is None:
            continue
        if name not in want:      # dz is None: nothing reaches the norm after
            assert not t.any()
            continue
        value, size = want[name]
        ref.close(t, value.reshape(t.shape), size)


@gpu
@pytest.mark.parametrize("columns", [1, 7, 8, 16, 33, 64, 100, 256, 264, 640, 1000, 2048, 4097, 4104, 8191, 8192])
@pytest.mark.parametrize("kind,dtype", [("rms", BF16), ("layer", F32)])
def test_widths(columns, kind, dtype):
    for rows in (1, 37):
        check(rows, columns, dtype, kind=kind)


@gpu
@pytest.mark.parametrize("gate,activation,kind", list(itertools.product(("none", "row", "element"), ("none", "sigmoid", "silu", "tanh"),
                                                                        ("rms", "layer"))))
def test_gates(gate, activation, kind):
    for columns in (24, 1032):
        check(19, columns, F32, gate=gate, activation=activation, kind=kind)


@gpu
@pytest.mark.parametrize("dtype,residual,param", [(BF16, BF16, BF16), (F16, F16, F32), (F16, F16, F16), (BF16, F32, F32),
                                                  (F16, F32, F16), (F32, F32, F32)])
def test_types(dtype, residual, param):
    for columns in (40, 777, 2048):
        check(33, columns, dtype, residual, kind="layer", param_dtype=param)


@gpu
@pytest.mark.parametrize("pad,shift", [(0, 1), (3, 0), (8, 0), (8, 8), (5, 3)])
def test_strides_and_alignment(pad, shift):
    for columns in (64, 512):
        check(21, columns, BF16, pad=pad, shift=shift)
        check(21, columns, F32, pad=pad, shift=shift, gate="row")


@gpu
def test_parts_left_out():
    check(11, 96, which=())
    check(11, 96, which=("pre_weight",), kind="layer")
    check(11, 96, post_norm=False)
    check(11, 96, pre_norm=False)
    check(11, 96, post_norm=False, pre_norm=False, gate="none")
    check(11, 96, with_y=False)
    check(11, 96, dh=False)
    check(11, 96, dz=False)
    check(0, 96)
    check(5000, 48, BF16, kind="layer")        # several rows for each block of the gradient


@gpu
def test_rows_without_variance():
    """Rows of zeros, of one value, and of a large value: epsilon alone holds the norm."""
    x = torch.zeros(3, 64, device="cuda")
    y = torch.zeros(3, 64, device="cuda")
    y[1] = 4.0
    y[2] = 3e18         # its square sum is still finite
    for kind in ("rms", "layer"):
        h, z = dense.block_norm(x, y, kind=kind, epsilon=EPS)
        wh, wz, _ = ref.block_norm(x, y, None, parameters(64, ()), 1.0, kind, "none", EPS, True, True)
        ref.close(h, wh, torch.ones(()).cuda())
        ref.close(z, wz, torch.full((), 1.0).cuda())


@gpu
def test_a_bad_row_stays_alone():
    x, y, g = values(1, 9, 128), values(2, 9, 128), values(3, 9, 128)
    clean = dense.block_norm(x, y, g)
    y2, g2 = y.clone(), g.clone()
    y2[4, 5], g2[6, 7] = float("nan"), float("inf")
    h, z = dense.block_norm(x, y2, g2, activation="sigmoid")
    assert h[4].isnan().all() and z[4].isnan().all()
    others = [0, 1, 2, 3, 5, 7, 8]
    assert torch.equal(h[others], clean[0][others]) and torch.equal(z[others], clean[1][others])
    n = ref.norm(y.double(), "rms", 1e-6)[0]
    ref.close(h[6, 7], (x.double() + n)[6, 7], torch.tensor(10.0, device="cuda"))     # an open gate


@gpu
@pytest.mark.parametrize("kind", ["rms", "layer"])
def test_gradients_against_differences(kind):
    """d loss along random directions, by central differences of the 64-bit forward."""
    rows, columns, step = 5, 40, 1e-6
    p = parameters(columns, ALL)
    t = {"x": values(1, rows, columns), "y": values(2, rows, columns), "gate": values(3, rows, columns), **p}
    gh, gz = values(4, rows, columns), values(5, rows, columns)
    how = dict(scale=0.7, kind=kind, activation="silu", epsilon=EPS)
    h, _ = dense.block_norm(t["x"], t["y"], t["gate"], **p, **how)
    got = dense.block_norm_backward(gh, gz, h, t["y"], t["gate"], **p, **how)

    def loss(t):
        q = {n: t[n] for n in ALL}
        h, z, _ = ref.block_norm(t["x"], t["y"], t["gate"], q, 0.7, kind, "silu", EPS, True, True)
        return ((h * gh).sum() + (z * gz).sum()).item()
    for i, name in enumerate(got._fields):
        d = values(70 + i, *t[name].shape).double()
        up = loss({**t, name: t[name].double() + step * d})
        down = loss({**t, name: t[name].double() - step * d})
        want, have = (up - down) / (2 * step), (getattr(got, name).double() * d).sum().item()
        # differences: step^2 of a third derivative and 1e-16 / step of the loss; the rest is float32
        assert abs(want - have) <= 1e-5 * (getattr(got, name).double() * d).abs().sum().item() + 1e-7


@gpu
def test_results_repeat_and_follow_the_stream():
    x, y, g = (values(i, 3001, 264, dtype=BF16) for i in (1, 2, 3))
    w = values(9, 264)
    torch.cuda.synchronize()
    first = dense.block_norm_backward(x, g, x, y, g, post_weight=w, pre_weight=w)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        late = torch.empty_like(y)
        torch.cuda._sleep(20_000_000)
        late.copy_(y)             # the call must run behind this copy
        second = dense.block_norm_backward(x, g, x, late, g, post_weight=w, pre_weight=w)
    torch.cuda.synchronize()
    for a, b in zip(first, second):
        assert (a is None) == (b is None) and (a is None or torch.equal(a, b))


@gpu
def test_graph_capture():
    x, y, g = (values(i, 50, 512, dtype=BF16) for i in (1, 2, 3))
    dense.block_norm(x, y, g)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        h, z = dense.block_norm(x, y, g)
    y.mul_(-0.5)
    graph.replay()
    wh, wz = dense.block_norm(x, y, g)
    assert torch.equal(h, wh) and torch.equal(z, wz)


@gpu
def test_refusals():
    x, y = values(1, 4, 32), values(2, 4, 32)
    bad = [lambda: dense.block_norm(x, values(2, 4, 31)), lambda: dense.block_norm(x, values(2, 5, 32)),
           lambda: dense.block_norm(x.to(BF16), y), lambda: dense.block_norm(x, y, values(3, 3)),
           lambda: dense.block_norm(x, None, values(3, 4)), lambda: dense.block_norm(x, y, kind="batch"),
           lambda: dense.block_norm(x, y, activation="relu"), lambda: dense.block_norm(x, y, epsilon=0.0),
           lambda: dense.block_norm(x, y, epsilon=float("nan")), lambda: dense.block_norm(x, y, scale=float("nan")),
           lambda: dense.block_norm(x, y, post_weight=values(3, 31)), lambda: dense.block_norm(x, y, pre_weight=values(3, 32, dtype=F16)),
           lambda: dense.block_norm(x.double(), y.double()), lambda: dense.block_norm(x.t(), None),
           lambda: dense.block_norm(values(1, 2, 8200)), lambda: dense.block_norm(x.cpu()),
           lambda: dense.block_norm_backward(x, x, x, y, pre_norm=False), lambda: dense.block_norm_backward(x, x.to(BF16), x, y),
           lambda: dense.block_norm_backward(x[:2], x, x, y)]
    for call in bad:
        with pytest.raises(EpsError) as e:
            call()
        assert e.value.code == INVALID_ARGUMENT
