"""Plain 64-bit restatements of the dense operators, for the tests of the kernels."""
import math

import torch

# half a unit in the last place of each type, relative
UNIT = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
# what one value may gather on its way: some 64 roundings of float32 (a chain of about
# twenty operations, exp's and division's few units, and a sum over lanes)
CHAIN = 64 * 2.0 ** -24


def close(got, want, size=None, dtype=None, rel=0.0):
    """|got - want| within the rounding to got's type plus CHAIN of `size`, the
    magnitude of the terms that make up the value (default: the largest result)."""
    want = want.double()
    assert got.shape == want.shape, (got.shape, want.shape)
    if not want.numel():
        return
    size = want.abs().max() if size is None else size
    limit = UNIT[dtype or got.dtype] * want.abs() + CHAIN * size + rel * want.abs()
    if got.dtype == torch.float16:
        limit = limit + 2.0 ** -25          # half the spacing of its subnormal values
    off = (got.double() - want).abs()
    assert bool((off <= limit).all()), f"off by {off.max().item():.3g}, {(off / limit).max().item():.3g} of the limit"


def act(g, name):
    """activation and slope"""
    if name == "none":
        return g, torch.ones_like(g)
    if name == "tanh":
        return torch.tanh(g), 1 - torch.tanh(g) ** 2
    s = torch.sigmoid(g)
    return (s, s * (1 - s)) if name == "sigmoid" else (g * s, s * (1 + g * (1 - s)))


def hat_size(v, r, kind):
    """The terms of a normed value: the value, and the mean that a layer norm takes from it."""
    return r * (v.abs() + (v.abs().mean(-1, keepdim=True) if kind == "layer" else 0))


def norm(v, kind, eps):
    mean = v.mean(-1, keepdim=True) if kind == "layer" else torch.zeros_like(v[..., :1])
    r = 1 / torch.sqrt(((v - mean) ** 2).mean(-1, keepdim=True) + eps)
    return (v - mean) * r, r


def per_row(gate, y):
    """The gate as a matrix: of y's shape, or of one column."""
    return gate if gate.dim() == y.dim() else gate[..., None]


def _d(t):
    return None if t is None else t.double()


def _param(t, like, missing):
    return torch.full((like.shape[-1],), missing, dtype=torch.float64, device=like.device) if t is None else t.double()


def block_norm(x, y, gate, p, scale, kind, activation, eps, post_norm, pre_norm):
    """(h, z, size of h's terms)"""
    x, y, gate = _d(x), _d(y), _d(gate)
    h, size = x, x.abs()
    if y is not None:
        n, ns = y, y.abs()
        if post_norm:
            w, b = _param(p["post_weight"], x, 1.0), _param(p["post_bias"], x, 0.0)
            hat, r = norm(y, kind, eps)
            n, ns = hat * w + b, hat_size(y, r, kind) * w.abs() + b.abs()
        a = 1.0 if gate is None else act(per_row(gate, y), activation)[0]
        c = scale * _param(p["channel_scale"], x, 1.0) * a
        h, size = x + c * n, x.abs() + c.abs() * ns
    z = None
    if pre_norm:
        z = norm(h, kind, eps)[0] * _param(p["pre_weight"], x, 1.0) + _param(p["pre_bias"], x, 0.0)
    return h, z, size


def block_norm_backward(dh, dz, h, y, gate, p, scale, kind, activation, eps, post_norm, pre_norm):
    """{name: (gradient, size of its terms)}"""
    h, y, gate, dz = _d(h), _d(y), _d(gate), _d(dz)
    mean = (lambda v: v.mean(-1, keepdim=True)) if kind == "layer" else (lambda v: torch.zeros_like(v[..., :1]))
    dot = lambda a, b: (a * b).mean(-1, keepdim=True)  # noqa: E731
    d = torch.zeros_like(h) if dh is None else dh.double()
    got = {}
    if dz is not None:
        hat, r = norm(h, kind, eps)
        q = dz * _param(p["pre_weight"], h, 1.0)
        d = d + r * (q - mean(q) - hat * dot(q, hat))
        got["pre_weight"] = ((dz * hat).sum(0), (dz.abs() * hat_size(h, r, kind)).sum(0))
        got["pre_bias"] = (dz.sum(0), dz.abs().sum(0))
        got["x"] = (d, (d.abs() + r * (q.abs() + hat.abs() * (q * hat).abs().mean(-1, keepdim=True))).amax(-1, keepdim=True))
    else:
        got["x"] = (d, d.abs().max() if d.numel() else 0)
    if y is None:
        return got
    size = got["x"][1]
    if post_norm:
        hat, r = norm(y, kind, eps)
        w = _param(p["post_weight"], h, 1.0)
        n = hat * w + _param(p["post_bias"], h, 0.0)
        ns = hat_size(y, r, kind) * w.abs() + _param(p["post_bias"], h, 0.0).abs()
    else:
        n, ns = y, y.abs()
    a, slope = (torch.ones_like(h[..., :1]), None) if gate is None else act(per_row(gate, y), activation)
    c = scale * _param(p["channel_scale"], h, 1.0)
    t = scale * d * a * n
    got["channel_scale"] = (t.sum(0), (scale * size * a * ns).abs().sum(0))
    if gate is not None:
        g = c * d * n * slope
        s = (c * size * ns).abs()
        got["gate"] = (g.sum(-1), s.sum(-1)) if gate.dim() < y.dim() else (g, s.amax(-1, keepdim=True) if s.numel() else s)
    dn = c * d * a
    sdn = (c * size * a).abs()
    if post_norm:
        got["post_weight"] = ((dn * hat).sum(0), (sdn * hat_size(y, r, kind)).sum(0))
        got["post_bias"] = (dn.sum(0), sdn.sum(0) + 0 * dn.sum(0))
        q = dn * w
        sq = sdn * w.abs()
        dy = r * (q - mean(q) - hat * dot(q, hat))
        got["y"] = (dy, (r * (sq + hat.abs() * (sq * hat.abs()).mean(-1, keepdim=True) + sq.mean(-1, keepdim=True))).amax(-1, keepdim=True))
    else:
        got["y"] = (dn, sdn.amax(-1, keepdim=True))
    return got


def scores(logits, score):
    x = logits.double()
    if score == "sigmoid":
        return torch.sigmoid(x)
    dead = (x == -math.inf).all(-1, keepdim=True)
    return torch.where(dead, 0.0, torch.softmax(torch.where(dead, 0.0, x), -1))


def ranked(key, groups, top_groups, top_k):
    """The chosen experts of each token by plain loops: groups, then experts, by (key, lower index)."""
    low = -3.4028234663852886e38
    out = []
    for row in key.tolist():
        row = [low if v != v or v < low else v for v in row]
        n = len(row) // groups
        tops = []
        for g in range(groups):
            best = sorted(row[g * n:(g + 1) * n], reverse=True)[:2]
            tops.append(sum(best))
        keep = sorted(range(groups), key=lambda g: (-tops[g], g))[:top_groups]
        inside = [e for e in range(len(row)) if e // n in keep]
        out.append(sorted(inside, key=lambda e: (-row[e], e))[:top_k])
    return out
