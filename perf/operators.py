"""The dense operators' measured cases: one mixture-of-experts block beside the embedding store.

Four operators, each in a plain form of elementary torch operations and, where `own` is set, as
calls of the package's `dense` module:

  norm    the norms before and after a block, fused with its gate and residual scale (and backward)
  route   routing to experts: scores, balance bias, groups, top-k, weights, the sort by expert (and
          backward)
  int8    the experts' matrix products in 8-bit integers, a scale for each token and channel
  adamw   one AdamW step over many tensors, states in 32 or in 8 bits
"""
import importlib
import math
import random

import torch

PACKAGE = "distributed-recommendation-model-training-system_b200"
own = False

DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
SIZE = {"float32": 4, "bfloat16": 2, "float16": 2}
BLOCK = 256          # elements that share one scale of an 8-bit optimizer state
LOWEST = -3.4028234663852886e38


def dense():
    return importlib.import_module(PACKAGE + ".dense")


# ------------------------------------------------------------------ the cases
def listed():
    return [
        # a handful of requests being served: latency counts, the data is nothing
        {"name": "norm_single", "op": "norm", "way": "forward", "rows": 4, "columns": 1024, "dtype": "bfloat16",
         "kind": "rms", "gate": "element", "activation": "sigmoid", "channel_scale": False, "bias": False},
        # a training batch between two blocks (an odd number of tokens)
        {"name": "norm_forward", "op": "norm", "way": "forward", "rows": 16381, "columns": 2048, "dtype": "bfloat16",
         "kind": "rms", "gate": "element", "activation": "silu", "channel_scale": True, "bias": False},
        # the same place in the backward pass, with every gradient of weights, biases and scales
        {"name": "norm_backward", "op": "norm", "way": "backward", "rows": 16381, "columns": 2048, "dtype": "bfloat16",
         "kind": "layer", "gate": "element", "activation": "sigmoid", "channel_scale": True, "bias": True},
        # one request's tokens routed with a balance bias inside the best groups
        {"name": "route_single", "op": "route", "way": "forward", "rows": 3, "experts": 128, "top_k": 6, "dtype": "float32",
         "score": "sigmoid", "bias": True, "groups": 8, "top_groups": 4, "renormalise": True, "masked": 0},
        # a training batch over many experts, sorted by expert for their products
        {"name": "route_prompt", "op": "route", "way": "forward", "rows": 32771, "experts": 256, "top_k": 8,
         "dtype": "float32", "score": "sigmoid", "bias": True, "groups": 8, "top_groups": 4, "renormalise": True, "masked": 0},
        # the router's gradient for such a batch, some experts masked out
        {"name": "route_backward", "op": "route", "way": "backward", "rows": 32771, "experts": 96, "top_k": 4,
         "dtype": "bfloat16", "score": "softmax", "bias": False, "groups": 1, "top_groups": 1, "renormalise": True, "masked": 3},
        # one token through one layer: the weights' bytes are what counts
        {"name": "int8_single", "op": "int8", "rows": 1, "experts": 1, "channels": 4096, "inner": 4096, "dtype": "bfloat16",
         "bias": False, "gather": False},
        # a few hundred requests over many experts: ragged groups, some empty, rows gathered by the router's order
        {"name": "int8_experts", "op": "int8", "rows": 1531, "experts": 32, "channels": 1408, "inner": 2048,
         "dtype": "bfloat16", "bias": True, "gather": True},
        # a large scoring batch through one wide layer
        {"name": "int8_prompt", "op": "int8", "rows": 8189, "experts": 1, "channels": 8192, "inner": 4096,
         "dtype": "bfloat16", "bias": True, "gather": False},
        # the ranking tower beside the tables: many small tensors
        {"name": "adamw_towers", "op": "adamw", "tensors": 40, "elements": 1300001, "layout": 5, "dtype": "float32",
         "gradient": "float32", "bits": 32, "master": False},
        # a large dense part in bf16 with 32-bit copies of the weights
        {"name": "adamw_master", "op": "adamw", "tensors": 24, "elements": 150000007, "layout": 6, "dtype": "bfloat16",
         "gradient": "bfloat16", "bits": 32, "master": True},
        # the same with its moments in 8 bits
        {"name": "adamw_8bit", "op": "adamw", "tensors": 24, "elements": 200000003, "layout": 7, "dtype": "float32",
         "gradient": "float32", "bits": 8, "master": False},
    ]


def spread(rng, low, high):
    """A whole number between low and high, even over the logarithm."""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["norm", "route", "int8", "adamw"])
    if op == "norm":
        columns = spread(rng, 16, 8192)
        columns = columns if rng.random() < 0.3 else max(16, columns // 8 * 8)
        return {"op": op, "way": rng.choice(["forward", "backward"]), "rows": min(spread(rng, 1, 65536), 16000 * 2048 // columns),
                "columns": columns, "dtype": rng.choice(["bfloat16", "bfloat16", "float16", "float32"]), "kind": rng.choice(["rms", "layer"]),
                "gate": rng.choice(["none", "row", "element", "element"]), "activation": rng.choice(["none", "sigmoid", "silu", "tanh"]),
                "channel_scale": rng.random() < 0.5, "bias": rng.random() < 0.5}
    if op == "route":
        groups = rng.choice([1, 1, 2, 4, 8])
        experts = max(4, spread(rng, 8, 512) // groups) * groups
        top_groups = rng.randint(max(1, groups // 2), groups)
        top_k = rng.randint(1, min(16, experts // groups * top_groups))
        return {"op": op, "way": rng.choice(["forward", "backward"]), "rows": min(spread(rng, 1, 65536), 32000 * 256 // experts),
                "experts": experts, "top_k": top_k,
                "dtype": rng.choice(["float32", "float32", "bfloat16", "float16"]), "score": rng.choice(["softmax", "sigmoid"]),
                "bias": rng.random() < 0.5, "groups": groups, "top_groups": top_groups, "renormalise": top_k > 1 and rng.random() < 0.7,   # one weight alone would always be 1
                "masked": rng.choice([0, 0, experts // 8])}
    if op == "int8":
        experts = rng.choice([1, 1, 4, 16, 64])
        channels, inner = spread(rng, 33, 8192), spread(rng, 48, 8192)
        if rng.random() < 0.6:
            channels, inner = max(64, channels // 64 * 64), max(64, inner // 64 * 64)
        while experts * channels * inner > 1 << 28:
            experts //= 4
        rows = spread(rng, 1, 8192)
        while rows > 1 and rows * channels * inner > 8000 * 8192 * 4096:
            rows = rows // 2 + 1
        return {"op": op, "rows": rows, "experts": experts, "channels": channels, "inner": inner,
                "dtype": rng.choice(["bfloat16", "bfloat16", "float16", "float32"]), "bias": rng.random() < 0.5,
                "gather": rng.random() < 0.5}
    dtype = rng.choice(["float32", "bfloat16", "float16"])
    return {"op": op, "tensors": rng.randint(1, 40), "elements": spread(rng, 1000, 100000000), "layout": rng.randint(0, 1 << 30),
            "dtype": dtype, "gradient": rng.choice([dtype, "float32"]), "bits": rng.choice([32, 8]),
            "master": dtype != "float32" and rng.random() < 0.7}


# ------------------------------------------------------- what is in hand before
def generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def normal(g, *shape, scale=1.0, dtype=torch.float32):
    return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)


def norm_inputs(case, seed):
    g, dt = generator(seed), DTYPES[case["dtype"]]
    T, D = case["rows"], case["columns"]
    loud = 1 + 9 * (torch.rand(D, generator=g, device="cuda") < 0.01)     # a few channels are loud, as in trained models
    s = {"y": (normal(g, T, D) * loud).to(dt), "gate": None, "channel_scale": None, "post_bias": None, "pre_bias": None,
         "post_weight": normal(g, D, scale=0.2) + 1, "pre_weight": normal(g, D, scale=0.2) + 1}
    if case["gate"] != "none":
        s["gate"] = normal(g, T, D, dtype=dt) if case["gate"] == "element" else normal(g, T, dtype=dt)
    if case["channel_scale"]:
        s["channel_scale"] = normal(g, D, scale=0.1) + 0.3
    if case["bias"]:
        s["post_bias"], s["pre_bias"] = normal(g, D, scale=0.1), normal(g, D, scale=0.1)
    if case["way"] == "forward":
        s["x"] = normal(g, T, D, scale=2.0, dtype=dt)
    else:
        s["h"] = normal(g, T, D, scale=2.0, dtype=dt)
        s["dh"], s["dz"] = normal(g, T, D, scale=1e-2, dtype=dt), normal(g, T, D, scale=1e-2, dtype=dt)
    return s


def route_inputs(case, seed):
    g, dt = generator(seed), DTYPES[case["dtype"]]
    T, E = case["rows"], case["experts"]
    logits = normal(g, T, E, scale=1.5)
    if case["masked"]:
        out = torch.rand(T, E, generator=g, device="cuda") < case["masked"] / E
        out[:, : case["top_k"]] &= T % 2 == 0    # with an odd number of tokens the first experts are never masked
        logits = logits.masked_fill(out, -math.inf)
    s = {"logits": logits.to(dt), "bias": normal(g, E, scale=0.05) if case["bias"] else None}
    if case["way"] == "backward":
        s["experts"] = route_plain(s["logits"], s["bias"], case)[0]
        s["dweights"] = normal(g, T, case["top_k"], scale=1e-2)
    return s


def group_sizes(case, seed):
    """Rows of each expert: uneven, some without any, as a router leaves them."""
    r = random.Random(seed)
    E, R = case["experts"], case["rows"]
    share = [0.0 if E > 1 and r.random() < 0.1 else r.gammavariate(2.0, 1.0) for _ in range(E)]
    share[r.randrange(E)] += 0.5
    cut, total, sizes = 0.0, sum(share), []
    for e in range(E):
        before, cut = round(R * cut / total), cut + share[e]
        sizes.append((R if e == E - 1 else round(R * cut / total)) - before)
    return sizes


def int8_inputs(case, seed):
    g, dt = generator(seed), DTYPES[case["dtype"]]
    R, E, N, K = case["rows"], case["experts"], case["channels"], case["inner"]
    tokens = -(-R // 2) if case["gather"] else R
    s = {"x": normal(g, tokens, K, dtype=dt), "rows": None, "sizes": group_sizes(case, seed),
         "weight": torch.randint(-127, 128, (E, N, K), generator=g, device="cuda", dtype=torch.int8),
         "weight_scale": (torch.rand(E, N, generator=g, device="cuda") + 0.5) / (127 * math.sqrt(K)),
         "bias": normal(g, E, N, scale=0.1) if case["bias"] else None}
    if case["gather"]:
        s["rows"] = torch.randint(0, tokens, (R,), generator=g, device="cuda", dtype=torch.int32)
    ends = [0]
    for n in s["sizes"]:
        ends.append(ends[-1] + n)
    s["offsets"] = torch.tensor(ends, device="cuda", dtype=torch.int32)
    return s


def tensor_sizes(case):
    """Uneven tensor sizes that add up to the case's elements: vectors beside matrices."""
    r = random.Random(case["layout"])
    n, total = case["tensors"], case["elements"]
    share = [math.exp(r.uniform(0, 6)) for _ in range(n)]
    sizes = [max(1, int(total * v / sum(share))) for v in share]
    sizes[0] += max(0, total - sum(sizes))
    return sizes


HYPER = {"learning_rate": 1e-3, "beta1": 0.9, "beta2": 0.999, "epsilon": 1e-8, "weight_decay": 0.01}
STEPS, SEED = 99, 2024     # steps already taken; seed of the rounding of 8-bit states


def adamw_inputs(case, seed):
    """Parameters, gradients and moments in the middle of a training run; the moments lie one tensor
    after the other, each from a multiple of BLOCK elements on."""
    g, dt = generator(seed), DTYPES[case["dtype"]]
    sizes = tensor_sizes(case)
    starts, at = [], 0
    for n in sizes:
        starts.append(at)
        at += -(-n // BLOCK) * BLOCK
    real = torch.zeros(at, dtype=torch.bool, device="cuda")
    for n, a in zip(sizes, starts):
        real[a:a + n] = True
    size = torch.exp(normal(g, at, scale=1.0)) * 1e-3      # each weight's own gradient size
    second = torch.where(real, size * size * (0.5 + torch.rand(at, generator=g, device="cuda")), 0.0)
    first = torch.where(real, size * normal(g, at, scale=0.3), 0.0)
    grads = [(size[a:a + n] * normal(g, n)).to(DTYPES[case["gradient"]]) for n, a in zip(sizes, starts)]
    masters = [normal(g, n, scale=0.05) for n in sizes]
    s = {"sizes": sizes, "starts": starts, "total": at, "steps": STEPS, "gradients": grads,
         "parameters": [p.to(dt) for p in masters], "master": None, "first": first, "second": second}
    if case["master"]:
        s["master"] = flat(masters, starts, at)
    if case["bits"] == 8:
        s["first"], s["first_scale"] = encode(first)
        s["second"], s["second_scale"] = encode(second.sqrt())
    return s


def prepare(case, seed):
    s = {"norm": norm_inputs, "route": route_inputs, "int8": int8_inputs, "adamw": adamw_inputs}[case["op"]](case, seed)
    s["case"] = case
    if own and case["op"] == "int8":
        s["handle"] = dense().QuantizedExperts(s.pop("weight"), s.pop("weight_scale"), bias=s["bias"])
    if own and case["op"] == "adamw":
        s["handle"] = dense().AdamW(s["parameters"], s["gradients"], state_bits=case["bits"], master=case["master"], seed=SEED, **HYPER)
        s["handle"].load_state(STEPS, **{k: s.pop(k) for k in ("first", "second", "first_scale", "second_scale", "master") if s.get(k) is not None})
    return s


# ------------------------------------------------------------------- one pass
def run(s):
    return {"norm": run_norm, "route": run_route, "int8": run_int8, "adamw": run_adamw}[s["case"]["op"]](s, s["case"])


EPS, SCALE = 1e-6, 0.7       # the norms' epsilon and the residual scale
ROUTE_SCALE = 2.5


def normed(v, kind):
    """v less its mean ("layer"), the reciprocal of its root mean square, and their product."""
    v = v - v.mean(-1, keepdim=True) if kind == "layer" else v
    r = 1 / torch.sqrt((v * v).mean(-1, keepdim=True) + EPS)
    return r, v * r


def activated(gate, name):
    """act(gate) and its derivative."""
    if name == "none":
        return gate, torch.ones_like(gate)
    if name == "tanh":
        t = torch.tanh(gate)
        return t, 1 - t * t
    s = 1 / (1 + torch.exp(-gate))
    return (s, s * (1 - s)) if name == "sigmoid" else (gate * s, s * (1 + gate * (1 - s)))


def norm_gradient(dn, r, vhat, kind):
    """The gradient of v where that of its norm, without weight and bias, is dn."""
    d = dn - vhat * (dn * vhat).mean(-1, keepdim=True)
    return r * (d - dn.mean(-1, keepdim=True) if kind == "layer" else d)


def run_norm(s, case):
    if own:
        more = {k: s[k] for k in ("channel_scale", "post_weight", "post_bias", "pre_weight", "pre_bias")}
        more |= {"kind": case["kind"], "activation": case["activation"], "scale": SCALE, "epsilon": EPS}
        if case["way"] == "forward":
            return list(dense().block_norm(s["x"], s["y"], s["gate"], **more))
        return list(dense().block_norm_backward(s["dh"], s["dz"], s["h"], s["y"], s["gate"], **more))
    dt, kind = DTYPES[case["dtype"]], case["kind"]
    y = s["y"].float()
    gate = None if s["gate"] is None else s["gate"].float().reshape(len(y), -1)
    a, da = (1.0, None) if gate is None else activated(gate, case["activation"])
    r1, yhat = normed(y, kind)
    n = yhat * s["post_weight"] + (0.0 if s["post_bias"] is None else s["post_bias"])
    c = SCALE if s["channel_scale"] is None else SCALE * s["channel_scale"]
    if case["way"] == "forward":
        h = s["x"].float() + c * (a * n)
        z = normed(h, kind)[1] * s["pre_weight"] + (0.0 if s["pre_bias"] is None else s["pre_bias"])
        return [h.to(dt), z.to(dt)]
    dz = s["dz"].float()
    r2, hhat = normed(s["h"].float(), kind)
    dh = s["dh"].float() + norm_gradient(dz * s["pre_weight"], r2, hhat, kind)
    e = c * dh
    dgate = None
    if gate is not None:
        dgate = (e * n * da) if case["gate"] == "element" else (e * n * da).sum(-1)
    dn = e * a
    dy = norm_gradient(dn * s["post_weight"], r1, yhat, kind)
    bias = case["bias"]
    return [dh.to(dt), dy.to(dt), None if dgate is None else dgate.to(dt), (dn * yhat).sum(0), dn.sum(0) if bias else None,
            (SCALE * dh * a * n).sum(0) if case["channel_scale"] else None, (dz * hhat).sum(0), dz.sum(0) if bias else None]


def scores(logits, name):
    x = logits.float()
    if name == "sigmoid":
        return 1 / (1 + torch.exp(-x))
    top = x.max(-1, keepdim=True).values
    e = torch.where(top == -math.inf, 0.0, torch.exp(x - top))
    # the sum in 64 bits, so that the ranking below does not hang on the order of its terms
    total = e.double().sum(-1, keepdim=True).float()
    return torch.where(total == 0, 0.0, e / total)


def route_plain(logits, bias, case):
    p = scores(logits, case["score"])
    key = p if bias is None else p + bias
    key = torch.where(torch.isnan(key), LOWEST, key).clamp(min=LOWEST)
    T, E = key.shape
    G = case["groups"]
    if G > 1:
        best = torch.sort(key.view(T, G, E // G), dim=-1, descending=True).values
        group = best[..., 0] + best[..., 1] if E // G > 1 else best[..., 0]
        chosen = torch.sort(group, dim=-1, descending=True, stable=True).indices[:, : case["top_groups"]]
        inside = torch.zeros(T, G, dtype=torch.bool, device=key.device).scatter_(1, chosen, True)
        key = torch.where(inside.repeat_interleave(E // G, dim=1), key, -math.inf)
    experts = torch.sort(key, dim=-1, descending=True, stable=True).indices[:, : case["top_k"]]
    w = p.gather(1, experts)
    if case["renormalise"]:
        total = w.sum(-1, keepdim=True)
        w = torch.where(total == 0, 0.0, w / total)
    return experts.to(torch.int32), w * ROUTE_SCALE


def run_route(s, case):
    how = {"score": case["score"], "renormalise": case["renormalise"], "scale": ROUTE_SCALE}
    if own:
        if case["way"] == "backward":
            return dense().route_backward(s["logits"], s["experts"], s["dweights"], **how)
        r = dense().route(s["logits"], case["top_k"], bias=s["bias"], groups=case["groups"], top_groups=case["top_groups"], **how)
        return [r.experts, r.weights, r.order, r.position, r.offsets]
    if case["way"] == "forward":
        experts, w = route_plain(s["logits"], s["bias"], case)
        found = experts.reshape(-1)
        order = torch.sort(found, stable=True).indices
        position = torch.empty_like(order)
        position[order] = torch.arange(len(order), device=order.device)
        offsets = torch.cat([torch.zeros(1, dtype=torch.int64, device=order.device), torch.bincount(found, minlength=case["experts"]).cumsum(0)])
        return [experts, w, order.to(torch.int32), position.view_as(experts).to(torch.int32), offsets.to(torch.int32)]
    p = scores(s["logits"], case["score"])
    experts = s["experts"].long()
    chosen, d = p.gather(1, experts), s["dweights"] * ROUTE_SCALE
    if case["renormalise"]:
        total = chosen.sum(-1, keepdim=True)
        d = torch.where(total == 0, 0.0, (d - (d * chosen).sum(-1, keepdim=True) / total) / total)
    ds = torch.zeros_like(p).scatter_(1, experts, d)
    if case["score"] == "sigmoid":
        return (ds * p * (1 - p)).to(s["logits"].dtype)
    return (p * (ds - (ds * p).sum(-1, keepdim=True))).to(s["logits"].dtype)


def run_int8(s, case):
    if own:
        return s["handle"].product(s["x"], offsets=s["offsets"], rows=s["rows"])
    x = s["x"].float()
    top = x.abs().amax(-1, keepdim=True)
    q = torch.round(x * (127 / top)) if s["rows"] is None else torch.round(x * (127 / top))[s["rows"]]
    scale = top / 127 if s["rows"] is None else (top / 127)[s["rows"]]
    parts = [(a @ w.float().T) * c for a, w, c in zip(q.split(s["sizes"]), s["weight"], s["weight_scale"])]
    out = torch.cat(parts) * scale
    if s["bias"] is not None:
        out = out + s["bias"].repeat_interleave(torch.diff(s["offsets"]), dim=0, output_size=case["rows"])
    return out.to(DTYPES[case["dtype"]])


def flat(tensors, starts, total):
    """One tensor after the other, each from its start on, zeros between them."""
    ends = [*starts[1:], total]
    return torch.cat([torch.nn.functional.pad(t.reshape(-1).float(), (0, e - a - t.numel())) for t, a, e in zip(tensors, starts, ends)])


def scales(v):
    """The scale of each block: its largest magnitude over e4m3's, 448."""
    return v.view(-1, BLOCK).abs().amax(-1) / 448


def scaled(v, scale):
    inverse = torch.where(scale == 0, 0.0, 1 / scale)
    return (v.view(-1, BLOCK) * inverse[:, None]).clamp(-448, 448)


def encode(v):
    """v in 8 bits: e4m3 values, rounded to the nearest, and a scale for each block."""
    scale = scales(v)
    return scaled(v, scale).to(torch.float8_e4m3fn).view(-1), scale


def hashed(pairs, steps):
    """32 bits for each pair of elements, from their index, the step and SEED (in 64-bit integers)."""
    def mix(h):
        h = ((h ^ (h >> 16)) * 0x85EBCA6B) & 0xFFFFFFFF
        h = ((h ^ (h >> 13)) * 0xC2B2AE35) & 0xFFFFFFFF
        return h ^ (h >> 16)
    key = mix(torch.tensor(SEED, device="cuda") ^ mix(torch.tensor(steps, device="cuda")))
    return mix((torch.arange(pairs, device="cuda") * 0x9E3779B1 + key) & 0xFFFFFFFF)


def encode_random(v, steps):
    """v >= 0 in 8 bits, rounded up or down by the hash so that it is right on average; above zero
    it stays above zero."""
    scale = scales(v)
    x = scaled(v, scale).view(-1)
    h = hashed(len(x) // 2, steps)
    u = torch.stack([h & 0xFFFF, h >> 16], -1).view(-1)           # 16 bits for each element
    coarse = ((x.view(torch.int32) + (u.to(torch.int32) << 4)) & -0x100000).view(torch.float32)
    fine = torch.floor(x * 512 + u.float() / 65536) / 512           # below 2^-6 the values lie 2^-9 apart
    code = torch.where(x < 2.0 ** -6, fine, coarse).clamp(max=448)
    code = torch.where(x > 0, code.clamp(min=2.0 ** -9), code)
    return code.to(torch.float8_e4m3fn), scale


def run_adamw(s, case):
    if own:
        o = s["handle"]
        o.step()
        return [o.parameters, o.master, o.first, o.first_scale, o.second, o.second_scale]
    s["steps"] += 1
    t, c = s["steps"], HYPER
    p = s["master"] if case["master"] else flat(s["parameters"], s["starts"], s["total"])
    g = flat(s["gradients"], s["starts"], s["total"])
    m, root = s["first"].float(), s["second"].float()
    if case["bits"] == 8:
        m = (m.view(-1, BLOCK) * s["first_scale"][:, None]).view(-1)
        root = (root.view(-1, BLOCK) * s["second_scale"][:, None]).view(-1)
    m = c["beta1"] * m + (1 - c["beta1"]) * g
    v = c["beta2"] * (root * root if case["bits"] == 8 else root) + (1 - c["beta2"]) * g * g
    down = torch.sqrt(v) / math.sqrt(1 - c["beta2"] ** t) + c["epsilon"]
    p = p * (1 - c["learning_rate"] * c["weight_decay"]) - c["learning_rate"] / (1 - c["beta1"] ** t) * (m / down)
    torch._foreach_copy_(s["parameters"], [p[a:a + n] for a, n in zip(s["starts"], s["sizes"])])
    if case["master"]:
        s["master"] = p
    if case["bits"] == 8:
        s["first"], s["first_scale"] = encode(m)
        s["second"], s["second_scale"] = encode_random(torch.sqrt(v), t)
    else:
        s["first"], s["second"] = m, v
    return [s["parameters"], s["master"], s["first"], s.get("first_scale"), s["second"], s.get("second_scale")]


# ------------------------------------------------- what a pass cannot do without
def work(case):
    if case["op"] == "norm":
        n = case["rows"] * case["columns"]
        gate = {"none": 0, "row": case["rows"], "element": n}[case["gate"]]
        values = 4 * n + gate if case["way"] == "forward" else 6 * n + 2 * gate
        return {"bytes": values * SIZE[case["dtype"]], "flops": (20 if case["way"] == "forward" else 45) * n}
    if case["op"] == "route":
        n, k = case["rows"] * case["experts"] * SIZE[case["dtype"]], case["rows"] * case["top_k"]
        return {"bytes": n + 16 * k + 4 * case["experts"] if case["way"] == "forward" else 2 * n + 8 * k,
                "flops": 10 * case["rows"] * case["experts"]}
    if case["op"] == "int8":
        R, N, K = case["rows"], case["channels"], case["inner"]
        used = sum(n > 0 for n in group_sizes(case, 1))
        tokens = -(-R // 2) if case["gather"] else R
        return {"bytes": (tokens * K + R * N) * SIZE[case["dtype"]] + used * N * (K + 4 + 4 * case["bias"]), "flops": 2 * R * N * K}
    p, g = SIZE[case["dtype"]], SIZE[case["gradient"]]
    state = 16 if case["bits"] == 32 else 4 + 16 / BLOCK
    return {"bytes": case["elements"] * ((p + 8 if case["master"] else 2 * p) + g + state), "flops": 16 * case["elements"]}


# ------------------------------------------------ the definition, in 64 bits
def exact(case, seed):
    return {"norm": exact_norm, "route": exact_route, "int8": exact_int8, "adamw": exact_adamw}[case["op"]](case, seed)


def exact_norm(case, seed):
    """The outputs from the definition, and the gradients by differentiating it."""
    s = {k: (v.double() if torch.is_tensor(v) else v) for k, v in norm_inputs(case, seed).items()}

    def norm(v, weight, bias):
        if case["kind"] == "layer":
            v = v - v.sum(-1, keepdim=True) / v.shape[-1]
        v = v / ((v ** 2).sum(-1, keepdim=True) / v.shape[-1] + EPS) ** 0.5 * weight
        return v if bias is None else v + bias

    def update():
        u = norm(s["y"], s["post_weight"], s["post_bias"]) * SCALE
        if s["channel_scale"] is not None:
            u = u * s["channel_scale"]
        if s["gate"] is not None:
            gate = s["gate"] if case["gate"] == "element" else s["gate"][:, None]
            u = u * {"none": lambda v: v, "sigmoid": torch.sigmoid, "tanh": torch.tanh, "silu": lambda v: v * torch.sigmoid(v)}[case["activation"]](gate)
        return u

    if case["way"] == "forward":
        h = s["x"] + update()
        return [h, norm(h, s["pre_weight"], s["pre_bias"])]
    names = ["h", "pre_weight", "pre_bias", "y", "gate", "post_weight", "post_bias", "channel_scale"]
    have = [n for n in names if s[n] is not None]
    for n in have:
        s[n].requires_grad_(True)
    early = [n for n in have if n in names[:3]]
    late = [n for n in have if n in names[3:]]
    got = dict(zip(early, torch.autograd.grad(norm(s["h"], s["pre_weight"], s["pre_bias"]), [s[n] for n in early], s["dz"])))
    dh = s["dh"] + got["h"]
    got |= dict(zip(late, torch.autograd.grad(update(), [s[n] for n in late], dh)))
    return [dh, got["y"], got.get("gate"), got["post_weight"], got.get("post_bias"), got.get("channel_scale"), got["pre_weight"], got.get("pre_bias")]


def exact_route(case, seed):
    s = route_inputs(case, seed)
    x = s["logits"].double()

    def score(x):
        p = torch.softmax(x, -1) if case["score"] == "softmax" else torch.sigmoid(x)
        return torch.nan_to_num(p) if case["masked"] else p

    def weights(p, experts):
        w = p.gather(1, experts)
        if case["renormalise"]:
            total = w.sum(-1, keepdim=True)
            w = w / torch.where(total == 0, 1.0, total)
        return w * ROUTE_SCALE

    if case["way"] == "backward":
        dead = torch.isinf(x).all(-1, keepdim=True)
        x = torch.where(dead, 0.0, x).requires_grad_(True)
        w = weights(score(x), s["experts"].long())
        d = torch.autograd.grad(w, x, s["dweights"].double())[0]
        return torch.where(dead, 0.0, d)
    p = score(x)
    key = p if s["bias"] is None else p + s["bias"].double()
    T, E = key.shape
    G = case["groups"]
    if G > 1:
        group = key.view(T, G, E // G).topk(min(2, E // G), -1).values.sum(-1)
        keep = torch.zeros_like(group, dtype=torch.bool).scatter_(1, group.topk(case["top_groups"], -1).indices, True)
        key = key.masked_fill(~keep.repeat_interleave(E // G, dim=1), -math.inf)
    # equal keys go to the lowest index
    experts = torch.argsort(-key, dim=-1, stable=True)[:, : case["top_k"]]
    return [None, weights(p, experts), None, None, None]


def exact_int8(case, seed):
    s = int8_inputs(case, seed)
    x = s["x"].double()
    if s["rows"] is not None:
        x = x[s["rows"].long()]
    step = x.abs().max(-1, keepdim=True).values / 127
    q, out, at = (x / step).round(), [], 0
    for e, n in enumerate(s["sizes"]):
        y = q[at:at + n] @ s["weight"][e].double().T * s["weight_scale"][e].double() * step[at:at + n]
        out.append(y if s["bias"] is None else y + s["bias"][e].double())
        at += n
    return torch.cat(out)


def exact_adamw(case, seed):
    s, h, t = adamw_inputs(case, seed), HYPER, STEPS + 1
    new, firsts, seconds, masters = [], [], [], []
    for i, (n, a) in enumerate(zip(s["sizes"], s["starts"])):
        end = a + -(-n // BLOCK) * BLOCK
        g = torch.zeros(end - a, dtype=torch.float64, device="cuda")
        p = torch.zeros_like(g)
        g[:n] = s["gradients"][i].double()
        p[:n] = s["master"][a:a + n].double() if case["master"] else s["parameters"][i].double()
        m, v = s["first"][a:end].double(), s["second"][a:end].double()
        if case["bits"] == 8:
            m = m * s["first_scale"][a // BLOCK:end // BLOCK].double().repeat_interleave(BLOCK)
            v = (v * s["second_scale"][a // BLOCK:end // BLOCK].double().repeat_interleave(BLOCK)) ** 2
        m = m + (1 - h["beta1"]) * (g - m)
        v = v + (1 - h["beta2"]) * (g * g - v)
        step = (m / (1 - h["beta1"] ** t)) / ((v / (1 - h["beta2"] ** t)).sqrt() + h["epsilon"])
        p = p - h["learning_rate"] * (step + h["weight_decay"] * p)
        new.append(p[:n])
        masters.append(p)
        firsts.append(m)
        seconds.append(v)
    first, second = torch.cat(firsts), torch.cat(seconds)
    master = torch.cat(masters) if case["master"] else None
    if case["bits"] == 32:
        return [new, master, first, None, second, None]
    # the codes' own values are a rounding, and not computed here; their scales are
    top = [v.view(-1, BLOCK).abs().max(-1).values / 448 for v in (first, second.sqrt())]
    return [new, master, None, top[0], None, top[1]]
