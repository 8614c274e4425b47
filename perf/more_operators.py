"""More measured cases of the dense block: what stands beside the optimizer, the router and the
served layers.

Three operators, each in a plain form of elementary torch operations and, where `own` is set, as
calls of the package's `dense` module:

  clip      the global norm over many gradients, the clip factor for AdamW, clipping in place
  balance   the router's balance loss and each expert's count (and backward)
  adapters  low-rank adapters of many requests at once, added to a shared layer's output
"""
import importlib
import math
import random

import torch

PACKAGE = "distributed-recommendation-model-training-system_b200"
own = False

DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
SIZE = {"float32": 4, "bfloat16": 2, "float16": 2}


def dense():
    return importlib.import_module(PACKAGE + ".dense")


# ------------------------------------------------------------------ the cases
def listed():
    return [
        # fp16 gradients of a small tower under a loss scale: the factor for its optimizer
        {"name": "clip_small", "op": "clip", "way": "measure", "kind": "l2", "tensors": 12, "elements": 37001, "layout": 3,
         "dtype": "float16", "scaled": True},
        # the ranking tower beside the tables, clipped where its gradients lie
        {"name": "clip_towers", "op": "clip", "way": "clip", "kind": "l2", "tensors": 40, "elements": 1300001, "layout": 5,
         "dtype": "float32", "scaled": False},
        # a large dense part in bf16: the factor for its optimizer
        {"name": "clip_dense", "op": "clip", "way": "measure", "kind": "l2", "tensors": 24, "elements": 150000007, "layout": 6,
         "dtype": "bfloat16", "scaled": False},
        # a large dense part in float32, clipped in place for an optimizer of the user's own
        {"name": "clip_in_place", "op": "clip", "way": "clip", "kind": "l2", "tensors": 24, "elements": 200000003, "layout": 7,
         "dtype": "float32", "scaled": False},
        # a handful of tokens: latency counts
        {"name": "balance_single", "op": "balance", "way": "forward", "rows": 3, "experts": 128, "top_k": 6, "dtype": "float32",
         "score": "sigmoid", "normalise": True, "padded": False, "masked": 0},
        # a training batch over many experts
        {"name": "balance_prompt", "op": "balance", "way": "forward", "rows": 32771, "experts": 256, "top_k": 8, "dtype": "float32",
         "score": "sigmoid", "normalise": True, "padded": False, "masked": 0},
        # a padded batch of 16-bit logits
        {"name": "balance_padded", "op": "balance", "way": "forward", "rows": 131071, "experts": 96, "top_k": 4, "dtype": "bfloat16",
         "score": "softmax", "normalise": True, "padded": True, "masked": 3},
        # the loss's gradient, added to that of the router's weights
        {"name": "balance_backward", "op": "balance", "way": "backward", "rows": 65521, "experts": 256, "top_k": 8, "dtype": "bfloat16",
         "score": "softmax", "normalise": True, "padded": True, "masked": 0},
        # one request's single row through one layer
        {"name": "adapters_single", "op": "adapters", "rows": 1, "requests": 1, "adapters": 16, "rank": 16, "inner": 4096,
         "channels": 4096, "dtype": "bfloat16"},
        # a batch of requests with one row each, every one with its adapter
        {"name": "adapters_requests", "op": "adapters", "rows": 61, "requests": 61, "adapters": 100, "rank": 16, "inner": 4096,
         "channels": 4096, "dtype": "bfloat16"},
        # a scoring batch of uneven requests
        {"name": "adapters_prompt", "op": "adapters", "rows": 8189, "requests": 40, "adapters": 32, "rank": 16, "inner": 4096,
         "channels": 4096, "dtype": "bfloat16"},
        # many requests over odd widths in float32
        {"name": "adapters_ragged", "op": "adapters", "rows": 1531, "requests": 200, "adapters": 64, "rank": 12, "inner": 2048,
         "channels": 1407, "dtype": "float32"},
    ]


def spread(rng, low, high):
    """A whole number between low and high, even over the logarithm."""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["clip", "balance", "adapters"])
    if op == "clip":
        dtype = rng.choice(["float32", "bfloat16", "float16"])
        return {"op": op, "way": rng.choice(["measure", "clip"]), "kind": rng.choice(["l2", "l2", "max"]), "tensors": rng.randint(1, 40),
                "elements": spread(rng, 1000, 190000000), "layout": rng.randint(0, 1 << 30), "dtype": dtype, "scaled": dtype == "float16"}
    if op == "balance":
        experts = spread(rng, 8, 1024)
        return {"op": op, "way": rng.choice(["forward", "backward"]), "rows": min(spread(rng, 1, 131072), 65000 * 256 // experts),
                "experts": experts, "top_k": rng.randint(1, min(16, experts)), "dtype": rng.choice(["float32", "float32", "bfloat16", "float16"]),
                "score": rng.choice(["softmax", "sigmoid"]), "normalise": rng.random() < 0.7, "padded": rng.random() < 0.5,
                "masked": rng.choice([0, 0, experts // 8])}
    inner, channels = spread(rng, 48, 8192), spread(rng, 48, 8192)
    if rng.random() < 0.7:
        inner, channels = max(64, inner // 64 * 64), max(64, channels // 64 * 64)
    rows, rank = spread(rng, 1, 8192), spread(rng, 1, 128)
    while rows > 1 and rows * (inner + 2 * channels) > 8000 * 12288:
        rows = rows // 2 + 1
    adapters = min(spread(rng, 1, 256), max(1, (1 << 27) // (rank * (inner + channels))))
    return {"op": op, "rows": rows, "requests": spread(rng, 1, rows) if rng.random() < 0.7 else rows, "adapters": adapters, "rank": rank,
            "inner": inner, "channels": channels, "dtype": rng.choice(["bfloat16", "bfloat16", "float16", "float32"])}


# ------------------------------------------------------- what is in hand before
def generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def normal(g, *shape, scale=1.0, dtype=torch.float32):
    return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)


def tensor_sizes(case):
    """Uneven tensor sizes that add up to the case's elements: vectors beside matrices."""
    r = random.Random(case["layout"])
    n, total = case["tensors"], case["elements"]
    share = [math.exp(r.uniform(0, 6)) for _ in range(n)]
    sizes = [max(1, int(total * v / sum(share))) for v in share]
    sizes[0] += max(0, total - sum(sizes))
    return sizes


LOSS_SCALE = 1024.0


def clip_inputs(case, seed):
    """Gradients as a backward pass leaves them, each tensor of its own size."""
    g, r = generator(seed), random.Random(seed)
    factor = LOSS_SCALE if case["scaled"] else 1.0
    s = {"gradients": [normal(g, n, scale=factor * 1e-3 * math.exp(r.gauss(0, 0.5)), dtype=DTYPES[case["dtype"]]) for n in tensor_sizes(case)]}
    # a limit below what such gradients come to
    s["limit"] = 0.4e-3 * math.sqrt(case["elements"]) if case["kind"] == "l2" else 0.6e-3
    if case["way"] == "clip":
        # a loss that was halved; what a pass has clipped is clipped again by the next, to a limit that
        # goes up and down a little
        s["unscale"], s["limit"], s["turn"] = 2.0, s["limit"] * factor, 1.02
    else:
        s["unscale"] = 1 / factor
    s["device_scale"] = None if s["unscale"] == 1 else torch.tensor(s["unscale"], device="cuda")
    return s


def balance_inputs(case, seed):
    g, dt = generator(seed), DTYPES[case["dtype"]]
    T, E = case["rows"], case["experts"]
    logits = normal(g, T, E, scale=1.5) + normal(g, E, scale=0.5)      # some experts are liked more than others
    if case["masked"]:
        out = torch.rand(T, E, generator=g, device="cuda") < case["masked"] / E
        out[:, : case["top_k"]] = False
        logits = logits.masked_fill(out, -math.inf)
    logits = logits.to(dt)
    s = {"logits": logits, "mask": None,
         "experts": torch.sort(logits.float(), dim=-1, descending=True, stable=True).indices[:, : case["top_k"]].to(torch.int32).contiguous()}
    if case["padded"]:      # a batch of sequences that end where they end: some two thirds of the tokens are real
        length = torch.randint(1, 33, (-(-T // 32),), generator=g, device="cuda")
        s["mask"] = (torch.arange(32, device="cuda") < length[:, None]).reshape(-1)[:T].contiguous()
    if case["way"] == "backward":
        s["counts"], s["tokens"] = counted(s, case)
        s["dloss"] = torch.full((), float(T), device="cuda")      # a loss that is summed over tokens, not their mean
        s["add"] = normal(g, T, E, scale=2e-5, dtype=dt)          # the gradient that comes by the weights
    return s


def adapters_inputs(case, seed):
    g, dt, r = generator(seed), DTYPES[case["dtype"]], random.Random(seed)
    T, n, rank, K, N = case["rows"], case["adapters"], case["rank"], case["inner"], case["channels"]
    # requests of uneven length one after the other, a tenth of them without an adapter
    share = [r.gammavariate(1.5, 1.0) + 1e-3 for _ in range(case["requests"])]
    ends = [0]
    ends += [round(T * sum(share[: i + 1]) / sum(share)) for i in range(len(share))] if len(share) < T else range(1, T + 1)
    ids = [a for b, c in zip(ends, ends[1:]) for a in [-1 if T > 1 and r.random() < 0.1 else r.randrange(n)] * (c - b)]
    s = {"x": normal(g, T, K, dtype=dt), "base": normal(g, T, N, dtype=dt), "ids": torch.tensor(ids, dtype=torch.int32, device="cuda"),
         "down": normal(g, n, rank, K, scale=1 / math.sqrt(K), dtype=dt), "up": normal(g, n, N, rank, scale=0.5 / math.sqrt(rank), dtype=dt),
         "scale": torch.rand(n, generator=g, device="cuda") + 0.5, "list": ids}
    return s


def prepare(case, seed):
    s = {"clip": clip_inputs, "balance": balance_inputs, "adapters": adapters_inputs}[case["op"]](case, seed)
    s["case"] = case
    if own and case["op"] == "clip":
        s["handle"] = dense().GradientNorm(s["gradients"], kind=case["kind"])
    if own and case["op"] == "adapters":
        s["handle"] = dense().Adapters(s.pop("down"), s.pop("up"), s["scale"])
    if case["op"] == "adapters":      # which rows each adapter has: a server knows what it put in its batch
        rows = {}
        [rows.setdefault(a, []).append(t) for t, a in enumerate(s.pop("list"))]
        s["members"] = [(a, torch.tensor(v, device="cuda")) for a, v in rows.items() if a >= 0]
    return s


# ------------------------------------------------------------------- one pass
def run(s):
    return {"clip": run_clip, "balance": run_balance, "adapters": run_adapters}[s["case"]["op"]](s, s["case"])


def run_clip(s, case):
    clip = case["way"] == "clip"
    if clip:
        s["limit"] *= s["turn"]
        s["turn"] = 1 / s["turn"]
    if own:
        r = (s["handle"].clip if clip else s["handle"].measure)(s["limit"], gradient_scale=s["device_scale"])
        return [r.norm, r.scale, r.skip, s["gradients"] if clip else None]
    if case["kind"] == "l2":
        norm = torch.stack([(g.float() * g.float()).sum(dtype=torch.float64) for g in s["gradients"]]).sum().sqrt()
    else:
        norm = torch.stack([g.float().abs().max() for g in s["gradients"]]).max().double()
    unscale = 1.0 if s["device_scale"] is None else s["device_scale"].double()
    norm = norm * unscale
    scale = torch.where(norm > s["limit"], s["limit"] / norm, 1.0) * unscale
    skip = ~torch.isfinite(norm.float())
    scale = torch.where(skip, 0.0, scale).float()
    if clip:
        factor = torch.where(skip, 1.0, scale)
        torch._foreach_copy_(s["gradients"], [g.float() * factor for g in s["gradients"]])
    return [norm.float(), scale, skip.to(torch.int32), s["gradients"] if clip else None]


WEIGHT = 0.01      # the loss's share in the model's


def scores(logits, case):
    """s and p, with 0 where a row has nothing."""
    x = logits.float()
    if case["score"] == "sigmoid":
        p = 1 / (1 + torch.exp(-x))
    else:
        top = x.max(-1, keepdim=True).values
        p = torch.where(top == -math.inf, 0.0, torch.exp(x - top))
    if case["score"] == "sigmoid" and not case["normalise"]:
        return p, p
    total = p.sum(-1, keepdim=True)
    return p, torch.where(total == 0, 0.0, p / total)


def counted(s, case):
    """Each expert's entries among the counted tokens, and the number of those."""
    keep = torch.ones(case["rows"], dtype=torch.bool, device="cuda") if s["mask"] is None else s["mask"]
    found = torch.where(keep[:, None], s["experts"], case["experts"]).reshape(-1)
    return torch.bincount(found, minlength=case["experts"] + 1)[:-1].to(torch.int32), keep.sum().to(torch.int32)


def run_balance(s, case):
    E, k = case["experts"], case["top_k"]
    how = {"score": case["score"], "normalise": case["normalise"], "mask": s["mask"], "weight": WEIGHT}
    if own:
        if case["way"] == "forward":
            return list(dense().balance_loss(s["logits"], s["experts"], **how))
        return dense().balance_loss_backward(s["logits"], s["counts"], s["tokens"], k, dloss=s["dloss"], add=s["add"], **how)
    raw, p = scores(s["logits"], case)
    if case["way"] == "forward":
        counts, n = counted(s, case)
        kept = p if s["mask"] is None else torch.where(s["mask"][:, None], p, 0.0)
        mass = kept.sum(0, dtype=torch.float64)
        loss = torch.where(n == 0, 0.0, WEIGHT * E / (k * n.double() ** 2) * (counts * mass).sum())
        return [loss.float(), counts, mass.float(), n]
    d = s["counts"].double() * (s["dloss"].double() * WEIGHT * E / (k * s["tokens"].double() ** 2))
    d = (d - d.mean()).float() if case["score"] == "softmax" or case["normalise"] else d.float()     # p adds up to 1: a constant drops out
    if case["score"] == "softmax":
        g = p * (d - (p * d).sum(-1, keepdim=True))
    elif case["normalise"]:
        g = p * (1 - raw) * (d - (p * d).sum(-1, keepdim=True))
    else:
        g = raw * (1 - raw) * d
    g = g if s["mask"] is None else torch.where(s["mask"][:, None], g, 0.0)
    return (g + s["add"].float()).to(s["logits"].dtype)


def run_adapters(s, case):
    if own:
        return s["handle"].product(s["x"], s["ids"], s["base"])
    out = s["base"].float()
    parts = [((s["x"][m].float() @ s["down"][a].float().T) @ s["up"][a].float().T) * s["scale"][a] for a, m in s["members"]]
    if parts:
        out = out.index_add(0, torch.cat([m for _, m in s["members"]]), torch.cat(parts))
    return out.to(s["base"].dtype)


# ------------------------------------------------- what a pass cannot do without
def work(case):
    if case["op"] == "clip":
        n = sum(tensor_sizes(case))
        return {"bytes": n * SIZE[case["dtype"]] * (2 if case["way"] == "clip" else 1), "flops": (3 if case["way"] == "clip" else 2) * n}
    if case["op"] == "balance":
        n = case["rows"] * case["experts"] * SIZE[case["dtype"]]
        entries = 4 * case["rows"] * case["top_k"] if case["way"] == "forward" else 2 * n
        return {"bytes": n + entries + case["rows"] * case["padded"] + 8 * case["experts"], "flops": 10 * case["rows"] * case["experts"]}
    T, rank, K, N = case["rows"], case["rank"], case["inner"], case["channels"]
    used = min(case["adapters"], case["requests"])
    return {"bytes": (T * (K + 2 * N) + used * rank * (K + N)) * SIZE[case["dtype"]] + 4 * T, "flops": 2 * T * rank * (K + N)}


# ------------------------------------------------ the definition, in 64 bits
def exact(case, seed):
    return {"clip": exact_clip, "balance": exact_balance, "adapters": exact_adapters}[case["op"]](case, seed)


def exact_clip(case, seed):
    s = clip_inputs(case, seed)
    order = 2 if case["kind"] == "l2" else math.inf
    norm = s["unscale"] * torch.linalg.vector_norm(torch.stack([torch.linalg.vector_norm(g.double(), order) for g in s["gradients"]]), order)
    clip = case["way"] == "clip"
    limit = s["limit"] * s["turn"] if clip else s["limit"]
    factor = s["unscale"] * min(1.0, limit / float(norm))
    return [norm, factor, None, [g.double() * factor for g in s["gradients"]] if clip else None]


def exact_balance(case, seed):
    s = balance_inputs(case, seed)
    T, E, k = case["rows"], case["experts"], case["top_k"]
    keep = torch.ones(T, device="cuda", dtype=torch.float64) if s["mask"] is None else s["mask"].double()
    x = s["logits"].double().requires_grad_(case["way"] == "backward")
    p = torch.softmax(x, -1) if case["score"] == "softmax" else torch.sigmoid(x)
    if case["normalise"] and case["score"] == "sigmoid":
        p = p / p.sum(-1, keepdim=True)
    chosen = torch.zeros(T, E, dtype=torch.float64, device="cuda").scatter_(1, s["experts"].long(), 1.0)
    f = (chosen * keep[:, None]).sum(0) / (k * keep.sum())
    loss = WEIGHT * E * (f * (p * keep[:, None]).sum(0) / keep.sum()).sum()
    if case["way"] == "forward":
        return [loss, None, (p * keep[:, None]).sum(0), None]
    return torch.autograd.grad(loss, x, s["dloss"].double())[0] + s["add"].double()


def exact_adapters(case, seed):
    s = adapters_inputs(case, seed)
    T, step = case["rows"], max(1, (1 << 26) // (case["rank"] * max(case["inner"], case["channels"])))
    if T * case["rank"] * (case["inner"] + case["channels"]) > 1 << 34:
        return None
    out = []
    for a in range(0, T, step):
        i = s["ids"][a:a + step].long()
        j = i.clamp(min=0)
        u = torch.einsum("tk,trk->tr", s["x"][a:a + step].double(), s["down"][j].double())
        d = torch.einsum("tr,tnr->tn", u, s["up"][j].double()) * s["scale"][j].double()[:, None]
        out.append(s["base"][a:a + step].double() + torch.where(i[:, None] >= 0, d, 0.0))
    return torch.cat(out)
