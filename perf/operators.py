"""The operators around the gated FFN whose speed counts, each in a plain form (elementary torch operations in 32 bits, rounded once)
and as a program calls it from the package.

  route    the router of a mixture of experts: the ``top_k`` largest of every token's logits, their softmax weights, and the tokens
           grouped by expert (``ops.moe_route``);
  grouped  matrix products grouped by expert with ragged sizes, on 2:4 weights: gate and up with SiLU.mul, the tokens read through the
           grouping (``ops.grouped_sparse_gemm_swiglu``), or one weight per expert with or without a bias, rows already in the order of
           the experts (``ops.grouped_sparse_gemm``);
  combine  the weighted sum of the experts' rows of every token (``ops.moe_combine``);
  norm     what stands between two blocks: the norm of a block's output, its gate and residual scale, the sum with the residual stream,
           and the norm before the next block (``ops.block_norm``);
  lora     low-rank adapters of many requests at once, added to the output of a shared projection (``ops.lora_add``).
"""
import math

import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
_BYTES = {"bf16": 2, "f16": 2, "f32": 4}


def listed():
    return [
        # a step of generation for 32 users: the smallest call, launch and latency
        {"name": "route_decode_32", "kind": "route", "tokens": 32, "experts": 64, "top_k": 6, "dtype": "bf16", "renorm": True, "padded": 0},
        # a batch of prompts with padding at its end, router in 32 bits
        {"name": "route_prompt_8192", "kind": "route", "tokens": 8192, "experts": 128, "top_k": 8, "dtype": "f32", "renorm": False, "padded": 500},
        # generation for one user, eight wide experts: the weights of two of them
        {"name": "gate_up_decode_1", "kind": "grouped", "form": "swiglu", "tokens": 1, "experts": 8, "top_k": 2, "hidden": 4096, "inter": 11008, "dtype": "bf16", "skew": 0.0, "bias": False},
        # a prompt through many narrow experts, their sizes ragged
        {"name": "gate_up_prompt_4096", "kind": "grouped", "form": "swiglu", "tokens": 4096, "experts": 32, "top_k": 4, "hidden": 2048, "inter": 1408, "dtype": "bf16", "skew": 0.5, "bias": False},
        # a step of generation for 64 users, a few tokens for each of many narrow experts
        {"name": "down_batch_64", "kind": "grouped", "form": "store", "tokens": 64, "experts": 64, "top_k": 6, "hidden": 2048, "inter": 1408, "dtype": "f16", "skew": 0.3, "bias": True},
        # a ragged prompt through eight wide experts
        {"name": "down_prompt_1001", "kind": "grouped", "form": "store", "tokens": 1001, "experts": 8, "top_k": 2, "hidden": 4096, "inter": 11008, "dtype": "bf16", "skew": 0.3, "bias": False},
        # the experts' rows of a step of generation
        {"name": "combine_batch_64", "kind": "combine", "tokens": 64, "top_k": 6, "hidden": 2048, "dtype": "f16", "residual": False, "padded": 0},
        # the experts' rows of a prompt with padding, onto the residual stream
        {"name": "combine_prompt_4096", "kind": "combine", "tokens": 4096, "top_k": 8, "hidden": 2048, "dtype": "bf16", "residual": True, "padded": 96},
        # between two blocks in a step of generation for 24 users
        {"name": "norm_decode_24", "kind": "norm", "norm": "rms", "tokens": 24, "hidden": 4096, "dtype": "bf16", "stream": "bf16", "post": False, "gate": "none"},
        # between two blocks of a prompt: a norm on both sides of the sum, a gate for each of four sequences, residual stream in 32 bits
        {"name": "norm_prompt_4096", "kind": "norm", "norm": "rms", "tokens": 4096, "hidden": 8192, "dtype": "bf16", "stream": "f32", "post": True, "gate": "sequence"},
        # a step of generation for 48 requests, each with its adapter
        {"name": "lora_decode_48", "kind": "lora", "tokens": 48, "requests": 48, "adapters": 64, "rank": 16, "K": 4096, "N": 4096, "dtype": "bf16"},
        # eleven prompts of different lengths, some without an adapter, through a wide projection
        {"name": "lora_prompt_4097", "kind": "lora", "tokens": 4097, "requests": 11, "adapters": 8, "rank": 64, "K": 4096, "N": 11008, "dtype": "f16"},
    ]


# The largest listed products bound the drawn ones: 2 * 1001 rows x 4096 x 11008, and eight experts' weights of that size.
_MOST_PRODUCTS = 2002 * 4096 * 11008
_MOST_WEIGHTS = 8 * 4096 * 11008


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _step(v, step, lo):
    return max(lo, v // step * step)


def draw(rng):
    kind = rng.choice(("route", "grouped", "grouped", "grouped", "combine", "norm", "norm", "lora", "lora"))
    dtype = rng.choice(("bf16", "f16"))
    if kind == "route":
        experts = _log(rng, 4, 256)
        tokens = _log(rng, 1, min(16384, 8192 * 128 // experts))
        return {"kind": kind, "tokens": tokens, "experts": experts, "top_k": rng.randint(1, min(8, experts)), "dtype": rng.choice(("bf16", "f16", "f32")),
                "renorm": rng.random() < 0.5, "padded": rng.choice((0, 0, tokens // 7))}
    if kind == "grouped":
        hidden = _step(_log(rng, 512, 4096), 64, 64)
        inter = _step(int(hidden * math.exp(rng.uniform(math.log(0.25), math.log(3.5)))), 64, 64)
        form = rng.choice(("swiglu", "store"))
        weight = hidden * inter * (2 if form == "swiglu" else 1)
        experts = _log(rng, 2, min(128, max(2, _MOST_WEIGHTS // weight)))
        top_k = rng.randint(1, min(8, experts))
        tokens = _log(rng, 1, max(1, min(8192, _MOST_PRODUCTS // weight // top_k)))
        return {"kind": kind, "form": form, "tokens": tokens, "experts": experts, "top_k": top_k, "hidden": hidden, "inter": inter, "dtype": dtype,
                "skew": rng.choice((0.0, 0.5, 1.5)), "bias": form == "store" and rng.random() < 0.5}
    if kind == "combine":
        hidden, top_k = _log(rng, 256, 8192), rng.randint(1, 8)
        hidden = rng.choice((_step(hidden, 64, 64), hidden))
        tokens = _log(rng, 1, max(1, min(16384, 4096 * 8 * 2048 // (hidden * top_k))))
        return {"kind": kind, "tokens": tokens, "top_k": top_k, "hidden": hidden, "dtype": dtype, "residual": rng.random() < 0.5, "padded": rng.choice((0, tokens // 7))}
    if kind == "norm":
        hidden = _log(rng, 128, 16384)
        hidden = rng.choice((_step(hidden, 64, 64), hidden))
        tokens = _log(rng, 1, max(1, min(16384, 4096 * 8192 // hidden)))
        return {"kind": kind, "norm": rng.choice(("rms", "layer")), "tokens": tokens, "hidden": hidden, "dtype": dtype, "stream": rng.choice((dtype, "f32")),
                "post": rng.random() < 0.5, "gate": rng.choice(("none", "channel", "sequence", "row"))}
    K, N = (_step(_log(rng, 1024, 8192), 64, 64) for _ in range(2))
    tokens = _log(rng, 1, max(1, min(8192, 4097 * 15104 // (K + N))))
    requests = rng.choice((tokens, _log(rng, 1, tokens)))
    return {"kind": kind, "tokens": tokens, "requests": min(requests, 256), "adapters": _log(rng, 1, 64), "rank": rng.choice((8, 16, 16, 32, 64)), "K": K, "N": N, "dtype": dtype}


# ------------------------------------------------------------------------------------------------ inputs


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _chosen(case, g):
    """Experts of every token, without repetition: a router's choice, some experts more popular than others."""
    bias = _randn(g, case["experts"]) * case["skew"]
    noise = -torch.log(-torch.log(torch.rand(case["tokens"], case["experts"], generator=g, device="cuda").clamp(1e-9, 1 - 1e-7)))
    return (noise + bias).topk(case["top_k"], dim=1).indices.to(torch.int32)


def _weights_24(g, dt, *shape):
    """2:4 weights N(0, 0.02): two of every four along the last dimension kept."""
    w = (_randn(g, *shape) * 0.02).to(dt).view(-1, 4)
    first = torch.randint(0, 4, (w.shape[0], 1), generator=g, device="cuda")
    second = (first + torch.randint(1, 4, (w.shape[0], 1), generator=g, device="cuda")) % 4
    keep = torch.zeros(w.shape, dtype=torch.bool, device="cuda").scatter_(1, first, True).scatter_(1, second, True)
    return torch.where(keep, w, torch.zeros((), dtype=dt, device="cuda")).view(*shape)


def _inputs(case, seed):
    g, kind, dt = _gen(seed), case["kind"], _TYPES[case["dtype"]]
    if kind == "route":
        logits = (_randn(g, case["tokens"], case["experts"]) * 1.5).to(dt)
        logits[case["tokens"] - case["padded"]:] = -math.inf          # rows of padding go nowhere
        return {"logits": logits}
    if kind == "grouped":
        E, H, I = case["experts"], case["hidden"], case["inter"]
        d = {"experts": _chosen(case, g)}
        if case["form"] == "swiglu":
            d["gate"], d["up"] = _weights_24(g, dt, E, I, H), _weights_24(g, dt, E, I, H)
            d["x"] = _randn(g, case["tokens"], H).to(dt)
        else:
            d["w"] = _weights_24(g, dt, E, H, I)
            d["x"] = _randn(g, case["tokens"] * case["top_k"], I).to(dt)
            d["bias"] = (_randn(g, E, H) * 0.2).to(dt) if case["bias"] else None
        return d
    if kind == "combine":
        n, k = case["tokens"], case["top_k"]
        routed = (n - case["padded"]) * k
        slots = torch.full((n * k,), -1, dtype=torch.int32, device="cuda")
        slots[:routed] = torch.randperm(routed, generator=g, device="cuda").to(torch.int32)
        d = {"y": _randn(g, n * k, case["hidden"]).to(dt), "slots": slots.view(n, k), "weights": torch.softmax(_randn(g, n, k), 1)}
        d["residual"] = _randn(g, n, case["hidden"]).to(dt) if case["residual"] else None
        return d
    if kind == "norm":
        n, H = case["tokens"], case["hidden"]
        vector = lambda m, s: (m + s * _randn(g, H)).to(dt)  # noqa: E731
        layer = case["norm"] == "layer"
        d = {"x": (_randn(g, n, H) * 3 + 0.5).to(_TYPES[case["stream"]]), "y": _randn(g, n, H).to(dt)}
        d["weight"], d["bias"] = vector(1, 0.1), vector(0, 0.1) if layer else None
        d["post_weight"], d["post_bias"] = (vector(1, 0.1), vector(0, 0.1) if layer else None) if case["post"] else (None, None)
        shape = {"none": None, "channel": (H,), "sequence": (4 if n % 4 == 0 else 1, H), "row": (n, 1)}[case["gate"]]
        d["gate"] = None if shape is None else _randn(g, *shape).to(dt)
        return d
    n, K, N, r, A = (case[f] for f in ("tokens", "K", "N", "rank", "adapters"))
    cuts = torch.randint(0, n + 1, (case["requests"] - 1,), generator=g, device="cuda")   # requests of different lengths, one after the other
    if case["requests"] == n:
        cuts = torch.arange(1, n, device="cuda")
    request = torch.bucketize(torch.arange(n, device="cuda"), cuts.sort().values, right=True)
    ids = torch.randint(-1, A, (case["requests"],), generator=g, device="cuda").to(torch.int32)[request]
    return {"ids": ids, "x": _randn(g, n, K).to(dt), "y": _randn(g, n, N).to(dt), "a": (_randn(g, A, r, K) * K ** -0.5).to(dt),
            "b": (_randn(g, A, N, r) * 0.3).to(dt), "scales": 0.25 + torch.rand(A, generator=g, device="cuda")}


def _grouping(ids, groups):
    """Entries of each group in order, padded to the longest: [groups that have any, longest] and which places hold one."""
    ids = ids.reshape(-1).long()
    count = torch.bincount(ids[ids >= 0], minlength=groups)
    active = count.nonzero().view(-1)
    order = torch.sort(torch.where(ids < 0, groups, ids), stable=True).indices
    start = (count.cumsum(0) - count)[active]
    place = torch.arange(int(count.max()) if count.numel() else 0, device=ids.device)
    full = place < count[active, None]
    at = torch.where(full, start[:, None] + place, 0)
    return {"active": active, "at": at, "full": full, "order": order, "count": count}


def prepare(case, seed):
    s = {"case": case, **_inputs(case, seed)}
    kind = case["kind"]
    if kind == "grouped":
        s["plan"] = _grouping(s["experts"], case["experts"])
    if kind == "lora":
        s["plan"] = _grouping(s["ids"], case["adapters"])
    if own:
        from sparseflow_b200 import ops
        if kind == "grouped":       # a program routes once per layer and lays its weights out once
            flat = s["experts"].reshape(-1)
            s["groups"] = ops.group_rows(flat, case["experts"], per_row=case["top_k"] if case["form"] == "swiglu" else 1)
            s["packed"] = ops.compress_gate_up_experts(s["gate"], s["up"]) if case["form"] == "swiglu" else ops.compress_experts(s["w"])
        if kind == "lora":          # the grouping of a batch serves every projection of every layer
            s["groups"] = ops.group_rows(s["ids"], case["adapters"])
            s["bank"] = ops.LoraBank(s["a"], s["b"], s["scales"])
    return s


# ------------------------------------------------------------------------------------------------ the operators


def run(s):
    case = s["case"]
    kind = case["kind"]
    if not own:
        return {"route": _route, "grouped": _grouped, "combine": _combine, "norm": _norm, "lora": _lora}[kind](s)
    from sparseflow_b200 import ops
    if kind == "route":
        r = ops.moe_route(s["logits"], case["top_k"], renormalize=case["renorm"])
        return {"weights": r.weights, "experts": r.experts, "offsets": r.groups.offsets, "rows": r.groups.rows, "slots": r.groups.slots}
    if kind == "grouped":
        if case["form"] == "swiglu":
            return ops.grouped_sparse_gemm_swiglu(s["x"], s["packed"], s["groups"], gather=True)
        return ops.grouped_sparse_gemm(s["x"], s["packed"], s["groups"], bias=s["bias"])
    if kind == "combine":
        return ops.moe_combine(s["y"], s["slots"], s["weights"], residual=s["residual"])
    if kind == "norm":
        return ops.block_norm(s["x"], s["y"], weight=s["weight"], bias=s["bias"], post_weight=s["post_weight"], post_bias=s["post_bias"],
                              gate=s["gate"], scale=0.75, eps=1e-5, kind=case["norm"])
    return ops.lora_add(s["y"], s["x"], s["bank"], s["groups"])


def _route(s):
    case, logits = s["case"], s["logits"].float()
    n, k, E = case["tokens"], case["top_k"], case["experts"]
    value, index = torch.sort(logits, dim=1, descending=True, stable=True)       # ties: the lowest index first
    value, index = value[:, :k], index[:, :k]
    routed = value > -math.inf
    e = torch.where(routed, torch.exp(value - value[:, :1]), 0.0)
    total = e.sum(1, keepdim=True) if case["renorm"] else torch.where(routed[:, :1], torch.exp(logits - value[:, :1]), 0.0).sum(1, keepdim=True)
    weights = torch.where(routed, e / total, 0.0)
    experts = torch.where(routed, index, -1).to(torch.int32)
    flat = torch.where(routed, index, E).reshape(-1)
    order = torch.sort(flat, stable=True).indices
    count = torch.zeros(E + 1, dtype=torch.int64, device=flat.device).scatter_add_(0, flat, torch.ones_like(flat))
    ends = count.cumsum(0)
    offsets = torch.cat([torch.zeros_like(ends[:1]), ends[:E]]).to(torch.int32)
    place = torch.arange(n * k, device=flat.device)
    rows = torch.where(place < ends[E - 1], order // k, -1).to(torch.int32)
    slots = torch.empty_like(place).scatter_(0, order, place)
    slots = torch.where(flat < E, slots, -1).to(torch.int32).view(n, k)
    return {"weights": weights, "experts": experts, "offsets": offsets, "rows": rows, "slots": slots}


def _products(x, w, plan):
    """[rows in the order of the groups, columns]: every row times its group's weight, groups padded to the longest."""
    y = torch.bmm(x, w.index_select(0, plan["active"]).float().transpose(1, 2))
    return y[plan["full"]]


def _grouped(s):
    case, plan = s["case"], s["plan"]
    if case["form"] == "swiglu":
        x = s["x"][plan["order"][plan["at"]] // case["top_k"]].float()
        gate = _products(x, s["gate"], plan)
        return (gate / (1 + torch.exp(-gate)) * _products(x, s["up"], plan)).to(s["x"].dtype)
    y = _products(s["x"][plan["at"]].float(), s["w"], plan)
    if s["bias"] is not None:
        y = y + s["bias"].float()[plan["active"]].unsqueeze(1).expand(-1, plan["at"].shape[1], -1)[plan["full"]]
    return y.to(s["x"].dtype)


def _combine(s):
    slots = s["slots"].long()
    rows = s["y"][slots.clamp(min=0)].float()
    out = (torch.where(slots >= 0, s["weights"], 0.0).unsqueeze(2) * rows).sum(1)
    return (out if s["residual"] is None else out + s["residual"].float()).to(s["y"].dtype)


def _normed(v, kind, weight, bias):
    if kind == "layer":
        v = v - v.mean(1, keepdim=True)
    v = v * torch.rsqrt((v * v).mean(1, keepdim=True) + 1e-5) * weight.float()
    return v if bias is None else v + bias.float()


def _norm(s):
    kind, x, y = s["case"]["norm"], s["x"].float(), s["y"].float()
    if s["post_weight"] is not None:
        y = _normed(y, kind, s["post_weight"], s["post_bias"])
    if s["gate"] is not None:
        g = s["gate"].float()
        y = y * (g.repeat_interleave(x.shape[0] // g.shape[0], 0) if g.dim() == 2 else g)
    r = x + 0.75 * y
    return [r.to(s["x"].dtype), _normed(r, kind, s["weight"], s["bias"]).to(s["y"].dtype)]


def _lora(s):
    plan, y = s["plan"], s["y"].float()
    x = s["x"][plan["order"][plan["at"]]].float()
    t = torch.bmm(x, s["a"].index_select(0, plan["active"]).float().transpose(1, 2))
    d = _products(t * s["scales"][plan["active"], None, None], s["b"], plan)
    return y.index_add_(0, plan["order"][:d.shape[0]], d).to(s["y"].dtype)


# ------------------------------------------------------------------------------------------------ work and 64 bits


def _active(case):
    """Experts that have a token, on average over equally popular experts."""
    E, n, k = case["experts"], case["tokens"], case["top_k"]
    return E * (1 - (1 - k / E) ** n)


def work(case):
    """Inputs read once and outputs written once; operations: the products of the kept half of 2:4 weights, multiply-adds as two."""
    kind, b = case["kind"], _BYTES[case["dtype"]]
    n = case["tokens"]
    if kind == "route":
        return {"bytes": n * case["experts"] * b + n * case["top_k"] * 16 + 4 * case["experts"], "flops": 4 * n * case["experts"]}
    if kind == "grouped":
        H, I, S = case["hidden"], case["inter"], n * case["top_k"]
        if case["form"] == "swiglu":
            return {"bytes": _active(case) * 2 * H * I * 1.125 + 2 * (n * H + S * I) + 4 * S, "flops": 2 * S * H * I}
        return {"bytes": _active(case) * (H * I * 1.125 + (2 * H if case["bias"] else 0)) + 2 * S * (H + I), "flops": S * H * I}
    if kind == "combine":
        routed = (n - case["padded"]) * case["top_k"]
        return {"bytes": 2 * case["hidden"] * (routed + n + (n if case["residual"] else 0)) + 8 * n * case["top_k"], "flops": 2 * routed * case["hidden"]}
    if kind == "norm":
        H = case["hidden"]
        return {"bytes": n * H * (2 * _BYTES[case["stream"]] + 2 * b), "flops": n * H * (12 if case["post"] else 8)}
    N, K, r = case["N"], case["K"], case["rank"]
    banks = min(case["adapters"], case["requests"])
    return {"bytes": b * (n * (K + 2 * N) + banks * r * (K + N)), "flops": 2 * n * r * (K + N)}


def exact(case, seed):
    d, kind = _inputs(case, seed), case["kind"]
    if kind == "route":
        # sorted by (expert, token) with a key per entry: the grouping written as counts of smaller keys
        n, k, E = case["tokens"], case["top_k"], case["experts"]
        lg = d["logits"].double()
        key = lg.clone()
        weights = torch.zeros(n, k, dtype=torch.float64, device=lg.device)
        experts = torch.full((n, k), -1, dtype=torch.int32, device=lg.device)
        everyone = torch.logsumexp(lg, 1)
        for j in range(k):
            top = key.max(1).values
            index = torch.where(key == top[:, None], torch.arange(E, device=lg.device), E).min(1).values
            some = top > -math.inf
            experts[:, j] = torch.where(some, index, -1).to(torch.int32)
            weights[:, j] = torch.where(some, torch.exp(top - everyone), 0.0)
            key[torch.arange(n, device=lg.device), index] = -math.inf
        if case["renorm"]:
            total = weights.sum(1, keepdim=True)
            weights = torch.where(total > 0, weights / total, 0.0)
        return {"weights": weights, "experts": experts, "offsets": None, "rows": None, "slots": None}
    if kind == "grouped":
        flat = d["experts"].reshape(-1).long()
        out = []
        for e in range(case["experts"]):
            entries = (flat == e).nonzero().view(-1)
            if not entries.numel():
                continue
            if case["form"] == "swiglu":
                x = d["x"][entries // case["top_k"]].double()
                gate = x @ d["gate"][e].double().t()
                out.append(gate * torch.sigmoid(gate) * (x @ d["up"][e].double().t()))
            else:
                first = sum(len(o) for o in out)
                y = d["x"][first:first + entries.numel()].double() @ d["w"][e].double().t()
                out.append(y if d["bias"] is None else y + d["bias"][e].double())
        return torch.cat(out)
    if kind == "combine":
        out = torch.zeros(case["tokens"], case["hidden"], dtype=torch.float64, device="cuda")
        for j in range(case["top_k"]):
            t = (d["slots"][:, j] >= 0).nonzero().view(-1)
            out[t] += d["weights"][t, j, None].double() * d["y"][d["slots"][t, j].long()].double()
        return out if d["residual"] is None else out + d["residual"].double()
    if kind == "norm":
        def normed(v, w, b):
            if case["norm"] == "layer":
                var, mean = torch.var_mean(v, 1, unbiased=False, keepdim=True)
                v = (v - mean) / torch.sqrt(var + 1e-5) * w.double()
            else:
                v = v / torch.sqrt(v.square().mean(1, keepdim=True) + 1e-5) * w.double()
            return v if b is None else v + b.double()

        y = d["y"].double()
        if d["post_weight"] is not None:
            y = normed(y, d["post_weight"], d["post_bias"])
        if case["gate"] == "sequence":
            n = d["gate"].shape[0]
            y = (y.view(n, -1, case["hidden"]) * d["gate"].double()[:, None]).view_as(y)
        elif d["gate"] is not None:
            y = y * d["gate"].double()
        r = d["x"].double() + 0.75 * y
        return [r, normed(r, d["weight"], d["bias"])]
    out = d["y"].double()
    for i in range(case["adapters"]):
        t = (d["ids"] == i).nonzero().view(-1)
        if t.numel():
            out[t] += d["scales"][i].double() * (d["x"][t].double() @ d["a"][i].double().t()) @ d["b"][i].double().t()
    return out
