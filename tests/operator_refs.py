"""64-bit references of the operators around the FFN, and the error that 32-bit sums and one rounding may leave."""
import torch

HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(g, *shape, dtype=torch.float32, scale=1.0):
    return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)


def close(got, ref, slack, dtype=None):
    """|got - ref| <= one rounding of ref + slack, everywhere; smallest numbers: a step of the subnormals."""
    dtype = dtype or got.dtype
    tiny = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134, torch.float32: 2.0 ** -150}[dtype]
    bound = HALF_STEP[dtype] * (ref.abs() + slack) + slack + tiny
    bad = ~((got.double() - ref).abs() <= bound)
    assert not bad.any(), (int(bad.sum()), ((got.double() - ref).abs() / bound).max().item())


def group_ref(ids, groups, per_row=1):
    """offsets, rows, slots of a grouping, one entry after the other."""
    flat = ids.reshape(-1).tolist()
    order = [i for g in range(groups) for i, v in enumerate(flat) if v == g]
    counts = [0] * (groups + 1)
    for v in flat:
        if 0 <= v < groups:
            counts[v + 1] += 1
    offsets = torch.tensor(counts).cumsum(0).to(torch.int32)
    rows = torch.full((len(flat),), -1, dtype=torch.int32)
    slots = torch.full((len(flat),), -1, dtype=torch.int32)
    for place, i in enumerate(order):
        rows[place] = i // per_row
        slots[i] = place
    return offsets, rows, slots.view(ids.shape)


def route_ref(logits, top_k, renormalize):
    lg = logits.double().cpu()
    lg = torch.where(torch.isnan(lg), -torch.inf, lg).clamp(max=torch.finfo(torch.float32).max)
    n, E = lg.shape
    experts = torch.full((n, top_k), -1, dtype=torch.int32)
    weights = torch.zeros(n, top_k, dtype=torch.float64)
    for t in range(n):
        live = [e for e in range(E) if lg[t, e] > -torch.inf]
        chosen = sorted(live, key=lambda e: (-lg[t, e].item(), e))[:top_k]
        if not chosen:
            continue
        p = torch.exp(lg[t] - lg[t].max())
        p = p / (p[chosen].sum() if renormalize else p.sum())
        experts[t, :len(chosen)] = torch.tensor(chosen, dtype=torch.int32)
        weights[t, :len(chosen)] = p[chosen]
    return weights, experts


def norm_ref(v, layer, w, b, eps):
    """norm(v) * w + b and the size of its terms."""
    mean = v.mean(1, keepdim=True) if layer else torch.zeros_like(v[:, :1])
    inv = 1 / torch.sqrt((v - mean).square().mean(1, keepdim=True) + eps)
    out = (v - mean) * inv * w.double()
    size = (v.abs() + mean.abs() + v.abs().mean(1, keepdim=True)) * inv * w.double().abs()
    return (out, size, inv) if b is None else (out + b.double(), size + b.double().abs(), inv)


def block_norm_ref(x, y, weight, bias, post_weight, post_bias, gate, scale, eps, post_eps, kind):
    """r, h in 64 bits and what 32-bit arithmetic may be off by: 64 roundings of the terms (the sums are trees of at most 20 levels over at most
    16 values a thread; the inverse square root is within two steps)."""
    layer, u = kind == "layer", 64 * 2.0 ** -24
    xd = x.double()
    if y is None:
        r, r_slack = xd, torch.zeros_like(xd)
    else:
        z, z_size = y.double(), y.double().abs()
        if post_weight is not None:
            z, z_size, _ = norm_ref(z, layer, post_weight, post_bias, post_eps)
        g = 1.0
        if gate is not None:
            g = gate.double()
            if g.dim() == 2:
                g = g.repeat_interleave(x.shape[0] // g.shape[0], 0)
        r = xd + scale * g * z
        r_slack = u * (xd.abs() + abs(scale) * (g * z_size if gate is None else g.abs() * z_size))
    h = h_slack = None
    if weight is not None:
        h, size, inv = norm_ref(r, layer, weight, bias, eps)
        # an error of r moves its own value and, through the sums, all of them
        moved = (r_slack + r_slack.mean(1, keepdim=True) + r.abs() * inv * r_slack.square().mean(1, keepdim=True).sqrt()) * inv * weight.double().abs()
        h_slack = u * size + 2 * moved
    return r, r_slack, h, h_slack
