"""``SparseFlowMoE``: a mixture of gated experts over 2:4 weights.

    p = router(x), the top_k experts of every token; out = sum_j p_j * down_e(silu(gate_e(x)) * up_e(x))   (+ residual)

The experts' weights are pruned and compressed once; a forward pass is the router's product, ``moe_route``, one grouped gate|up
product that reads the tokens through the grouping and applies SiLU.mul, one grouped down product, and ``moe_combine``.  Group sizes
stay on the device, so the pass never waits for the GPU and can be captured into a CUDA graph.  No counterpart upstream, whose gated FFN
(sparseflow/nn/sparseflow_mlp.py:15-130) is one expert; interface and error behaviour follow ``SparseFlowMLP``.
"""
from __future__ import annotations

from typing import Optional

import torch
import torch.nn as nn
import torch.nn.functional as F

from .. import ops


class SparseFlowMoE(nn.Module):
    """``router_weight`` [experts, hidden] (float16, bfloat16, float32 or float64: the router's product runs in it); ``gate_weight`` / ``up_weight`` [experts, intermediate,
    hidden], ``down_weight`` [experts, hidden, intermediate] float16 or bfloat16 on CUDA; biases [experts, features] or None.
    ``renormalize``: the weights of a token's experts sum to one."""

    def __init__(
        self,
        router_weight: torch.Tensor,
        gate_weight: torch.Tensor,
        up_weight: torch.Tensor,
        down_weight: torch.Tensor,
        top_k: int,
        renormalize: bool = True,
        gate_bias: Optional[torch.Tensor] = None,
        up_bias: Optional[torch.Tensor] = None,
        down_bias: Optional[torch.Tensor] = None,
        router_bias: Optional[torch.Tensor] = None,
    ):
        super().__init__()
        if gate_weight.dim() != 3:
            raise ValueError(f"gate_weight must be [experts, intermediate, hidden], got {gate_weight.dim()}D")
        E, I, H = gate_weight.shape
        if up_weight.shape != gate_weight.shape or tuple(down_weight.shape) != (E, H, I):
            raise ValueError(f"gate {tuple(gate_weight.shape)}, up {tuple(up_weight.shape)} and down {tuple(down_weight.shape)} do not form experts")
        if tuple(router_weight.shape) != (E, H):
            raise ValueError(f"router_weight must be [{E}, {H}], got {tuple(router_weight.shape)}")
        if not 1 <= top_k <= min(32, E):
            raise ValueError(f"top_k must be 1 .. {min(32, E)}, got {top_k}")
        if H % 64 or I % 64:
            raise ValueError(f"hidden and intermediate size must be multiples of 64, got {H} and {I}")
        self.experts, self.hidden_size, self.intermediate_size = E, H, I
        self.top_k, self.renormalize = int(top_k), bool(renormalize)
        gu = ops.compress_gate_up_experts(gate_weight.detach(), up_weight.detach())
        down = ops.compress_experts(down_weight.detach())
        for name, t in (("router_weight", router_weight), ("router_bias", router_bias), ("gu_values", gu.values), ("gu_meta", gu.meta),
                        ("down_values", down.values), ("down_meta", down.meta), ("gate_bias", gate_bias), ("up_bias", up_bias), ("down_bias", down_bias)):
            self.register_buffer(name, None if t is None else t.detach().contiguous(), persistent=False)

    def _weights(self):
        E, H, I = self.experts, self.hidden_size, self.intermediate_size
        return (ops.CompressedExperts(self.gu_values, self.gu_meta, E, 2 * I, H, gate_up=True),
                ops.CompressedExperts(self.down_values, self.down_meta, E, H, I))

    def route(self, x2d: torch.Tensor) -> ops.Routing:
        logits = F.linear(x2d.to(self.router_weight.dtype), self.router_weight, self.router_bias)
        if logits.dtype == torch.float64:      # the product was in it; the choice is among 32-bit logits
            logits = logits.float()
        return ops.moe_route(logits, self.top_k, renormalize=self.renormalize)

    @torch.no_grad()
    def forward(self, x: torch.Tensor, residual: Optional[torch.Tensor] = None) -> torch.Tensor:
        if x.shape[-1] != self.hidden_size:
            raise ValueError(f"Expected last dim {self.hidden_size}, got {x.shape[-1]}")
        x2d = x.reshape(-1, self.hidden_size)
        routing = self.route(x2d)
        gu, down = self._weights()
        hidden = ops.grouped_sparse_gemm_swiglu(x2d, gu, routing.groups, gather=True, gate_bias=self.gate_bias, up_bias=self.up_bias)
        y = ops.grouped_sparse_gemm(hidden, down, routing.groups, bias=self.down_bias)
        out = ops.moe_combine(y, routing.groups.slots, routing.weights, residual=None if residual is None else residual.reshape(-1, self.hidden_size))
        return out.view(*x.shape)


def _stacked(linears, what: str):
    weights = torch.stack([m.weight.detach() for m in linears])
    biases = [getattr(m, "bias", None) for m in linears]
    if any(b is None for b in biases) != all(b is None for b in biases):
        raise ValueError(f"some experts' {what} projections have a bias and some have none")
    return weights, None if biases[0] is None else torch.stack([b.detach() for b in biases])


def is_moe(module: nn.Module) -> bool:
    """Whether a module has the layout ``make_sparseflow_moe`` reads: a Linear ``gate`` and a list of experts (not their number, a module that
    holds them stacked, or a mapping)."""
    experts = getattr(module, "experts", None)
    return (isinstance(getattr(module, "gate", None), nn.Linear) and isinstance(experts, (nn.ModuleList, nn.Sequential, list, tuple))
            and len(experts) > 0 and all(isinstance(e, nn.Module) for e in experts))


def _is_silu(act) -> bool:
    """SiLU itself, torch's or the module of this name that model libraries have: a name that only contains "silu" or "swish" may be a
    relative of it (Hardswish, a Swish with a slope)."""
    if isinstance(act, str):
        return act.lower() in ("silu", "swish")
    return act is F.silu or type(act) is nn.SiLU or type(act).__name__ == "SiLUActivation"


def _beside(module: nn.Module, read):
    """(name, what) a module can apply beside its children in ``read``, under whatever name: other children, functions, names of functions
    ("act", "hidden_act", ...).  Not what changes nothing: Identity, and Dropout, which inference does not run."""
    for name, m in module.named_children():
        if not any(m is r for r in read) and not isinstance(m, (nn.Identity, nn.Dropout)):
            yield name, m
    for name, v in vars(module).items():
        if callable(v):
            yield name, v
        elif "act" in name.lower() and isinstance(v, str):
            yield name, v


def _is_routing(v) -> bool:
    """Of what a block may apply: the softmax that gives the weights, or the name of its experts' activation."""
    return v is F.softmax or v is torch.softmax or type(v) is nn.Softmax or (isinstance(v, str) and _is_silu(v))


_FACTORS, _BOUNDS = ("scal", "multiplier", "alpha", "beta"), ("softcap", "limit", "clamp", "clip", "capacity")


def _other_settings(module: nn.Module) -> list:
    """Settings of a block (or of the configuration it keeps) or of an expert by which it computes otherwise: a factor, a bound on values or on the
    tokens of an expert, another function of the logits, a choice inside groups of experts."""
    config = getattr(module, "config", None)
    named = ("routed_scaling_factor", "scoring_func", "score_function", "topk_method", "n_group", "topk_group")
    settings = {**{n: getattr(config, n) for n in named if hasattr(config, n)}, **vars(module)}
    found = []
    for name, v in settings.items():
        n, number = name.lower(), isinstance(v, (int, float)) and not isinstance(v, bool)
        has = lambda *words: any(w in n for w in words)  # noqa: E731
        if (number and (has(*_FACTORS) and v != 1 or has(*_BOUNDS) and v != 0 or has("group") and v > 1)
                or isinstance(v, str) and (has("scor") and v != "softmax" or has("method") and v != "greedy")):
            found.append(f"{name} = {v!r}")
    return found


def make_sparseflow_moe(module: nn.Module, top_k: Optional[int] = None, renormalize: Optional[bool] = None) -> SparseFlowMoE:
    """From a module with a router ``gate`` (``nn.Linear``) and a list ``experts`` of gated MLPs (``gate_proj / up_proj / down_proj`` or
    ``w1 / w3 / w2``, all ``nn.Linear``).  A block that has more, and would become another function without it, is refused: other parameters,
    any buffer, another activation than SiLU, another way to weigh or choose the experts.  ``top_k`` and ``renormalize`` default to the module's
    ``top_k`` and ``norm_topk_prob`` (its configuration's where it has none, True without either)."""
    from .surgery import _get_mlp_projections
    if not is_moe(module):
        raise RuntimeError(f"Unsupported MoE layout: {type(module)}")
    projections = [_get_mlp_projections(e) for e in module.experts]
    linears = [module.gate, *(m for three in projections for m in three)]
    for m in linears:
        if not isinstance(m, nn.Linear):
            raise RuntimeError(f"Unsupported MoE layout: {type(m)} as a projection, nn.Linear is what is read")
    read = {id(p) for m in linears for p in (m.weight, m.bias)}
    parts = (module, *module.experts)      # experts in a plain list are not the module's children
    others = [name for part in parts for name, p in part.named_parameters() if id(p) not in read]
    if others:      # an expert that every token takes, a gate on it, a norm inside an expert: leaving them out would change the function
        raise RuntimeError(f"Unsupported MoE layout: {type(module)} has {others} beside its router and its experts' projections")
    buffers = [name for part in parts for name, _ in part.named_buffers()]
    if buffers:     # a bias on the router's choice, say: what a buffer does to the result cannot be seen from here
        raise RuntimeError(f"Unsupported MoE layout: {type(module)} has the buffers {buffers}")
    for e, three in zip(module.experts, projections):
        for name, act in _beside(e, three):
            if not _is_silu(act):
                raise RuntimeError(f"Unsupported MoE layout: experts with {name} = {act}, SiLU is what the products apply")
        if _other_settings(e):
            raise RuntimeError(f"Unsupported MoE layout: experts with {_other_settings(e)}")
    beside = [name for name, v in _beside(module, (module.gate, module.experts)) if not _is_routing(v)] + _other_settings(module)
    if beside:
        raise RuntimeError(f"Unsupported MoE layout: {type(module)} with {beside}: the weights are the softmax of the top_k logits")
    if top_k is None:
        top_k = getattr(module, "top_k", None)
        if top_k is None:
            raise ValueError("top_k is not given and the module has none")
    if renormalize is None:
        renormalize = getattr(module, "norm_topk_prob", getattr(getattr(module, "config", None), "norm_topk_prob", None))
        others = [name for name, v in vars(module).items() if isinstance(v, bool) and "norm" in name.lower()]
        if renormalize is None and others:
            raise RuntimeError(f"Unsupported MoE layout: {type(module)} with {others}: pass renormalize")
        renormalize = True if renormalize is None else bool(renormalize)
    gates, ups, downs = zip(*projections)
    (g, gb), (u, ub), (d, db) = _stacked(gates, "gate"), _stacked(ups, "up"), _stacked(downs, "down")
    router = module.gate
    return SparseFlowMoE(router.weight, g, u, d, top_k, renormalize, gb, ub, db, router.bias)
