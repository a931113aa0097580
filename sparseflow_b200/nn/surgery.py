"""Swap the gated MLP of every decoder layer for ``SparseFlowMLP``.

Interface of the reference's ``sparseflow/nn/surgery.py:22-99`` (``replace_llama_mlp_module(model,
policy, verbose)`` -> number of layers replaced): walks ``model.model.layers`` or ``model.layers``,
accepts the ``gate_proj/up_proj/down_proj`` and ``w1/w3/w2`` layouts, and builds the replacement from
the layer's own weights.  ``down_mode`` is passed through (default "dense", the reference's function).
A mixture of experts (a router ``gate`` and a list ``experts`` of such MLPs) becomes a ``SparseFlowMoE``, whose products are all sparse, the down
projection included: with ``down_mode="dense"`` it is taken where the experts' down weights are 2:4 already, so that pruning leaves them as they
are, and refused otherwise.  ``policy`` goes to ``SparseFlowMLP``; like its gate and up projections, those of a mixture are sparse for every
number of tokens.
"""
from __future__ import annotations

import torch
import torch.nn as nn

from .sparseflow_mlp import SparseFlowMLP
from .sparseflow_moe import is_moe, make_sparseflow_moe


def _get_mlp_projections(mlp: nn.Module):
    if all(hasattr(mlp, n) for n in ("gate_proj", "up_proj", "down_proj")):
        return mlp.gate_proj, mlp.up_proj, mlp.down_proj
    if all(hasattr(mlp, n) for n in ("w1", "w3", "w2")):      # w1 = gate, w3 = up, w2 = down
        return mlp.w1, mlp.w3, mlp.w2
    raise RuntimeError(f"Unsupported MLP layout: {type(mlp)}")


def _layers_of(model: nn.Module):
    if hasattr(model, "model") and hasattr(model.model, "layers"):
        return model.model.layers
    if hasattr(model, "layers"):
        return model.layers
    raise RuntimeError("Could not locate transformer layers (expected model.model.layers or model.layers).")


def _is_24(w: torch.Tensor) -> bool:
    return w.shape[-1] % 4 == 0 and not ((w.detach().reshape(-1, 4) != 0).sum(1) > 2).any().item()


def replace_llama_mlp_module(model: nn.Module, policy, verbose: bool = False, down_mode: str = "dense") -> int:
    replaced = 0
    for i, layer in enumerate(_layers_of(model)):
        if not hasattr(layer, "mlp"):
            continue
        if is_moe(layer.mlp):
            if down_mode not in ("dense", "sparse"):
                raise ValueError("down_mode must be 'dense' or 'sparse'")
            if down_mode == "dense" and not all(_is_24(_get_mlp_projections(e)[2].weight) for e in layer.mlp.experts):
                raise RuntimeError("Unsupported MoE layout: down_mode='dense' keeps unpruned down projections, and the experts' products are sparse: "
                                   "pass down_mode='sparse' to prune them, or prune the weights first")
            with torch.inference_mode(False):
                layer.mlp = make_sparseflow_moe(layer.mlp)
            replaced += 1
            if verbose:
                print(f"  layer {i:02d} mlp -> SparseFlowMoE")
            continue
        gate, up, down = _get_mlp_projections(layer.mlp)
        bias = lambda m: None if getattr(m, "bias", None) is None else m.bias.detach()
        with torch.inference_mode(False):
            layer.mlp = SparseFlowMLP(
                hidden_size=gate.in_features, intermediate_size=gate.out_features,
                gate_weight=gate.weight.detach(), up_weight=up.weight.detach(), down_weight=down.weight.detach(),
                gate_bias=bias(gate), up_bias=bias(up), down_bias=bias(down), policy=policy,
                device=str(gate.weight.device), dtype=gate.weight.dtype, down_mode=down_mode)
        replaced += 1
        if verbose:
            print(f"  layer {i:02d} mlp -> SparseFlowMLP")
    return replaced
