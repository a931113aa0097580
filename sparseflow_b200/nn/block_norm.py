"""``SparseFlowBlockNorm``: what stands between two blocks of a decoder, as one kernel (``ops.block_norm``).

    z = y  or  norm(y) * post_weight + post_bias;   r = x + scale * gate * z;   h = norm(r) * weight + bias

``forward(x, y)`` returns ``(r, h)``: the residual stream and the input of the next block.  Without ``y`` (in front of the first
block) ``r`` is ``x``.
"""
from __future__ import annotations

from typing import Optional

import torch
import torch.nn as nn

from .. import ops


class SparseFlowBlockNorm(nn.Module):
    def __init__(
        self,
        weight: torch.Tensor,
        bias: Optional[torch.Tensor] = None,
        post_weight: Optional[torch.Tensor] = None,
        post_bias: Optional[torch.Tensor] = None,
        gate: Optional[torch.Tensor] = None,
        scale: float = 1.0,
        eps: float = 1e-5,
        post_eps: Optional[float] = None,
        kind: str = "rms",
    ):
        super().__init__()
        if kind not in ("rms", "layer"):
            raise ValueError(f"kind must be 'rms' or 'layer', got {kind!r}")
        for name, t in (("weight", weight), ("bias", bias), ("post_weight", post_weight), ("post_bias", post_bias), ("gate", gate)):
            self.register_buffer(name, None if t is None else t.detach())
        self.scale, self.eps, self.post_eps, self.kind = float(scale), float(eps), post_eps, kind

    @torch.no_grad()
    def forward(self, x: torch.Tensor, y: Optional[torch.Tensor] = None, gate: Optional[torch.Tensor] = None):
        """``gate`` replaces the module's own: [features], or [sequences, features] / [sequences, 1] for equally long sequences."""
        shape = x.shape
        x = x.reshape(-1, shape[-1])
        if y is None:
            r, h = ops.block_norm(x, weight=self.weight, bias=self.bias, eps=self.eps, kind=self.kind)
        else:
            r, h = ops.block_norm(x, y.reshape(-1, shape[-1]), weight=self.weight, bias=self.bias, post_weight=self.post_weight,
                                  post_bias=self.post_bias, gate=self.gate if gate is None else gate, scale=self.scale, eps=self.eps,
                                  post_eps=self.post_eps, kind=self.kind)
        return r.view(shape), h.view(shape)
