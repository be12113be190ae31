"""The gated feed-forward block that may end a stage (no counterpart in the reference): all channels of a token are
mixed, where a BiGEMM block mixes 16 tokens and the channels of one group.

    x + gamma * ((silu(n W_g^T) * (n W_u^T)) W_d^T),   n = LayerNorm(x)

On the hip backend the norm is ``layer_norm_hip``, both projections with their gate are ``gated_linear_hip``, and LayerScale with
the residual is ``block_norms_hip``; the projection back is a plain Linear.  Drop-path is for the BiGEMM blocks: this one runs always.
"""

from __future__ import annotations

import torch
import torch.nn as nn
import torch.nn.functional as F
from torch import Tensor

from omniwave_amd.gated import gated_linear_hip
from omniwave_amd.hip import SUPPORTED_DTYPES
from omniwave_amd.norms import MAX_CHANNELS, block_norms_hip, gpu_reason, layer_norm_hip

EPS = 1e-6


class GatedFeedForward(nn.Module):
    """``[..., dim]`` -> ``[..., dim]`` over ``hidden`` gated values."""

    def __init__(self, dim: int, hidden: int, layer_scale_init: float = 1e-5, backend: str = "auto") -> None:
        super().__init__()
        if hidden < 1:
            raise ValueError(f"hidden must be at least 1, got {hidden}")
        self.dim = dim
        self.backend = backend
        self.norm_weight = nn.Parameter(torch.ones(dim))
        self.norm_bias = nn.Parameter(torch.zeros(dim))
        self.gate = nn.Linear(dim, hidden, bias=False)
        self.up = nn.Linear(dim, hidden, bias=False)
        self.down = nn.Linear(hidden, dim, bias=False)
        self.gamma = nn.Parameter(torch.full((dim,), layer_scale_init))

    def _hip(self, x: Tensor) -> bool:
        if self.backend not in ("hip", "auto"):
            return False
        reason = gpu_reason(x)
        if reason is None and x.dtype not in SUPPORTED_DTYPES:
            reason = f"dtype {x.dtype}"
        if reason is None and self.dim > MAX_CHANNELS:
            reason = f"{self.dim} channels; at most {MAX_CHANNELS}"
        if reason is not None and self.backend == "hip":
            raise RuntimeError(f"hip feed-forward not supported: {reason}")
        return reason is None

    def forward(self, x: Tensor) -> Tensor:
        if self._hip(x):
            normed = layer_norm_hip(x, self.norm_weight, self.norm_bias, EPS)
            # Under autocast the weights are of another type than x, and so is what the projection back returns; the products
            # are x's (in fp32 where x is).
            hidden = gated_linear_hip(normed, self.gate.weight.to(x.dtype), self.up.weight.to(x.dtype))
            return block_norms_hip(x, self.down(hidden).to(x.dtype), gate=self.gamma)[0]
        normed = F.layer_norm(x, (self.dim,), self.norm_weight.to(x.dtype), self.norm_bias.to(x.dtype), EPS)
        return x + self.gamma.to(x.dtype) * self.down(F.silu(self.gate(normed)) * self.up(normed))
