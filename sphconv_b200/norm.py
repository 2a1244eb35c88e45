"""Norms of feature rows, and the norms before and after a block fused with the block's gate and residual scale: what a head puts
around its attention and its linear layers.  They take the rows [n, C] that ``SparseConvTensor.feature`` and a head's queries are
(any leading dimensions), so ``RowNorm`` stands in a ``Sequential`` where BatchNorm1d does.  No reference counterpart.

    normed = row_norm(x, weight)                                           # before the first block
    x, normed = residual_norm(block(normed), x, weight, gate=g, scale=s, next_weight=w)   # behind a block, before the next one
"""
from typing import Optional, Tuple

import torch
from torch import nn

from . import _capi as C


def row_norm(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None, eps: float = 1e-6,
             center: bool = False) -> torch.Tensor:
    """x / sqrt(mean(x^2) + eps) * weight + bias over the last dimension, or (center) the layer norm
    (x - mean) / sqrt(var + eps) * weight + bias.

    x: contiguous float32, float16 or bfloat16 rows of at most 8192 channels.  weight, bias [C]: any of these types.  Statistics are
    float32; the result has the dtype of x.  Differentiable once, backward."""
    return C.host().residual_norm(None, x, None, None, None, None, weight, bias, eps, center)[1]


def residual_norm(block: torch.Tensor, residual: torch.Tensor, weight: Optional[torch.Tensor] = None,
                  bias: Optional[torch.Tensor] = None, *, gate: Optional[torch.Tensor] = None, scale: Optional[torch.Tensor] = None,
                  next_weight: Optional[torch.Tensor] = None, next_bias: Optional[torch.Tensor] = None, eps: float = 1e-6,
                  center: bool = False) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """What follows a block, in one pass over the rows -> (out, normed):

        inner  = norm(block) * weight + bias                       the block itself without a weight
        out    = residual + scale * sigmoid(gate) * inner
        normed = norm(out) * next_weight + next_bias               None without a next_weight; from `out` before it is rounded

    norm is row_norm's.  block, residual: contiguous rows of one shape and dtype.  gate: logits of that dtype, the rows' shape or
    one value a row [..., 1].  weight, bias, scale, next_weight, next_bias [C]: float32, float16 or bfloat16.  All of them are
    differentiable (once, backward); gradients of the parameters are summed in float32 in a fixed order, without atomics."""
    return C.host().residual_norm(block, residual, gate, weight, bias, scale, next_weight, next_bias, eps, center)


class RowNorm(nn.Module):
    """row_norm with its parameters: RMS norm, or with center=True layer norm with a bias."""

    def __init__(self, channels: int, eps: float = 1e-6, center: bool = False):
        super().__init__()
        self.channels, self.eps, self.center = channels, eps, center
        self.weight = nn.Parameter(torch.ones(channels))
        self.register_parameter("bias", nn.Parameter(torch.zeros(channels)) if center else None)

    def extra_repr(self):
        return "{}, eps={}, center={}".format(self.channels, self.eps, self.center)

    def forward(self, x):
        return row_norm(x, self.weight, self.bias, self.eps, self.center)


class ResidualNorm(nn.Module):
    """residual_norm with its parameters: forward(block, residual, gate=None) -> (out, normed).  `initial_scale`: the residual scale
    per channel at the start (None: no scale); `norm_block`: a norm behind the block too, not only in front of the next one."""

    def __init__(self, channels: int, eps: float = 1e-6, center: bool = False, norm_block: bool = True,
                 initial_scale: Optional[float] = None):
        super().__init__()
        self.channels, self.eps, self.center = channels, eps, center

        def vector(value, wanted=True):
            return nn.Parameter(torch.full((channels,), float(value))) if wanted else None

        self.register_parameter("weight", vector(1.0, norm_block))
        self.register_parameter("bias", vector(0.0, norm_block and center))
        self.register_parameter("scale", vector(initial_scale or 0.0, initial_scale is not None))
        self.next_weight = vector(1.0)
        self.register_parameter("next_bias", vector(0.0, center))

    def extra_repr(self):
        return "{}, eps={}, center={}".format(self.channels, self.eps, self.center)

    def forward(self, block, residual, gate=None):
        return residual_norm(block, residual, self.weight, self.bias, gate=gate, scale=self.scale, next_weight=self.next_weight,
                             next_bias=self.next_bias, eps=self.eps, center=self.center)
