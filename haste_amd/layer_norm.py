"""Layer norm over the last axis, with the residual sum of an encoder layer in the same pass.

``layer_norm`` (also ``ops.layer_norm``) and ``LayerNorm``, a torch.nn.LayerNorm whose forward
takes a residual, run on the HIP kernels of libhaste_ffi.so:

  h = x + residual, rounded to x's dtype;  y = (h - mean) / sqrt(var + eps) * weight + bias

with fp32 statistics over h as it is stored, so that a call with a residual gives the bits
of the addition followed by a call without.  The backward keeps h and the rows'
statistics, and sums the gradients of weight and bias in a fixed order (no atomics).
x: bfloat16, float16 or float32; weight and bias: x's dtype, or float32.
"""
from __future__ import annotations

from typing import Optional

import torch

from ._lib import host

__all__ = ["layer_norm", "LayerNorm"]


def layer_norm(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None,
               eps: float = 1e-5, residual: Optional[torch.Tensor] = None):
    """y = (h - mean) / sqrt(var + eps) * weight + bias over the last axis of h = x, or, with
    ``residual`` (of x's shape or one that broadcasts to it), (y, h) with h = x + residual.
    Differentiable once, in reverse mode; checks, outputs and the autograd node are native."""
    return host().layer_norm(x, weight, bias, eps, residual)


class LayerNorm(torch.nn.LayerNorm):
    """torch.nn.LayerNorm over one axis (same constructor, parameters and state-dict keys)
    whose forward may take a residual: ``norm(x)`` or ``y, h = norm(x, residual)``."""

    def __init__(self, *args, **kwargs):
        super().__init__(*args, **kwargs)
        if len(self.normalized_shape) != 1 or self.weight is None:
            raise ValueError("LayerNorm: one normalised axis with a weight is supported (got "
                             f"normalized_shape={self.normalized_shape}, "
                             f"elementwise_affine={self.elementwise_affine})")

    def forward(self, x: torch.Tensor, residual: Optional[torch.Tensor] = None):
        return layer_norm(x, self.weight, self.bias, self.eps, residual)
