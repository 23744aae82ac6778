"""The gated feed-forward block of an encoder layer, forward and backward.

``gated_mlp`` (also ``ops.gated_mlp``) and ``GatedMLP`` run on the HIP kernels of libhaste_ffi.so:

  y = (act(x w_gate^T) * (x w_up^T)) w_down^T

with both projections, the activation and their product in one kernel, and the gradients of x and
all three weights (those that autograd wants; w_gate's and w_up's come together).  Sums are fp32; what lies
between the products (the hidden values and the gradients of the projections) is rounded to x's dtype, as the matrix
instructions take it (float16: past 65,504 they are infinite).  The backward needs
8 bytes for each hidden value of 16-bit matrices, 14 of float32.  x and the weights: bfloat16,
float16 or float32, all of one dtype; each float32 product is six of bfloat16 parts, whose rounding is
float32's, but where an infinity comes in a NaN may come out.
"""
from __future__ import annotations

import math
from typing import Optional

import torch

from ._lib import host

__all__ = ["gated_mlp", "GatedMLP"]

# HASTE_ACT_* of include/haste_ffi.h
_ACTIVATIONS = {"silu": 0, "gelu": 1, "gelu_tanh": 2}


def _code(activation: str) -> int:
    if activation not in _ACTIVATIONS:
        raise ValueError(f"gated_mlp: activation must be one of {', '.join(_ACTIVATIONS)} (got "
                         f"{activation!r})")
    return _ACTIVATIONS[activation]


def gated_mlp(x: torch.Tensor, w_gate: torch.Tensor, w_up: torch.Tensor, w_down: torch.Tensor,
              activation: str = "silu") -> torch.Tensor:
    """(act(x w_gate^T) * (x w_up^T)) w_down^T for x [..., D], w_gate and w_up [H, D], w_down [O, H].
    ``activation``: "silu", "gelu" (by erf) or "gelu_tanh".  Differentiable once, in reverse mode."""
    return host().gated_mlp(x, w_gate, w_up, w_down, _code(activation))


class GatedMLP(torch.nn.Module):
    """The block with its weights: ``w_gate`` and ``w_up`` [hidden_features, in_features], ``w_down``
    [out_features, hidden_features], initialised like torch.nn.Linear's.  No biases."""

    def __init__(self, in_features: int, hidden_features: int, out_features: Optional[int] = None,
                 activation: str = "silu", device=None, dtype=None):
        super().__init__()
        _code(activation)
        self.in_features, self.hidden_features = in_features, hidden_features
        self.out_features = in_features if out_features is None else out_features
        self.activation = activation
        make = lambda *s: torch.nn.Parameter(torch.empty(*s, device=device, dtype=dtype))  # noqa: E731
        self.w_gate = make(hidden_features, in_features)
        self.w_up = make(hidden_features, in_features)
        self.w_down = make(self.out_features, hidden_features)
        self.reset_parameters()

    def reset_parameters(self) -> None:
        for w in (self.w_gate, self.w_up, self.w_down):
            bound = 1.0 / math.sqrt(max(w.shape[1], 1))
            torch.nn.init.uniform_(w, -bound, bound)

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        return gated_mlp(x, self.w_gate, self.w_up, self.w_down, self.activation)

    def extra_repr(self) -> str:
        return (f"in_features={self.in_features}, hidden_features={self.hidden_features}, "
                f"out_features={self.out_features}, activation={self.activation!r}")
