"""Embedding lookup with scaling, and its table's gradient by sorted tokens.

``embedding`` (also ``ops.embedding``) and ``Embedding``, a torch.nn.Embedding with a scale, run on the
HIP kernels of libhaste_ffi.so:

  y[..., :] = scale * weight[tokens];  dweight[v] = scale * sum of dy over the places of token v

The gradient is dense, summed in fp32 in a fixed order (the tokens are sorted; no atomics), so
two runs give the same bits.  weight: bfloat16, float16 or float32; tokens: int64 or int32.  A
token outside [0, V) gives a row of zeros and takes no gradient (torch's aborts).
"""
from __future__ import annotations

from typing import Optional

import torch

from ._lib import host

__all__ = ["embedding", "Embedding"]


def embedding(tokens: torch.Tensor, weight: torch.Tensor, scale: float = 1.0,
              padding_idx: Optional[int] = None) -> torch.Tensor:
    """scale * weight[tokens], of tokens' shape and a last axis of weight's width.  The row of
    ``padding_idx`` (negative: from the end) takes no gradient.  Differentiable once, in reverse
    mode, with respect to ``weight``."""
    return host().embedding(tokens, weight, scale, padding_idx)


class Embedding(torch.nn.Embedding):
    """torch.nn.Embedding (same parameters and state-dict keys) whose rows are multiplied by
    ``scale``.  ``max_norm``, ``scale_grad_by_freq`` and ``sparse`` are not taken."""

    def __init__(self, *args, scale: float = 1.0, **kwargs):
        super().__init__(*args, **kwargs)
        if self.max_norm is not None or self.scale_grad_by_freq or self.sparse:
            raise ValueError("Embedding: max_norm, scale_grad_by_freq and sparse are not supported")
        self.scale = float(scale)

    def forward(self, tokens: torch.Tensor) -> torch.Tensor:
        return embedding(tokens, self.weight, self.scale, self.padding_idx)

    def extra_repr(self) -> str:
        return super().extra_repr() + (f", scale={self.scale}" if self.scale != 1.0 else "")
