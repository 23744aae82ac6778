"""Log probabilities of given labels under rows of logits, with entropy and the likeliest labels.

``label_log_probs`` (also ``ops.label_log_probs``) runs on the HIP kernels of libhaste_ffi.so: one pass
over the logits for all of its results, one more for the logits' gradient.  It is the softmax side
of an output layer: ``-label_log_probs(z, labels).log_probs`` is its loss, ``top_labels`` its answer.
logits: bfloat16, float16 or float32, rows of any pitch (as ``ops.group_ffi_mul`` gives them); sums and
results are fp32.
"""
from __future__ import annotations

from typing import NamedTuple, Optional

import torch

from ._lib import host

__all__ = ["label_log_probs", "LabelLogProbs"]


class LabelLogProbs(NamedTuple):
    log_probs: Optional[torch.Tensor]      # [..., L], None without labels
    entropy: torch.Tensor                  # [...]
    top_log_probs: Optional[torch.Tensor]  # [..., top], None for top = 0
    top_labels: Optional[torch.Tensor]     # [..., top] int64, None for top = 0


def label_log_probs(logits: torch.Tensor, labels: Optional[torch.Tensor] = None,
                    top: int = 0) -> LabelLogProbs:
    """For logits [..., O] and labels [..., L] (int64 or int32; entries outside [0, O) stand for no
    label and give 0): log softmax at the labels, the rows' entropy, and the ``top`` (up to 128)
    largest log probabilities with their labels, equal logits in the labels' order.  Differentiable
    once, in reverse mode, through ``log_probs`` (of up to 4096 labels a row) and ``entropy``.  Labels
    with a logit of -infinity are ruled out: they have log probability -infinity, no part in the entropy
    and no gradient but that of their own log probability, where ``labels`` ask for it.  A row that
    rules out all of them, or has a NaN or +infinity, gives NaN."""
    return LabelLogProbs(*host().label_log_probs(logits, labels, top))
