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

from typing import Any, Optional

import torch
from torch.autograd.function import once_differentiable

from . import _C, _lib

__all__ = ["layer_norm", "LayerNorm"]


def _rows(t: torch.Tensor, D: int):
    """(t2, ld): t as rows [N, D] with contiguous columns, ld elements apart (0: one row for
    all), copied only where it has no such view."""
    if t.is_neg():
        t = t.resolve_neg()
    if t.dim() != 2:
        t = t.reshape(-1, D)
    ld = t.stride(0) if t.shape[0] > 1 else D
    if (t.stride(1) != 1 and D > 1) or (ld < D and ld != 0):
        t, ld = t.contiguous(), D
    return t, ld


def _check(x, weight, bias, residual) -> None:
    _C.require_device(x, "x")
    _C.dtype_code(x.dtype)
    if x.dim() < 1 or x.shape[-1] < 1:
        raise RuntimeError(f"layer_norm: x must have a last axis to normalise (got {list(x.shape)})")
    for name, t in (("weight", weight), ("bias", bias)):
        if t is None and name == "bias":
            continue
        _C.require_device(t, name)
        if t.dim() != 1 or t.shape[0] != x.shape[-1]:
            raise RuntimeError(f"layer_norm: {name} must be [{x.shape[-1]}] (got {list(t.shape)})")
        if t.dtype != weight.dtype or t.dtype not in (x.dtype, torch.float32):
            raise RuntimeError(f"layer_norm: weight and bias must both be of x's dtype "
                               f"({x.dtype}) or float32 (got {name} {t.dtype})")
        if t.device != x.device:
            raise RuntimeError(f"layer_norm: {name} is on {t.device}, x on {x.device}")
    if residual is not None:
        _C.require_device(residual, "residual")
        if residual.dtype != x.dtype or residual.device != x.device:
            raise RuntimeError(f"layer_norm: residual must be {x.dtype} on {x.device} "
                               f"(got {residual.dtype} on {residual.device})")


def _forward(x, weight, bias, eps, residual, with_stats):
    """(y, h or None, rows of h, weight, stats or None)."""
    D = x.shape[-1]
    rows, ldx = _rows(x, D)
    N = rows.shape[0]
    weight = weight.contiguous()
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    h = res = stats = None
    ldr = 0
    if residual is not None:
        res, ldr = _rows(residual, D)
        h = torch.empty_like(y)
    if with_stats:
        stats = torch.empty(N, 2, dtype=torch.float32, device=x.device)
    if bias is not None:
        bias = bias.contiguous()
    _lib.call("haste_layer_norm", rows.data_ptr(), ldx, None if res is None else res.data_ptr(),
              ldr, weight.data_ptr(), None if bias is None else bias.data_ptr(), y.data_ptr(),
              None if h is None else h.data_ptr(), None if stats is None else stats.data_ptr(), N, D,
              float(eps), _C.dtype_code(x.dtype), _C.dtype_code(weight.dtype), _C.stream_of(x))
    return y, h, rows if h is None else h, weight, stats


class LayerNormFunction(torch.autograd.Function):
    @staticmethod
    @torch.amp.custom_fwd(device_type="cuda")
    def forward(ctx: Any, x, weight, bias, eps, residual):
        y, h, rows, w, stats = _forward(x, weight, bias, eps, residual, True)
        ctx.save_for_backward(rows, w, stats)
        ctx.set_materialize_grads(False)
        ctx.shape, ctx.has_bias = x.shape, bias is not None
        return y if h is None else (y, h)

    @staticmethod
    @once_differentiable
    @torch.amp.custom_bwd(device_type="cuda")
    def backward(ctx, dy, dh=None):
        h, weight, stats = ctx.saved_tensors
        need_x = ctx.needs_input_grad[0] or ctx.needs_input_grad[4]
        need_w = ctx.needs_input_grad[1]
        need_b = ctx.has_bias and ctx.needs_input_grad[2]
        if dy is None:  # only the sum's gradient: it passes through
            dx = dh if need_x else None
            return dx, None, None, None, dx
        D = ctx.shape[-1]
        rows, ldh = _rows(h, D)
        N = rows.shape[0]
        dy, lddy = _rows(dy, D)
        lddh = 0
        if dh is not None:
            dh, lddh = _rows(dh, D)
        dx = torch.empty(ctx.shape, dtype=dy.dtype, device=dy.device) if need_x else None
        dw = torch.empty_like(weight) if need_w else None
        db = torch.empty_like(weight) if need_b else None
        ws = None
        if need_w or need_b:
            n = _lib.lib().haste_layer_norm_bwd_workspace_size(N, D)
            ws = torch.empty(n, dtype=torch.uint8, device=dy.device)
        ptr = lambda t: None if t is None else t.data_ptr()  # noqa: E731
        _lib.call("haste_layer_norm_bwd", dy.data_ptr(), lddy, ptr(dh), lddh, rows.data_ptr(), ldh,
                  weight.data_ptr(), stats.data_ptr(), ptr(dx), ptr(dw), ptr(db), ptr(ws),
                  0 if ws is None else ws.numel(), N, D, _C.dtype_code(dy.dtype),
                  _C.dtype_code(weight.dtype), _C.stream_of(dy))
        return (dx if ctx.needs_input_grad[0] else None, dw, db, None,
                dx if ctx.needs_input_grad[4] else None)


def layer_norm(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None,
               eps: float = 1e-5, residual: Optional[torch.Tensor] = None):
    """y = (h - mean) / sqrt(var + eps) * weight + bias over the last axis of h = x, or, with
    ``residual`` (of x's shape or one that broadcasts to it), (y, h) with h = x + residual."""
    _check(x, weight, bias, residual)
    if residual is not None and residual.shape != x.shape:
        residual = residual.expand(x.shape)
    if torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad
                                    or (bias is not None and bias.requires_grad)
                                    or (residual is not None and residual.requires_grad)):
        return LayerNormFunction.apply(x, weight, bias, eps, residual)
    y, h, _, _, _ = _forward(x, weight, bias, eps, residual, False)
    return y if h is None else (y, h)


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
