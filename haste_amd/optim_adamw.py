"""AdamW over many tensors at once, for the encoder in front of an FFI layer, and the norm that
clips its gradients.

``AdamW`` takes the place of torch.optim.AdamW (decoupled weight decay, bias-corrected
moments, in fp32); beside it:
  * bfloat16 and float16 parameters are stepped in place, with stochastic rounding (as
    SRSgd does; per param group ``seed`` is read and then incremented every step), so that no
    fp32 copy of them is needed; float32 parameters are rounded to nearest;
  * ``state_bits=8`` keeps the first moment and the root of the second as float8_e4m3fn with
    one power-of-two scale (float8_e8m0fnu) for each 128 elements, rounded stochastically:
    2.03 bytes an element instead of 8.  The root then has a standing spread of about 15 % from
    its rounding (with 32 bits 1.6 % from the gradients alone, at beta2 = 0.999);
  * ``step(grad_scale=...)`` takes a factor for all gradients that is on the device, such as
    ``grad_norm``'s; a NaN there leaves parameters and states as they are.
The tensors of a group are stepped by one launch for each 64 of them (and for each dtype of
parameters and gradients, and each count of steps).  Random bits: Philox4x32-10 keyed by the
group's seed, with the position of a tensor among those of all groups and of an element in it as
counters, so a step's results depend on nothing else and groups of one seed draw apart.

State of a parameter (created at its first step): ``step``, an int; with 32 bits ``exp_avg`` and
``exp_avg_sq``, fp32 of its shape; with 8 bits ``exp_avg`` and ``rms`` (codes, of its elements in
order, padded to a multiple of 128) with ``exp_avg_scale`` and ``rms_scale``.
"""
from __future__ import annotations

import math
from typing import Iterable, Tuple

import torch
from torch.optim import Optimizer

from . import _C, _lib
from .optim_sr import run_hooked

__all__ = ["AdamW", "grad_norm"]

STATE_BLOCK = 128  # elements of an 8-bit state that share a scale
_STATE = {32: {"exp_avg": torch.float32, "exp_avg_sq": torch.float32},
          8: {"exp_avg": torch.float8_e4m3fn, "rms": torch.float8_e4m3fn,
              "exp_avg_scale": torch.float8_e8m0fnu, "rms_scale": torch.float8_e8m0fnu}}


def _dense(t: torch.Tensor, name: str) -> torch.Tensor:
    """t with its values in memory in order, as the kernels read it."""
    if t.layout is not torch.strided:
        raise RuntimeError(f"{name} must be dense (got {t.layout})")
    if t.is_neg():
        t = t.resolve_neg()
    return t if t.is_contiguous() else t.contiguous()


def grad_norm(tensors: Iterable[torch.Tensor], max_norm: float = math.inf
              ) -> Tuple[torch.Tensor, torch.Tensor]:
    """(norm, coef): the 2-norm over all the tensors and min(1, max_norm / (norm + 1e-6)), the
    factor of torch.nn.utils.clip_grad_norm_, as fp32 scalars on their device, without a
    sync and without touching the tensors: ``AdamW.step(grad_scale=coef)`` applies it.
    coef is NaN where norm is not finite.  Neither is differentiable."""
    tensors = list(tensors)
    if not tensors:
        raise RuntimeError("grad_norm: no tensors")
    got = _lib.host().grad_norm(tensors, float(max_norm))
    if got is not None:
        return got
    for t in tensors:
        _C.require_device(t, "gradients")
    n, dev = len(tensors), tensors[0].device
    tensors = [_dense(t, "gradients") for t in tensors]
    for t in tensors:
        if t.device != dev:
            raise RuntimeError(f"grad_norm: tensors must be on one device (got {dev}, {t.device})")
    arr = (_lib.GradTensor * n)(*[(t.data_ptr(), t.numel(), _C.dtype_code(t.dtype))
                                  for t in tensors])
    out = torch.empty(2, dtype=torch.float32, device=dev)
    size = _lib.lib().haste_grad_norm_workspace_size(n)
    ws = torch.empty(size, dtype=torch.uint8, device=dev)
    # (torch's default stream is handle 0 on every device, which means the current one's)
    with torch.cuda.device(dev):
        _lib.call("haste_grad_norm", arr, n, float(max_norm), out.data_ptr(), ws.data_ptr(), size,
                  _C.stream_of(out))
    return out[0], out[1]


class AdamW(Optimizer):
    def __init__(self, params, lr: float = 1e-3, betas: Tuple[float, float] = (0.9, 0.999),
                 eps: float = 1e-8, weight_decay: float = 1e-2, state_bits: int = 32,
                 stochastic_rounding: bool = True, seed: int = 123):
        if not lr >= 0.0:
            raise ValueError(f"Invalid learning rate: {lr}")
        if not eps >= 0.0:
            raise ValueError(f"Invalid epsilon value: {eps}")
        if not all(0.0 <= b < 1.0 for b in betas):
            raise ValueError(f"Invalid beta parameters: {betas}")
        if not weight_decay >= 0.0:
            raise ValueError(f"Invalid weight_decay value: {weight_decay}")
        super().__init__(params, dict(lr=lr, betas=tuple(betas), eps=eps,
                                      weight_decay=weight_decay, state_bits=state_bits,
                                      stochastic_rounding=stochastic_rounding, seed=seed))

    def add_param_group(self, param_group) -> None:
        if isinstance(param_group, dict):  # (torch refuses anything else)
            bits = param_group.get("state_bits", self.defaults["state_bits"])
            if bits not in _STATE:
                raise ValueError(f"state_bits must be 8 or 32 (got {bits})")
        super().add_param_group(param_group)

    @staticmethod
    def _state_size(key: str, bits: int, p: torch.Tensor) -> int:
        blocks = -(-p.numel() // STATE_BLOCK)
        return p.numel() if bits == 32 else blocks if key.endswith("_scale") else blocks * STATE_BLOCK

    def _new_state(self, p: torch.Tensor, bits: int) -> dict:
        state = self.state[p]
        state["step"] = 0
        for key, dtype in _STATE[bits].items():
            if bits == 32:
                state[key] = torch.zeros(p.shape, dtype=dtype, device=p.device)
            else:  # code 127 of a scale is 1
                fill = 127 if key.endswith("_scale") else 0
                state[key] = torch.full((self._state_size(key, bits, p),), fill, dtype=torch.uint8,
                                        device=p.device).view(dtype)
        return state

    def load_state_dict(self, state_dict) -> None:
        # torch casts floating-point state to the parameter's dtype: put the states back as they
        # were saved.  All of it is checked before any of it replaces anything, by a hook behind
        # the others, which sees what they made of the saved state.
        saved = []
        check = self.register_load_state_dict_pre_hook(
            lambda _, state: saved.append(self._check_saved(state)))
        try:
            super().load_state_dict(state_dict)
        finally:
            check.remove()
        params = [p for group in self.param_groups for p in group["params"]]
        for p, got in zip(params, saved[0]):
            for key, t in got.items():
                self.state[p][key] = t if key == "step" else t.to(device=p.device).clone()

    def _check_saved(self, state_dict) -> list:
        """What a saved state holds for each parameter, in order ({} for nothing); ValueError where
        it does not fit them."""
        found, groups = [], state_dict["param_groups"]
        if [len(g["params"]) for g in groups] != [len(g["params"]) for g in self.param_groups]:
            return found  # (torch refuses it)
        for group, saved in zip(self.param_groups, groups):
            bits = saved.get("state_bits")
            if bits not in _STATE:
                raise ValueError(f"AdamW: state_bits of the saved groups must be 8 or 32 (got {bits})")
            for p, index in zip(group["params"], saved["params"]):
                got = state_dict["state"].get(index)
                found.append({})
                if not got:
                    continue
                if "step" not in got:
                    raise ValueError("AdamW: a saved state has no step")
                found[-1]["step"] = int(got["step"])
                for key, dtype in _STATE[bits].items():
                    t = got.get(key)
                    if not isinstance(t, torch.Tensor) or t.dtype != dtype or \
                            t.numel() != self._state_size(key, bits, p):
                        raise ValueError(f"AdamW: saved state {key} does not fit a parameter of "
                                         f"shape {list(p.shape)} with {bits}-bit states")
                    found[-1][key] = t
        return found

    def step(self, closure=None, *, grad_scale=None):
        """One step, torch.optim.Optimizer.step semantics, hooks included.  ``grad_scale``: an
        fp32 tensor of one element on the parameters' device that multiplies every gradient
        as it is read (1 when None); where it is NaN the kernels change no parameter and no
        moment (the counts of steps and the seed go on)."""
        return run_hooked(self, "_adamw_step", (closure,),
                          {} if grad_scale is None else {"grad_scale": grad_scale})

    step.hooked = True  # Optimizer.__init__ then leaves it unwrapped

    def _adamw_step(self, closure=None, *, grad_scale=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        if torch.cuda.is_initialized() and torch._C._cuda_isCurrentStreamCapturing():
            raise RuntimeError("AdamW.step cannot be captured: the count of steps and the seed "
                               "are the host's, and a replay would repeat one step's")
        if grad_scale is not None:
            _C.require_device(grad_scale, "grad_scale")
            if grad_scale.dtype != torch.float32 or grad_scale.numel() != 1:
                raise RuntimeError(f"grad_scale must be one float32 (got {list(grad_scale.shape)} "
                                   f"{grad_scale.dtype})")
        stream = 0  # (of the group's first parameter)
        for group in self.param_groups:
            self._step_group(group, stream, grad_scale)
            stream += len(group["params"])
        return loss

    def _step_group(self, group, stream, grad_scale) -> None:
        bits, seed = group["state_bits"], group["seed"]
        (beta1, beta2), sr = group["betas"], bool(group["stochastic_rounding"])
        args = (float(group["lr"]), float(beta1), float(beta2), float(group["eps"]),
                float(group["weight_decay"]))
        if not _lib.host().adamw_step(group["params"], self.state, bits, *args, sr, seed, stream,
                                      grad_scale):
            with torch.no_grad():
                self._step_any(group["params"], bits, args, sr, seed, stream, grad_scale)
        group["seed"] += 1

    def _step_any(self, params, bits, args, sr, seed, first, grad_scale) -> None:
        """The step of any parameters: those that are not plain through copies, with states made
        where there are none yet."""
        batches, device = self._rows(params, bits, first)
        if not batches:
            return
        scale = None
        if grad_scale is not None:
            if grad_scale.get_device() != device:
                raise RuntimeError(f"AdamW: grad_scale is on {grad_scale.device}, the parameters "
                                   f"on cuda:{device}")
            grad_scale = _dense(grad_scale, "grad_scale")
            scale = grad_scale.data_ptr()
        # torch's default stream is handle 0 on every device, which means the current one's
        with torch.cuda.device(device):
            self._launch(batches, bits, args, sr, seed, scale,
                         torch._C._cuda_getCurrentRawStream(device))

    @staticmethod
    def _launch(batches, bits, args, sr, seed, scale, stream) -> None:
        for (w_code, g_code, step), stepped in batches.items():
            rows = (_lib.AdamwTensor * len(stepped))(*[s[1] for s in stepped])
            _lib.call("haste_adamw_step", rows, len(stepped), w_code, g_code, bits, *args, step,
                      int(sr), int(seed), scale, stream)
            # (only now: a refused step leaves the counts as they were)
            for state, _, p, w, _ in stepped:
                state["step"] = step
                if w.data_ptr() != p.data_ptr():
                    p.copy_(w)
            # written through raw pointers: move the version counters as torch would
            torch.autograd.graph.increment_version([s[2] for s in stepped])

    def _rows(self, params, bits, first):
        """The tables of the step of any parameters, whose random streams count from `first`:
        ({(w dtype, g dtype, step): [(state, row, parameter, its contiguous tensor or copy, the
        gradient's)]}, device)."""
        batches, device = {}, None
        for index, p in enumerate(params, first):
            grad = p.grad
            if grad is None:
                continue
            _C.require_device(p, "parameters")
            device = p.device if device is None else device
            for t, name in ((grad, "a gradient"), (p, "a parameter")):
                if t.device != device:
                    raise RuntimeError(f"AdamW: {name} is on {t.device}, its group on {device}")
            if grad.numel() != p.numel():
                raise RuntimeError(f"AdamW: gradient {list(grad.shape)} of a parameter "
                                   f"{list(p.shape)}")
            w, g = _dense(p.detach(), "parameters"), _dense(grad, "gradients")
            codes = _C.dtype_code(w.dtype), _C.dtype_code(g.dtype)
            state = self.state[p]
            if "step" not in state:
                state = self._new_state(p, bits)
            row = [w.data_ptr(), g.data_ptr()]
            for key, dtype in _STATE[bits].items():
                t = state[key]
                if t.dtype != dtype or t.device != device or t.is_neg() or \
                        not t.is_contiguous() or t.numel() != self._state_size(key, bits, p):
                    raise RuntimeError(f"AdamW: state {key} does not fit a parameter of shape "
                                       f"{list(p.shape)} with {bits}-bit states")
                align = 1 if key.endswith("_scale") else 16 if bits == 32 else 8
                if t.data_ptr() % align:
                    raise RuntimeError(f"AdamW: state {key} must start at a multiple of {align} bytes")
                row.append(t.data_ptr())
            row += [None] * (6 - len(row)) + [p.numel(), index]
            batches.setdefault((*codes, state["step"] + 1), []).append((state, tuple(row), p, w, g))
        return batches, None if device is None else device.index
