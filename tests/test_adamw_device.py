"""CPU: the device that the launches of AdamW and of the gradients' norm run under."""
from contextlib import contextmanager

import pytest
import torch

from haste_amd import _lib, optim_adamw
from haste_amd.optim_adamw import AdamW


class Guard:
    """Stands in for torch.cuda.device and the library: what was current at each launch."""

    def __init__(self, monkeypatch):
        self.current, self.launches = 0, []

        @contextmanager
        def device(d):
            before, self.current = self.current, torch.device(d).index if isinstance(d, (str, torch.device)) else d
            yield
            self.current = before

        class Host:
            grad_norm = staticmethod(lambda *a: None)
            adamw_step = staticmethod(lambda *a: None)

        class Lib:
            haste_grad_norm_workspace_size = staticmethod(lambda n: 64)
        monkeypatch.setattr(torch.cuda, "device", device)
        monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda d: 0)
        monkeypatch.setattr(_lib, "host", lambda: Host)
        monkeypatch.setattr(_lib, "lib", lambda: Lib)
        monkeypatch.setattr(_lib, "call", lambda name, *a: self.launches.append((name, self.current)))


class On(torch.Tensor):
    """A tensor that says it is on cuda:1."""
    device = property(lambda self: torch.device("cuda", 1))
    is_cuda = property(lambda self: True)

    def get_device(self):
        return 1


@pytest.mark.parametrize("bits", [32, 8])
def test_a_step_of_new_parameters_runs_under_their_device(monkeypatch, bits):
    guard = Guard(monkeypatch)
    zeros, full = torch.zeros, torch.full
    monkeypatch.setattr(torch, "zeros", lambda *a, device=None, **k: zeros(*a, **k).as_subclass(On))
    monkeypatch.setattr(torch, "full", lambda *a, device=None, **k: full(*a, **k).as_subclass(On))
    p = torch.nn.Parameter(zeros(300).as_subclass(On))
    opt = AdamW([p], state_bits=bits)
    p.grad = zeros(300).as_subclass(On)
    opt.step()
    assert guard.launches == [("haste_adamw_step", 1)] and guard.current == 0


def test_a_norm_through_copies_runs_under_its_tensors_device(monkeypatch):
    guard = Guard(monkeypatch)
    empty = torch.empty
    monkeypatch.setattr(torch, "empty", lambda *a, device=None, **k: empty(*a, **k).as_subclass(On))
    optim_adamw.grad_norm([torch.ones(6, 4).as_subclass(On)])
    assert guard.launches == [("haste_grad_norm", 1)] and guard.current == 0
