"""GPU: what reaches the backwards of layer norm, embedding, gated block and label log probabilities without having
passed their forwards: gradients with a tangent, and a tracer that is there for the backward alone."""
import pytest
import torch
import torch.autograd.forward_ad as fwAD
from torch.fx.experimental.proxy_tensor import make_fx

from haste_amd import ops

pytestmark = pytest.mark.gpu


def inputs(dev):
    g = torch.Generator(device=dev).manual_seed(0)
    r = lambda *s: torch.randn(*s, generator=g, device=dev)  # noqa: E731
    return dict(x=r(20, 24).requires_grad_(True), w=r(24), b=r(24), tokens=torch.randint(0, 20, (30,), device=dev),
                labels=torch.randint(0, 24, (20, 2), device=dev), res=r(20, 24), gate=r(40, 24), up=r(40, 24),
                down=r(16, 40))


CALLS = {"layer_norm": lambda t: ops.layer_norm(t["x"], t["w"], t["b"]),
         "layer_norm of a sum": lambda t: ops.layer_norm(t["x"], t["w"], t["b"], residual=t["res"])[0],
         "layer_norm's sum alone": lambda t: ops.layer_norm(t["x"], t["w"], t["b"], residual=t["res"])[1],
         "embedding": lambda t: ops.embedding(t["tokens"], t["x"]),
         "gated_mlp": lambda t: ops.gated_mlp(t["x"], t["gate"], t["up"], t["down"]),
         "label_log_probs": lambda t: ops.label_log_probs(t["x"], t["labels"]).log_probs,
         "label_log_probs' entropy": lambda t: ops.label_log_probs(t["x"], t["labels"]).entropy}


@pytest.mark.parametrize("name", list(CALLS))
def test_a_gradient_with_a_tangent(dev, name):
    """Forward-over-reverse with respect to something behind the operator."""
    t = inputs(dev)
    y = CALLS[name](t)
    with fwAD.dual_level():
        dy = fwAD.make_dual(torch.ones_like(y), torch.ones_like(y))
        with pytest.raises(NotImplementedError, match=name.split()[0].rstrip("'s") + ".*forward-mode"):
            torch.autograd.grad([y], [t["x"]], [dy])


@pytest.mark.parametrize("name", list(CALLS))
def test_a_tracer_over_the_backward_alone(dev, name):
    t = inputs(dev)
    y = CALLS[name](t)
    with pytest.raises(RuntimeError, match=name.split()[0].rstrip("'s") + ".*traced"):
        make_fx(lambda dy: torch.autograd.grad([y], [t["x"]], [dy])[0])(torch.ones_like(y))


@pytest.mark.parametrize("name", list(CALLS))
def test_afterwards_a_plain_backward_runs(dev, name):
    t = inputs(dev)
    y = CALLS[name](t)
    with fwAD.dual_level(), pytest.raises(NotImplementedError):
        torch.autograd.grad([y], [t["x"]], [fwAD.make_dual(torch.ones_like(y), torch.ones_like(y))],
                            retain_graph=True)
    got, = torch.autograd.grad([y], [t["x"]], [torch.ones_like(y)])
    assert got.isfinite().all() and got.shape == t["x"].shape
