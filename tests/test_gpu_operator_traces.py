"""GPU: under a tracer the operators that are handed addresses refuse, since the graph would hold
their empty outputs and not what fills them."""
import pytest
import torch
from torch.fx.experimental.proxy_tensor import make_fx

from haste_amd import ops
from haste_amd.optim_adamw import AdamW, grad_norm

pytestmark = pytest.mark.gpu


def record(how, f, x):
    if how == "jit":
        torch.jit.trace(f, (x,), check_trace=False)
    else:
        make_fx(f)(x)


@pytest.mark.parametrize("how", ["jit", "fx"])
@pytest.mark.parametrize("grad", [False, True])
def test_layer_norm_in_a_trace(dev, how, grad):
    w = torch.ones(64, device=dev, requires_grad=grad)
    x = torch.randn(4, 64, device=dev)
    with pytest.raises(RuntimeError, match="layer_norm: .*traced"):
        record(how, lambda x: ops.layer_norm(x, w), x)


@pytest.mark.parametrize("how", ["jit", "fx"])
@pytest.mark.parametrize("plain", [True, False])
def test_grad_norm_in_a_trace(dev, how, plain):
    x = torch.randn(4, 64, device=dev)
    with pytest.raises(RuntimeError, match="grad_norm: .*traced"):
        record(how, lambda x: grad_norm([x if plain else x.t()], 1.0)[0], x)


@pytest.mark.parametrize("how", ["jit", "fx"])
def test_a_step_in_a_trace(dev, how):
    p = torch.nn.Parameter(torch.ones(64, device=dev))
    opt = AdamW([p])
    p.grad = torch.ones_like(p)
    opt.step()
    kept, seed = p.detach().clone(), opt.param_groups[0]["seed"]

    def f(x):
        opt.step()
        return x + 1
    with pytest.raises(RuntimeError, match="AdamW.step: .*traced"):
        record(how, f, torch.randn(4, device=dev))
    assert torch.equal(p, kept) and opt.state[p]["step"] == 1 and opt.param_groups[0]["seed"] == seed
