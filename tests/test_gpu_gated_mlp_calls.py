"""GPU: calls of the gated block that the tests of its numbers do not make."""
import pytest
import torch

from haste_amd import ops

pytestmark = pytest.mark.gpu
TYPES = [torch.bfloat16, torch.float16, torch.float32]


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("sizes", [(24, 40, 16), (23, 41, 15), (64, 1003, 301)])
def test_no_rows(dev, dt, sizes):
    """Empty outputs and zero gradients of the weights, and no copy or split of weights that no product uses."""
    D, H, O = sizes
    x = torch.zeros(0, D, device=dev, dtype=dt, requires_grad=True)
    w = [torch.full(s, float("nan"), device=dev, dtype=dt, requires_grad=True) for s in ((H, D), (H, D), (O, H))]
    for _ in range(2):
        y = ops.gated_mlp(x, *w)
        got = torch.autograd.grad([y], [x, *w], [torch.zeros_like(y)])
        assert y.shape == (0, O) and [g.shape for g in got] == [t.shape for t in (x, *w)]
        assert not any(g.any() for g in got)     # (NaN counts as true)
