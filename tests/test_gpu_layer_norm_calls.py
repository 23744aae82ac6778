"""GPU: calls of layer norm that could end in a wrong answer without an error."""
import pytest
import torch
import torch.autograd.forward_ad as fwAD

from haste_amd import ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("which", ["x", "weight", "bias", "residual"])
@pytest.mark.parametrize("grad", [False, True])
def test_forward_mode_is_refused(dev, which, grad):
    """A tangent that the kernels would drop, with and without a backward to record."""
    t = {k: torch.randn(s, device=dev) for k, s in
         dict(x=(4, 64), weight=(64,), bias=(64,), residual=(4, 64)).items()}
    if grad:
        t["x" if which != "x" else "weight"].requires_grad_(True)
    with fwAD.dual_level():
        t[which] = fwAD.make_dual(t[which], torch.ones_like(t[which]))
        with pytest.raises(NotImplementedError, match="forward-mode"):
            ops.layer_norm(t["x"], t["weight"], t["bias"], residual=t["residual"])
