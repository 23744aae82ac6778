"""GPU: forms of inputs to embedding and label log probabilities beside those of the tests of their numbers."""
import pytest
import torch

from haste_amd import ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dt", [torch.int64, torch.int32])
def test_lazily_negated_tokens_and_labels(dev, dt):
    """Whole numbers whose sign is pending, contiguous or not."""
    g = torch.Generator(device=dev).manual_seed(0)
    table = torch.randn(50, 24, generator=g, device=dev)
    z = torch.randn(30, 60, generator=g, device=dev)
    for step in (1, 2):
        tokens = torch.randint(0, 50, (30 * step,), generator=g, device=dev).to(dt)
        labels = torch.randint(-1, 60, (30, 3 * step), generator=g, device=dev).to(dt)
        late = torch._neg_view(-tokens)[::step], torch._neg_view(-labels)[:, ::step]
        assert all(t.is_neg() for t in late)
        tokens, labels = tokens[::step], labels[:, ::step]
        grads = []
        for t, l in ((tokens, labels), late):
            w, x = table.clone().requires_grad_(True), z.clone().requires_grad_(True)
            y, lp = ops.embedding(t, w, padding_idx=3), ops.label_log_probs(x, l).log_probs
            grads.append([y.detach(), lp.detach(), torch.autograd.grad([y], [w], [torch.ones_like(y)])[0],
                          torch.autograd.grad([lp], [x], [torch.ones_like(lp)])[0]])
        for a, b in zip(*grads):
            assert torch.equal(a, b)


@pytest.mark.parametrize("N", [262143, 262144, 262145, 400000])
def test_one_token_in_more_than_1024_windows(dev, N):
    """Windows are 256 places, and longer from 262,144 tokens on.  Whole numbers: every partial sum is exact."""
    g = torch.Generator(device=dev).manual_seed(N)
    w = torch.zeros(5, 24, device=dev, requires_grad=True)
    tokens = torch.where(torch.rand(N, generator=g, device=dev) < 0.97, 2, 4)
    dy = torch.randint(-3, 4, (N, 24), generator=g, device=dev).float()
    dw, = torch.autograd.grad([ops.embedding(tokens, w)], [w], [dy])
    for v in range(5):
        assert torch.equal(dw[v], dy[tokens == v].sum(0)), v
