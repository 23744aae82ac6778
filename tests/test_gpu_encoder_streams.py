"""GPU: embedding, gated block and label log probabilities on a stream that is still busy when they are called, forward
and backward: work on any other stream would meet inputs that are not there yet."""
import importlib.util

import pytest
import torch

from haste_amd import ops
from test_gpu_encoder_calls import PATH, WEIGHTS, chain, inputs

pytestmark = pytest.mark.gpu


def step(t):
    log_probs, entropy, top = chain(t)
    g = torch.autograd.grad([log_probs, entropy], [t[k] for k in WEIGHTS],
                            [torch.full_like(log_probs, -1.0), torch.full_like(entropy, 0.1)])
    return [log_probs.detach(), entropy.detach(), top, *g]


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32])
def test_on_a_busy_stream(dev, dt):
    t = inputs(dev, dt, N=4000, D=256, H=512, O=5001)
    for k in WEIGHTS:
        t[k].requires_grad_(True)
    want = step(t)
    late = {k: torch.zeros_like(v) for k, v in t.items()}
    for k in WEIGHTS:
        late[k].requires_grad_(True)
    big = torch.randn(8192, 8192, device=dev)
    out = torch.empty_like(big)
    torch.cuda.synchronize()
    stream = torch.cuda.Stream(dev)
    with torch.cuda.stream(stream):
        for _ in range(16):                   # (some 100 ms)
            torch.mm(big, big, out=out)
        with torch.no_grad():
            for k, v in t.items():
                late[k].copy_(v)
        got = step(late)
        assert not stream.query()             # the host was ahead all along
    stream.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a, b)


def test_two_streams_at_once(dev):
    """Steps of other inputs on two streams, queued in turn while both are busy: workspaces are not shared."""
    both = [inputs(dev, torch.bfloat16, seed=s, N=3000, D=136, H=264, O=5001) for s in (1, 2)]
    for t in both:
        for k in WEIGHTS:
            t[k].requires_grad_(True)
    want = [step(t) for t in both]
    big = torch.randn(4096, 4096, device=dev)
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream(dev) for _ in both], [[], []]
    for s in streams:
        with torch.cuda.stream(s):
            for _ in range(4):
                torch.mm(big, big)
    for _ in range(4):
        for t, s, g in zip(both, streams, got):
            with torch.cuda.stream(s):
                g.append(step(t))
    torch.cuda.synchronize()
    for g, w in zip(got, want):
        for one in g:
            assert all(torch.equal(a, b) for a, b in zip(one, w))


def test_gradients_of_the_example(dev):
    """The encoder of examples/train_softmax.py in fp32: gradients of its loss against the same model of torch's
    operations in float64.  Some 10^3 fp32 operations lie between a weight and the loss, in sums of at most 4100 terms that
    are of either sign: 2^-24 times 4100 rounds to 3e-4 of a gradient's largest element."""
    spec = importlib.util.spec_from_file_location("train_softmax", PATH)
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    torch.manual_seed(0)
    g = torch.Generator(device=dev).manual_seed(0)
    encoder = example.Encoder(device=dev, dtype=torch.float32)
    head = torch.randn(example.LABELS, example.WIDTH, generator=g, device=dev) / 16
    ids, right = example.batch(g, dev)
    loss = -ops.label_log_probs(encoder(ids) @ head.t(), right).log_probs.mean()
    names, params = zip(*encoder.named_parameters())
    got = torch.autograd.grad(loss, params)

    d = {k: p.detach().double().requires_grad_(True) for k, p in encoder.named_parameters()}
    rows = d["tokens.weight"][ids]
    stream = torch.where((ids != 0)[..., None], rows, rows.detach()) * example.WIDTH ** 0.5
    norm = lambda x, k: torch.nn.functional.layer_norm(  # noqa: E731
        x, (example.WIDTH,), d[f"norms.{k}.weight"], d[f"norms.{k}.bias"], encoder.norms[k].eps)
    x = norm(stream, 0)
    for k in range(len(encoder.blocks)):
        a = torch.nn.functional.silu(x @ d[f"blocks.{k}.w_gate"].t()) * (x @ d[f"blocks.{k}.w_up"].t())
        stream = stream + a @ d[f"blocks.{k}.w_down"].t()
        x = norm(stream, k + 1)
    want_loss = torch.nn.functional.cross_entropy(x.mean(1) @ head.double().t(), right[:, 0])
    want = torch.autograd.grad(want_loss, [d[k] for k in names])
    assert abs(loss.item() - want_loss.item()) < 3e-4 * abs(want_loss.item())
    for k, a, b in zip(names, got, want):
        assert (a.double() - b).abs().max() <= 3e-4 * b.abs().max(), k
