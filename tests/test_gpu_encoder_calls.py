"""GPU: embedding, gated block and label log probabilities as they are called together, and calls that
could end in a wrong answer without an error: tracers, tangents, other streams, inputs changed before
the backward, two graphs side by side, recomputation."""
import importlib.util
import os

import pytest
import torch
import torch.autograd.forward_ad as fwAD
from torch.fx.experimental.proxy_tensor import make_fx
from torch.utils.checkpoint import checkpoint

from haste_amd import ops

pytestmark = pytest.mark.gpu
PATH = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples",
                    "train_softmax.py")


def inputs(dev, dt=torch.float32, seed=0, N=90, V=50, D=24, H=40, O=130):
    g = torch.Generator(device=dev).manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, device=dev).to(dt)  # noqa: E731
    return dict(tokens=torch.randint(0, V, (N,), generator=g, device=dev), table=r(V, D),
                w_gate=r(H, D) / D ** 0.5, w_up=r(H, D) / D ** 0.5, w_down=r(O, H) / H ** 0.5,
                labels=torch.randint(-1, O, (N, 2), generator=g, device=dev))


WEIGHTS = ("table", "w_gate", "w_up", "w_down")


def chain(t):
    """tokens -> rows -> gated block -> log probabilities: (log_probs, entropy, top_labels)."""
    x = ops.embedding(t["tokens"], t["table"], scale=2.0, padding_idx=1)
    z = ops.gated_mlp(x, t["w_gate"], t["w_up"], t["w_down"], activation="gelu")
    r = ops.label_log_probs(z, t["labels"], top=3)
    return r.log_probs, r.entropy, r.top_labels


def plain(t):
    """The same in float64."""
    d = {k: t[k].detach().double().requires_grad_(True) for k in WEIGHTS}
    live = (t["tokens"] != 1)[:, None]
    rows = d["table"][t["tokens"]]
    x = 2.0 * torch.where(live, rows, rows.detach())
    z = (torch.nn.functional.gelu(x @ d["w_gate"].t()) * (x @ d["w_up"].t())) @ d["w_down"].t()
    lp = torch.log_softmax(z, 1)
    given = t["labels"] >= 0
    out = torch.where(given, lp.gather(1, t["labels"].clamp(min=0)), 0.0)
    return d, out, -(lp.exp() * lp).sum(1), z


def test_together(dev):
    """Forward and gradients of the chain against float64.  Its fp32 products have 24 to 130 terms and its
    values are of order 1: 2^-24 times some 200 rounds to 2e-5 of the largest."""
    t = inputs(dev)
    for k in WEIGHTS:
        t[k].requires_grad_(True)
    log_probs, entropy, top = chain(t)
    d, lp, ent, z = plain(t)
    assert (log_probs.double() - lp).abs().max() < 2e-5 * lp.abs().max()
    assert (entropy.double() - ent).abs().max() < 2e-5 * ent.abs().max()
    assert torch.equal(top, z.sort(dim=1, descending=True, stable=True).indices[:, :3])
    loss, want = -log_probs.mean() + 0.1 * entropy.mean(), -lp.mean() + 0.1 * ent.mean()
    got = torch.autograd.grad(loss, [t[k] for k in WEIGHTS])
    for a, b in zip(got, torch.autograd.grad(want, [d[k] for k in WEIGHTS])):
        assert (a.double() - b).abs().max() < 1e-4 * b.abs().max()
    assert not got[0][1].any()


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16, torch.float32])
def test_a_captured_step_beside_eager_ones(dev, dt):
    """A training step in a graph, replayed between eager steps of other leaves: every replay gives the
    eager step's bits."""
    t = inputs(dev, dt, N=300, D=64, H=96, O=1000)

    def step(t):
        log_probs, entropy, top = chain(t)
        g = torch.autograd.grad([log_probs, entropy], [t[k] for k in WEIGHTS],
                                [torch.full_like(log_probs, -1.0), torch.full_like(entropy, 0.1)])
        return [log_probs.detach(), entropy.detach(), top, *g]
    fixed = {k: v.clone().requires_grad_(k in WEIGHTS) for k, v in t.items()}
    stream = torch.cuda.Stream(dev)
    stream.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(stream):
        step(fixed)
    torch.cuda.current_stream(dev).wait_stream(stream)
    graphs, outs = [], []
    for _ in range(2):    # two graphs that share a pool of memory
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, pool=graphs[0].pool() if graphs else None):
            outs.append(step(fixed))
        graphs.append(graph)
    for seed in range(4):
        fresh = inputs(dev, dt, seed=seed + 1, N=300, D=64, H=96, O=1000)
        with torch.no_grad():
            for k, v in fresh.items():
                fixed[k].copy_(v)
        graphs[seed % 2].replay()
        torch.cuda.synchronize()
        kept = [x.clone() for x in outs[seed % 2]]
        eager = {k: v.requires_grad_(k in WEIGHTS) for k, v in fresh.items()}
        for a, b in zip(kept, step(eager)):
            assert torch.equal(a, b)


def test_on_a_stream_of_its_own(dev):
    t = inputs(dev, torch.bfloat16, N=4000, D=256, H=512, O=5000)
    want = [x.detach() for x in chain(t)]
    torch.cuda.synchronize()
    stream = torch.cuda.Stream(dev)
    with torch.cuda.stream(stream):
        late = {k: v.clone() for k, v in t.items()}
        for _ in range(3):
            got = [x.detach() for x in chain(late)]
    stream.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a, b)


def test_recomputation(dev):
    """Under torch.utils.checkpoint the gradients are the same bits."""
    a, b = inputs(dev, torch.bfloat16), inputs(dev, torch.bfloat16)
    grads = []
    for t, again in ((a, False), (b, True)):
        for k in WEIGHTS:
            t[k].requires_grad_(True)
        f = lambda *w: chain(dict(t, **dict(zip(WEIGHTS, w))))[0]  # noqa: E731
        w = [t[k] for k in WEIGHTS]
        out = checkpoint(f, *w, use_reentrant=False) if again else f(*w)
        grads.append(torch.autograd.grad([out], w, [torch.ones_like(out)]))
    assert all(torch.equal(x, y) for x, y in zip(*grads))


def test_inputs_changed_before_the_backward_are_noticed(dev):
    for k in ("tokens", "w_gate", "w_up", "w_down"):
        t = inputs(dev)
        leaves = [t[w].requires_grad_(True) for w in WEIGHTS]
        out = chain(t)[0]
        with torch.no_grad():
            t[k].add_(0)
        with pytest.raises(RuntimeError, match="modified by an inplace"):
            torch.autograd.grad([out.sum()], leaves)


CALLS = {"embedding": lambda t: ops.embedding(t["tokens"], t["table"]),
         "gated_mlp": lambda t: ops.gated_mlp(t["table"], t["w_gate"], t["w_up"], t["w_down"]),
         "label_log_probs": lambda t: ops.label_log_probs(t["table"], top=2).entropy}


@pytest.mark.parametrize("name", list(CALLS))
@pytest.mark.parametrize("grad", [False, True])
@pytest.mark.parametrize("how", ["jit", "fx"])
def test_in_a_trace(dev, name, grad, how):
    t = inputs(dev)
    t["table"].requires_grad_(grad)
    f = lambda x: CALLS[name](dict(t, table=x))  # noqa: E731
    with pytest.raises(RuntimeError, match=name + ": .*traced"):
        if how == "jit":
            torch.jit.trace(f, (t["table"],), check_trace=False)
        else:
            make_fx(f)(t["table"])


@pytest.mark.parametrize("name", list(CALLS))
@pytest.mark.parametrize("grad", [False, True])
def test_forward_mode_is_refused(dev, name, grad):
    t = inputs(dev)
    if grad:
        t["w_up"].requires_grad_(True)
    with fwAD.dual_level():
        x = fwAD.make_dual(t["table"], torch.ones_like(t["table"]))
        with pytest.raises(NotImplementedError, match="forward-mode"):
            CALLS[name](dict(t, table=x))


def test_lazily_negated_inputs(dev):
    """A tensor whose sign is pending: what the address holds is not what it stands for."""
    t = inputs(dev)
    c = torch.complex(torch.zeros_like(t["table"]), t["table"])
    x = c.conj().imag            # -table, by its sign bit
    assert x.is_neg()
    assert torch.equal(ops.embedding(t["tokens"], x), ops.embedding(t["tokens"], -t["table"]))
    assert torch.equal(ops.gated_mlp(x, t["w_gate"], t["w_up"], t["w_down"]),
                       ops.gated_mlp(-t["table"], t["w_gate"], t["w_up"], t["w_down"]))
    assert torch.equal(ops.label_log_probs(x, top=2).top_labels,
                       ops.label_log_probs(-t["table"], top=2).top_labels)


def test_example_runs_and_has_gradients(dev):
    spec = importlib.util.spec_from_file_location("train_softmax", PATH)
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    model, losses, share = example.train(steps=12)
    assert len(losses) == 3 and all(x == x and x < 100 for x in losses) and 0 <= share <= 1
    for name, p in model.named_parameters():
        assert p.grad is not None and p.grad.isfinite().all() and p.grad.any(), name
    assert not model.encoder.tokens.weight.grad[0].any()    # (the padding's row)
