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


def positive(N, D, H, O, dt, dev):
    """Everything above zero: sums of infinities of one sign are infinite."""
    g = torch.Generator(device=dev).manual_seed(N + H)
    r = lambda *s: (torch.rand(*s, generator=g, device=dev) * 0.5 + 0.25).to(dt)  # noqa: E731
    return dict(x=r(N, D), wg=r(H, D), wu=r(H, D), wd=r(O, H), dy=r(N, O))


@pytest.mark.parametrize("N", [40, 70, 300])
@pytest.mark.parametrize("H", [3, 8, 13, 1003])
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("name", ["silu", "gelu", "gelu_tanh"])
def test_an_infinite_input_among_positive_ones(dev, N, H, dt, name):
    """Both projections, h and y of its row are +infinity, whatever the hidden width."""
    d = positive(N, 8, H, 5, dt, dev)
    clean = ops.gated_mlp(d["x"], d["wg"], d["wu"], d["wd"], activation=name)
    d["x"][7, 2] = float("inf")
    y = ops.gated_mlp(d["x"], d["wg"], d["wu"], d["wd"], activation=name)
    assert (y[7] == float("inf")).all(), y[7]
    keep = torch.arange(N, device=dev) != 7
    assert torch.equal(y[keep], clean[keep])


@pytest.mark.parametrize("N", [40, 300])
@pytest.mark.parametrize("H", [3, 8, 13, 1003])
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
def test_an_infinite_gradient_among_positive_ones(dev, N, H, dt):
    """With gates above zero silu rises: dh, dg, du and dx of the row are +infinity."""
    d = positive(N, 8, H, 5, dt, dev)
    x = d["x"].requires_grad_(True)
    y = ops.gated_mlp(x, d["wg"], d["wu"], d["wd"])
    d["dy"][7, 2] = float("inf")
    dx, = torch.autograd.grad([y], [x], [d["dy"]])
    assert (dx[7] == float("inf")).all(), dx[7]
    assert dx[torch.arange(N, device=dev) != 7].isfinite().all()


def test_gradients_that_the_engine_does_not_want(dev):
    """autograd.grad of some inputs takes no memory for the others' gradients, and gives the same bits."""
    N, D, H, O = 80, 1024, 4096, 1024
    g = torch.Generator(device=dev).manual_seed(0)
    r = lambda *s: torch.randn(*s, generator=g, device=dev).to(torch.bfloat16)  # noqa: E731
    leaves = [t.requires_grad_(True) for t in (r(N, D), r(H, D), r(H, D), r(O, H))]
    dy = r(N, O)
    want = torch.autograd.grad([ops.gated_mlp(*leaves)], leaves, [dy])
    weight = H * D * 2                                     # bytes of any one weight's gradient
    for some in ([0], [3], [0, 3]):
        y = ops.gated_mlp(*leaves)
        torch.cuda.synchronize()
        torch.cuda.reset_peak_memory_stats(dev)
        before = torch.cuda.memory_allocated(dev)
        got = torch.autograd.grad([y], [leaves[k] for k in some], [dy])
        torch.cuda.synchronize()
        # what is returned, and a workspace: dg, du and the parts of the products, all under two weights' size
        room = (weight if 3 in some else 0) + 2 * weight
        assert torch.cuda.max_memory_allocated(dev) - before < room, some
        assert all(torch.equal(a, want[k]) for a, k in zip(got, some))


def test_copies_of_more_than_a_launch(dev):
    """Two projections of 2^34 elements each, whose rows do not start on 16 bytes: their copies take 2^32 threads and
    more.  Every weight is a power of two of its row and column, so that both projections are known exactly."""
    N, H, D = 65, 1 << 17, (1 << 17) + 1
    torch.cuda.empty_cache()
    if torch.cuda.mem_get_info(dev)[0] < 170 << 30:
        pytest.skip("needs 170 GiB")
    # x is 1 in three columns; a weight is 2^-(row mod 8) there (the up projection: 2^-(row mod 4)), else rubbish
    # that a zero of x takes out
    cols = [0, D // 2, D - 1]
    x = torch.zeros(N, D, device=dev, dtype=torch.bfloat16)
    x[:, cols] = 1
    rows = torch.arange(H, device=dev)
    w = []
    for mod in (8, 4):
        t = torch.full((H, D), 3.0, device=dev, dtype=torch.bfloat16)
        for c in cols:
            t[:, c] = torch.exp2(-(rows % mod).float())
        w.append(t)
    down = torch.zeros(8, H, device=dev, dtype=torch.bfloat16)
    pick = torch.tensor([0, 1, 7, 4096, 70001, H // 2 + 5, H - 2, H - 1], device=dev)
    down[torch.arange(8, device=dev), pick] = 1
    y = ops.gated_mlp(x, *w, down)
    del w, t
    g, u = (3 * torch.exp2(-(pick % mod).double()) for mod in (8, 4))
    h = g * torch.sigmoid(g) * u
    # (act within 2^-20 of itself, h rounded to bf16, then exact)
    assert ((y.double() - h).abs() <= h * (2.0 ** -8 + 2.0 ** -19)).all()
    torch.cuda.empty_cache()
