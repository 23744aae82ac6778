"""GPU: embedding lookup and its table's gradient against float64, over widths, types, token counts
and the ways in which tokens repeat.

Tolerances: the lookup is one fp32 product, rounded once, so its bits are known.  A row of the gradient is
a sum of n terms in some order, off by at most n u of their absolute sum (u = 2^-24), a product
with the scale (u) and one rounding to the table's type (half a step)."""
import pytest
import torch

from haste_amd import ops
from haste_amd.embedding import Embedding

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
UD = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 0.0, torch.bfloat16: 0.0, torch.float16: 2.0 ** -25}
TYPES = list(UD)


def gradient(tokens, dy, V, scale, padding=None):
    """float64 gradient and its error bound."""
    t, d = tokens.reshape(-1).long(), dy.reshape(-1, dy.shape[-1])
    live = (t >= 0) & (t < V)
    if padding is not None:
        live &= t != padding % V
    t, d = t[live], d[live].double()
    z = lambda: torch.zeros(V, dy.shape[-1], dtype=torch.float64, device=dy.device)  # noqa: E731
    n = torch.bincount(t, minlength=V).double()[:, None]
    dw = z().index_add_(0, t, d) * scale
    terms = z().index_add_(0, t, d.abs()) * abs(scale)
    return dw, UD[dy.dtype] * dw.abs() + 1.01 * (n + 1) * U * terms + TINY[dy.dtype]


def check(tokens, w, dy, scale=1.0, padding=None):
    V = w.shape[0]
    w = w.detach().requires_grad_(True)
    y = ops.embedding(tokens, w, scale=scale, padding_idx=padding)
    t = tokens.long()
    inside = ((t >= 0) & (t < V))[..., None]
    want = torch.where(inside, w.detach()[t.clamp(0, V - 1)].float() * scale,
                       torch.zeros((), device=w.device)).to(w.dtype)
    assert y.shape == want.shape and torch.equal(y, want)
    dw, = torch.autograd.grad([y], [w], [dy])
    want, tol = gradient(tokens, dy, V, scale, padding)
    assert dw.dtype == w.dtype and dw.shape == w.shape
    off = (dw.double() - want).abs() - tol
    assert not (off > 0).any(), float(off.max())
    none = torch.ones(V, dtype=torch.bool, device=w.device)
    seen = t[inside[..., 0]]
    none[seen if padding is None else seen[seen != padding % V]] = False
    assert not dw[none].any()
    return y.detach(), dw


def data(N, V, D, dt, dev, seed=0):
    g = torch.Generator(device=dev).manual_seed(seed)
    tokens = torch.randint(0, V, (N,), generator=g, device=dev)
    r = lambda *s: torch.randn(*s, generator=g, device=dev)  # noqa: E731
    return tokens, r(V, D).to(dt), r(N, D).to(dt)


@pytest.mark.parametrize("D", [1, 2, 3, 4, 7, 8, 9, 15, 16, 63, 64, 65, 100, 301, 512, 513, 768, 1000,
                               2048, 4100])
@pytest.mark.parametrize("dt", TYPES)
def test_widths(dev, D, dt):
    check(*data(257, 101, D, dt, dev, seed=D), scale=0.7)


@pytest.mark.parametrize("N", [0, 1, 2, 63, 64, 65, 127, 128, 129, 2047, 2048, 2049, 10000])
@pytest.mark.parametrize("V", [1, 2, 255, 256, 1023, 1024, 1025, 70001])
def test_counts(dev, N, V):
    check(*data(N, V, 40, torch.bfloat16, dev, seed=N + V), padding=0 if N % 2 else None)


@pytest.mark.parametrize("N,V", [(65536, 32000), (65537, 32000), (100000, 70001), (300000, 513)])
def test_tokens_by_their_rank(dev, N, V):
    """The sort's forms past 64 tiles, and tokens of every frequency."""
    tokens, w, dy = data(N, V, 24, torch.float32, dev, seed=N)
    tokens = torch.exp(torch.rand(N, device=dev).double() * torch.tensor(V, device=dev).log()).long() - 1
    check(tokens.clamp_(0, V - 1), w, dy)


@pytest.mark.parametrize("D", [4, 8, 24, 100])
def test_narrow_rows_of_frequent_tokens(dev, D):
    """Rows of few threads: many tokens to a workgroup, summed by a group or together."""
    g = torch.Generator(device=dev).manual_seed(D)
    counts = torch.randint(0, 400, (700,), generator=g, device=dev)
    tokens = torch.arange(700, device=dev).repeat_interleave(counts)
    tokens = tokens[torch.randperm(len(tokens), generator=g, device=dev)]
    for dt in (torch.bfloat16, torch.float32):
        check(tokens, torch.randn(700, D, generator=g, device=dev).to(dt),
              torch.randn(len(tokens), D, generator=g, device=dev).to(dt))


@pytest.mark.parametrize("times", [1, 15, 16, 17, 63, 64, 65, 66, 127, 128, 129, 191, 192, 193, 255, 256, 257,
                                   511, 512, 513, 1000, 5000])
def test_a_token_met_many_times(dev, times):
    """Parts of a frequent token that begin and end anywhere in a window, next to others."""
    g = torch.Generator(device=dev).manual_seed(times)
    counts = torch.tensor([3, times, 64, 65, times, 1, 130, 0, times + 1], device=dev)
    tokens = torch.arange(9, device=dev).repeat_interleave(counts)
    tokens = tokens[torch.randperm(len(tokens), generator=g, device=dev)]
    w = torch.randn(9, 100, generator=g, device=dev)
    check(tokens, w, torch.randn(len(tokens), 100, generator=g, device=dev), scale=-2.0)


def test_one_token_200000_times(dev):
    """More places than 1024 windows of 192.  Whole numbers: every partial sum is exact."""
    N = 200000
    w = torch.zeros(3, 24, device=dev, requires_grad=True)
    dy = torch.randint(-3, 4, (N, 24), device=dev).float()
    y = ops.embedding(torch.ones(N, dtype=torch.int64, device=dev), w)
    dw, = torch.autograd.grad([y], [w], [dy])
    assert torch.equal(dw[1], dy.sum(0)) and not dw[0].any() and not dw[2].any()


def test_order_of_the_sum_is_fixed(dev):
    tokens, w, dy = data(20000, 50, 64, torch.float32, dev)
    first = check(tokens, w, dy)[1]
    for _ in range(5):
        assert torch.equal(check(tokens, w, dy)[1], first)


@pytest.mark.parametrize("dt", TYPES)
def test_tokens_outside_and_padding(dev, dt):
    tokens, w, dy = data(3000, 77, 96, dt, dev)
    tokens[::7] = -1
    tokens[3::7] = 77
    tokens[5::97] = 2 ** 40
    tokens[6::97] = -2 ** 40
    dy[::7] = float("nan")   # (what nobody asked for is not read)
    dy[3::7] = float("inf")
    dy[5::97], dy[6::97] = float("nan"), float("nan")
    dy[tokens == 9] = float("nan")
    check(tokens, w, torch.where(((tokens >= 0) & (tokens < 77) & (tokens != 9))[:, None], dy,
                                 torch.zeros((), device=dev, dtype=dt)), padding=9)
    w = w.requires_grad_(True)
    for padding in (9, 9 - 77):
        y = ops.embedding(tokens, w, padding_idx=padding)
        dw, = torch.autograd.grad([y], [w], [dy])
        assert dw.isfinite().all() and not dw[9].any()


def test_what_is_not_finite_stays_in_its_token(dev):
    tokens, w, dy = data(500, 20, 16, torch.float32, dev)
    tokens[100] = 3
    dy[100, 5] = float("inf")
    w = w.requires_grad_(True)
    dw, = torch.autograd.grad([ops.embedding(tokens, w)], [w], [dy])
    bad = ~dw.isfinite()
    assert bad[3, 5] and int(bad.sum()) == 1


@pytest.mark.parametrize("kind", ["int32", "strided", "shape", "transposed_table", "pitched_table",
                                  "one_row_gradient", "strided_gradient", "pitched_gradient"])
def test_layouts(dev, kind):
    tokens, w, dy = data(600, 90, 56, torch.bfloat16, dev)
    if kind == "int32":
        tokens = tokens.int()
    elif kind == "strided":
        tokens = tokens.repeat_interleave(2)[::2]
    elif kind == "shape":
        tokens, dy = tokens.view(20, 5, 6), dy.view(20, 5, 6, 56)
    elif kind == "transposed_table":
        w = w.t().contiguous().t()
    elif kind == "pitched_table":
        w = torch.cat([w, w], 1)[:, 3:59]
    elif kind == "one_row_gradient":
        dy = dy[:1].expand(600, 56)
    elif kind == "strided_gradient":
        dy = dy.t().contiguous().t()
    elif kind == "pitched_gradient":
        dy = torch.cat([dy, dy], 1)[:, 5:61]
    check(tokens, w, dy, scale=3.0)


def test_offsets_past_32_bits(dev):
    """A table of 2.2e9 elements: rows at its end, and its gradient."""
    V, D = 1_100_000, 2000
    torch.cuda.empty_cache()
    if torch.cuda.mem_get_info(dev)[0] < 24 << 30:
        pytest.skip("needs 24 GiB")
    w = torch.zeros(V, D, dtype=torch.bfloat16, device=dev)
    tokens = torch.tensor([V - 1, 0, V - 1, V - 2, 1_073_742], device=dev)
    w[tokens] = torch.randn(5, D, device=dev).to(w.dtype)
    w.requires_grad_(True)
    y = ops.embedding(tokens, w)
    assert torch.equal(y, w.detach()[tokens])
    dy = torch.randint(-2, 3, (5, D), device=dev).to(w.dtype)
    dw, = torch.autograd.grad([y], [w], [dy])
    assert torch.equal(dw[V - 1], dy[0] + dy[2]) and torch.equal(dw[V - 2], dy[3])
    assert torch.equal(dw[0], dy[1]) and torch.equal(dw[1_073_742], dy[4])
    dw[tokens] = 0
    assert not any(part.any() for part in dw.split(100_000))


def test_module(dev):
    e = Embedding(50, 24, padding_idx=0, scale=24 ** 0.5, device=dev, dtype=torch.bfloat16)
    plain = torch.nn.Embedding(50, 24, padding_idx=0, device=dev, dtype=torch.bfloat16)
    plain.load_state_dict(e.state_dict())
    tokens = torch.randint(0, 50, (4, 9), device=dev)
    y = e(tokens)
    assert torch.equal(y, (plain(tokens).float() * 24 ** 0.5).to(torch.bfloat16))
    y.float().square().sum().backward()
    assert e.weight.grad.shape == (50, 24) and not e.weight.grad[0].any()
    with pytest.raises(ValueError, match="max_norm"):
        Embedding(50, 24, max_norm=1.0)
    with torch.no_grad():
        assert not e(tokens).requires_grad


def test_gradient_against_differences(dev):
    tokens, w, dy = data(30, 7, 5, torch.float32, dev)
    f = lambda w: (ops.embedding(tokens, w, scale=1.5).double() * dy.double()).sum()  # noqa: E731
    w.requires_grad_(True)
    dw, = torch.autograd.grad([ops.embedding(tokens, w, scale=1.5)], [w], [dy])
    for i in (0, 3, 6):
        step = torch.zeros_like(w)
        step[i, 2] = 0.5
        # (linear: the difference is the gradient, but for the outputs' roundings)
        got = (f(w.detach() + step) - f(w.detach() - step)).item()
        bound = (dy.double().abs().sum() * w.detach().abs().max() * 8 * U).item()
        assert abs(got - dw[i, 2].item()) <= bound


def test_refusals(dev):
    tokens, w, dy = data(8, 5, 16, torch.float32, dev)
    for bad, match in ((tokens.float(), "int64 or int32"), (tokens.cpu(), "HIP device")):
        with pytest.raises(RuntimeError, match=match):
            ops.embedding(bad, w)
    with pytest.raises(RuntimeError, match="dtype"):
        ops.embedding(tokens, w.double())
    with pytest.raises(RuntimeError, match=r"\[V, D\]"):
        ops.embedding(tokens, w[0])
    for p in (5, -6):
        with pytest.raises(RuntimeError, match="padding_idx"):
            ops.embedding(tokens, w, padding_idx=p)
    y = ops.embedding(tokens, w.requires_grad_(True))
    g, = torch.autograd.grad([y], [w], [dy.requires_grad_(True)], create_graph=True)
    with pytest.raises(RuntimeError, match="cannot be differentiated"):
        g.sum().backward()


def test_replays_of_a_graph(dev):
    tokens, w, dy = data(5000, 300, 128, torch.bfloat16, dev)
    w.requires_grad_(True)
    stream = torch.cuda.Stream(dev)
    stream.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(stream):
        for _ in range(2):
            torch.autograd.grad([ops.embedding(tokens, w)], [w], [dy])
    torch.cuda.current_stream(dev).wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = ops.embedding(tokens, w, padding_idx=1)
        dw, = torch.autograd.grad([y], [w], [dy])
    for seed in range(4):
        fresh = data(5000, 300, 128, torch.bfloat16, dev, seed=seed + 10)
        with torch.no_grad():
            tokens.copy_(fresh[0])
            w.copy_(fresh[1])
            dy.copy_(fresh[2])
        graph.replay()
        torch.cuda.synchronize()
        a, b = y.clone(), dw.clone()
        want = check(tokens, w, dy, padding=1)
        torch.cuda.synchronize()
        assert torch.equal(a, want[0]) and torch.equal(b, want[1])
