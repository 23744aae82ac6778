"""GPU: layer norm forward and backward against float64, over widths, types, strides and
broadcasts, and where rows are constant, far from zero or not finite.

Tolerances: u = 2^-24 (fp32), u_d the half-spacing of the output's type.  A row's sums have at
most d = 8 + D / 64 additions after one another, so mean and rstd are off by at most d u of
their terms' size, n = (h - mean) rstd by 2 d u (max|h| rstd + |n|), and every output by what
that and its own few operations give; sums over rows are bounded in any order."""
import pytest
import torch

from haste_amd import ops
from haste_amd.layer_norm import LayerNorm

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
UD = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 0.0, torch.bfloat16: 0.0, torch.float16: 2.0 ** -24}  # fp16 subnormals
TYPES = [(torch.bfloat16, torch.bfloat16), (torch.bfloat16, torch.float32),
         (torch.float16, torch.float16), (torch.float16, torch.float32),
         (torch.float32, torch.float32)]
EPS = 1e-5


def data(N, D, dt, wt, dev, residual=False, pitch=0, seed=0, mean=0.3):
    g = torch.Generator(device=dev).manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, device=dev)  # noqa: E731
    x = (r(N, D + pitch) + mean).to(dt)[:, :D]
    return dict(x=x, res=r(N, D).to(dt) if residual else None, w=(1 + 0.2 * r(D)).to(wt),
                b=(0.2 * r(D)).to(wt), dy=r(N, D).to(dt), dh=r(N, D).to(dt) if residual else None)


def reference(x, w, b, dy=None, dh=None, res=None, eps=EPS):
    """float64 outputs and their error bounds."""
    dt, D = x.dtype, x.shape[1]
    N = x.shape[0]
    h = x if res is None else (x.float() + res.float()).to(dt)
    hd, wd = h.double(), w.double()
    bd = torch.zeros_like(wd) if b is None else b.double()
    mean = hd.mean(1, keepdim=True)
    rstd = 1 / ((hd - mean).square().mean(1, keepdim=True) + eps).sqrt()
    n = (hd - mean) * rstd
    d = 8 + D / 64
    en = 2 * d * U * (hd.abs().amax(1, keepdim=True) * rstd + n.abs())
    y = n * wd + bd
    out = {"y": y, "h": hd}
    tol = {"y": UD[dt] * y.abs() + (en + 2 * U * n.abs()) * wd.abs() + U * bd.abs() + TINY[dt],
           "h": torch.zeros_like(hd)}
    if dy is not None:
        g = dy.double()
        a = g * wd
        c1, c2 = a.mean(1, keepdim=True), (a * n).mean(1, keepdim=True)
        dx = rstd * (a - c1 - n * c2)
        m1, m2 = a.abs().mean(1, keepdim=True), (a * n).abs().mean(1, keepdim=True)
        ec2 = (a.abs() * en).mean(1, keepdim=True) + d * U * m2
        e = rstd * (4 * U * a.abs() + d * U * m1 + en * c2.abs() + n.abs() * ec2
                    + 4 * U * (n * c2).abs() + d * U * (a - c1 - n * c2).abs())
        if dh is not None:
            dx = dx + dh.double()
            e = e + U * dh.double().abs()
        out |= {"dx": dx, "dw": (g * n).sum(0), "db": g.sum(0)}
        uw = UD[w.dtype]
        tol |= {"dx": UD[dt] * dx.abs() + 2 * e + TINY[dt],
                "dw": uw * out["dw"].abs() + 2 * (g.abs() * en).sum(0)
                + (N + 2) * U * (g * n).abs().sum(0) + TINY[w.dtype],
                "db": uw * out["db"].abs() + N * U * g.abs().sum(0) + TINY[w.dtype]}
    return out, tol


def close(name, got, want, tol):
    assert got.shape == want.shape, name
    off = (got.double() - want).abs() - tol
    assert not (off > 0).any(), (name, float(off.max()), int((off > 0).sum()))


def run(dat, eps=EPS, need=("x", "w", "b")):
    t = {k: dat[k].detach().requires_grad_(k in need) if dat[k] is not None else None
         for k in ("x", "w", "b")}
    res = dat["res"]
    if res is not None:
        res = res.detach().requires_grad_("x" in need)
        y, h = ops.layer_norm(t["x"], t["w"], t["b"], eps=eps, residual=res)
        outs, grads = [y, h], [dat["dy"], dat["dh"]]
        if grads[1] is None:
            outs, grads = outs[:1], grads[:1]
    else:
        y = ops.layer_norm(t["x"], t["w"], t["b"], eps=eps)
        h, outs, grads = None, [y], [dat["dy"]]
    leaves = [v for k, v in t.items() if k in need and v is not None]
    got = dict(zip([k for k in t if k in need and t[k] is not None],
                   torch.autograd.grad(outs, leaves, grads))) if leaves else {}
    out = {"y": y.detach()} | ({"h": h.detach()} if h is not None else {})
    return out | {"d" + k: v for k, v in got.items()}


def check(dat, eps=EPS):
    got = run(dat, eps)
    want, tol = reference(dat["x"], dat["w"], dat["b"], dat["dy"], dat["dh"], dat["res"], eps)
    for k, v in got.items():
        close(k, v, want[k], tol[k])
    return got


@pytest.mark.parametrize("D", [1, 2, 3, 7, 8, 9, 63, 64, 65, 100, 255, 256, 257, 512, 768, 769,
                               1000, 1024, 1025, 2047, 2048, 4096, 4100, 8191, 8192, 10000, 16384,
                               16392, 20001, 70000])
@pytest.mark.parametrize("types", range(len(TYPES)))
def test_widths(dev, D, types):
    dt, wt = TYPES[types]
    check(data(37 if D < 20000 else 5, D, dt, wt, dev, residual=D % 2 == 0, seed=D))


@pytest.mark.parametrize("N", [1, 2, 3, 4, 15, 16, 17, 64, 255, 1000, 5000, 20011])
@pytest.mark.parametrize("D", [24, 768, 1537, 4096])
def test_row_counts(dev, N, D):
    if N * D > 2 ** 25:
        pytest.skip("a large matrix of this width adds nothing")
    check(data(N, D, torch.bfloat16, torch.float32, dev, residual=N % 2 == 0, seed=N))


@pytest.mark.parametrize("pitch", [1, 3, 4, 8, 500])
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16, torch.float32])
def test_row_pitch_and_alignment(dev, pitch, dt):
    dat = data(50, 768, dt, dt, dev, pitch=pitch, seed=pitch)
    check(dat)
    # the same rows from an odd start, and gradients with a pitch of their own
    wide = torch.zeros(50, 768 + 7, dtype=dt, device=dev)
    wide[:, 1:769] = dat["dy"]
    a = run(dat)
    b = run(dat | {"dy": wide[:, 1:769]})
    for k in a:
        assert torch.equal(a[k], b[k]), k


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("D", [768, 1001, 5000])
def test_residual_gives_the_bits_of_a_sum_before(dev, dt, D):
    dat = data(40, D, dt, torch.float32, dev, residual=True)
    a = run(dat)
    b = run(dat | {"x": dat["x"] + dat["res"], "res": None, "dh": None})
    assert torch.equal(a["h"], dat["x"] + dat["res"]) and torch.equal(a["y"], b["y"])
    assert torch.equal(a["dw"], b["dw"]) and torch.equal(a["db"], b["db"])


@pytest.mark.parametrize("need", [("x",), ("w",), ("b",), ("w", "b"), ("x", "b"), ()])
def test_only_the_gradients_asked_for(dev, need):
    dat = data(33, 768, torch.bfloat16, torch.bfloat16, dev)
    full, part = run(dat), run(dat, need=need)
    assert set(part) == {"y"} | {"d" + k for k in need}
    for k, v in part.items():
        assert torch.equal(v, full[k]), k


def test_shapes_broadcasts_and_missing_parts(dev):
    g = torch.Generator(device=dev).manual_seed(3)
    x = torch.randn(4, 6, 96, generator=g, device=dev).requires_grad_(True)
    pos = torch.randn(1, 6, 96, generator=g, device=dev).requires_grad_(True)
    norm = LayerNorm(96, device=dev)
    y, h = norm(x, pos)
    y2 = torch.nn.functional.layer_norm(x + pos, (96,), norm.weight, norm.bias)
    w = torch.randn(4, 6, 96, generator=g, device=dev)
    got = torch.autograd.grad((y * w).sum(), [x, pos, norm.weight, norm.bias])
    want = torch.autograd.grad((y2 * w).sum(), [x, pos, norm.weight, norm.bias])
    for a, b in zip(got, want):
        assert a.shape == b.shape
        torch.testing.assert_close(a, b, rtol=1e-4, atol=1e-4)
    # the sum's gradient alone, and both
    (gx,) = torch.autograd.grad((norm(x, pos)[1] * w).sum(), [x])
    assert torch.equal(gx, w)
    # expanded rows (pitch 0), a vector, columns that are not contiguous, a negated view
    row = torch.randn(1, 96, generator=g, device=dev)
    one = ops.layer_norm(row[0], norm.weight, None)
    assert one.shape == (96,)
    assert torch.equal(ops.layer_norm(row.expand(5, 96), norm.weight), one.expand(5, 96))
    t = torch.randn(96, 7, generator=g, device=dev).t()
    assert torch.equal(ops.layer_norm(t, norm.weight), ops.layer_norm(t.contiguous(), norm.weight))
    neg = torch._neg_view(t.contiguous())
    assert torch.equal(ops.layer_norm(neg, norm.weight), ops.layer_norm(-t, norm.weight))
    # no rows
    e = torch.empty(0, 96, device=dev, requires_grad=True)
    y = norm(e)
    gx, gw, gb = torch.autograd.grad(y, [e, norm.weight, norm.bias], torch.empty_like(y))
    assert y.shape == (0, 96) and gx.shape == (0, 96) and not gw.any() and not gb.any()


@pytest.mark.parametrize("D", [5, 768, 3001, 20000])
def test_constant_rows_and_rows_far_from_zero(dev, D):
    dat = data(12, D, torch.float32, torch.float32, dev)
    dat["x"][:4] = torch.tensor([0.0, 1.0, -2.5, 1e20], device=dev)[:, None]
    y = ops.layer_norm(dat["x"][:4], dat["w"], dat["b"])
    assert torch.equal(y[0], dat["b"]) and torch.isfinite(y).all()
    dat["x"][4:8] = dat["x"][4:8] + 3e4            # spread 1 around 30,000
    dat["x"], dat["dy"] = dat["x"][4:], dat["dy"][4:]
    check(dat)


def test_largest_fp16_values(dev):
    dat = data(9, 1024, torch.float16, torch.float32, dev)
    dat["x"] = dat["x"].sign() * 65504
    got = check(dat)
    assert torch.isfinite(got["y"]).all()


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("D", [70, 768, 9000])
def test_what_is_not_finite_stays_in_its_row(dev, bad, D):
    dat = data(21, D, torch.bfloat16, torch.bfloat16, dev, residual=True)
    clean = run(dat)
    x = dat["x"].clone()
    x[7, D // 2] = bad
    got = run(dat | {"x": x})
    keep = torch.arange(21, device=dev) != 7
    for k in ("y", "h", "dx"):
        assert torch.equal(got[k][keep], clean[k][keep]), k
    assert torch.isnan(got["y"][7]).all() and torch.isnan(got["dx"][7]).all()
    assert torch.isnan(got["dw"]).all() and torch.equal(got["db"], clean["db"])


@pytest.mark.parametrize("N,D", [(64, 768), (3000, 768), (256, 4096), (7, 30000), (4096, 96)])
def test_the_same_bits_again_and_on_another_stream(dev, N, D):
    dat = data(N, D, torch.bfloat16, torch.float32, dev, residual=True)
    a = run(dat)
    s = torch.cuda.Stream(dev)
    s.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(s):
        b = run(dat)
    s.synchronize()
    for k in a:
        assert torch.equal(a[k], b[k]), k


@pytest.mark.parametrize("D", [6, 96, 300])
def test_gradients_against_differences_of_the_forward(dev, D):
    """A step of 2^-6 along a random direction: central differences of the fp32 forward have a
    truncation of about 2^-12 |third derivative| / 6 and a rounding of u |sum| 2^6, both far
    below 2e-3 of the product of the norms."""
    dat = data(16, D, torch.float32, torch.float32, dev, residual=True, seed=D)
    got = run(dat)
    g = torch.Generator(device=dev).manual_seed(9)

    def f(x, w, b):
        y, h = ops.layer_norm(x, w, b, eps=EPS, residual=dat["res"])
        return float((y.double() * dat["dy"].double()).sum() + (h.double() * dat["dh"].double()).sum())

    for k in ("x", "w", "b"):
        v = torch.randn(dat[k].shape, generator=g, device=dev)
        v /= v.norm()
        hi = {q: dat[q] + (v * 2 ** -6 if q == k else 0) for q in ("x", "w", "b")}
        lo = {q: dat[q] - (v * 2 ** -6 if q == k else 0) for q in ("x", "w", "b")}
        diff = (f(**hi) - f(**lo)) / 2 ** -5
        grad = float((got["d" + k].double() * v.double()).sum())
        assert abs(diff - grad) <= 2e-3 * float(got["d" + k].norm()), k


def test_offsets_past_2_31_elements(dev):
    D, N = 2056, (2 ** 31 + 2 ** 20) // 2056
    x = torch.randn(1000, D, device=dev).to(torch.bfloat16).repeat(N // 1000 + 1, 1)[:N]
    w = torch.ones(D, device=dev, dtype=torch.bfloat16).requires_grad_(True)
    dy = x.flip(1)
    x.requires_grad_(True)
    y = ops.layer_norm(x, w)
    dx, dw = torch.autograd.grad(y, [x, w], dy)
    tail = slice(N - 700, N)
    xs = x.detach()[tail].requires_grad_(True)
    ys = ops.layer_norm(xs, w)
    (dxs,) = torch.autograd.grad(ys, [xs], dy[tail])
    assert torch.equal(y[tail], ys) and torch.equal(dx[tail], dxs)
    assert torch.isfinite(dw).all()


def test_replays_of_a_graph(dev):
    dat = data(200, 768, torch.bfloat16, torch.bfloat16, dev, residual=True)
    x, w = dat["x"].clone().requires_grad_(True), dat["w"].requires_grad_(True)

    def step():
        y, h = ops.layer_norm(x, w, dat["b"], residual=dat["res"])
        return [y, h, *torch.autograd.grad([y, h], [x, w], [dat["dy"], dat["dh"]])]

    s = torch.cuda.Stream(dev)
    s.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream(dev).wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for k in range(3):
        with torch.no_grad():
            x.copy_(dat["x"] * (k + 1))
        graph.replay()
        torch.cuda.synchronize()
        got = [o.detach().clone() for o in outs]
        for a, b in zip(got, step()):
            assert torch.equal(a, b.detach()), k


def test_refusals(dev):
    x = torch.randn(4, 64, device=dev)
    w = torch.ones(64, device=dev)
    for args, kw, match in [
            ((x.cpu(), w), {}, "HIP device"), ((x, w.cpu()), {}, "HIP device"),
            ((x, w[:63]), {}, "weight must be"), ((x, w, w[:1]), {}, "bias must be"),
            ((x.bfloat16(), w.half()), {}, "x's dtype"), ((x, w, w.bfloat16()), {}, "x's dtype"),
            ((x.double(), w), {}, "unsupported dtype"), ((x.long(), w), {}, "unsupported dtype"),
            ((x, w), {"residual": x.bfloat16()}, "residual must be"),
            ((x[:, :0], w[:0]), {}, "last axis"), ((x, w), {"eps": -1.0}, "eps")]:
        with pytest.raises(RuntimeError, match=match):
            ops.layer_norm(*args, **kw)
    with pytest.raises(RuntimeError):
        ops.layer_norm(x, w, residual=torch.randn(5, 64, device=dev))
    for bad in (dict(normalized_shape=(4, 64)), dict(normalized_shape=64, elementwise_affine=False)):
        with pytest.raises(ValueError, match="one normalised axis"):
            LayerNorm(**bad)


def test_its_backward_is_not_differentiable(dev):
    x = torch.randn(4, 64, device=dev, requires_grad=True)
    w = torch.ones(64, device=dev, requires_grad=True)
    y = ops.layer_norm(x, w)
    gx, gw = torch.autograd.grad(y.square().sum(), [x, w], create_graph=True)
    with pytest.raises(RuntimeError, match="cannot be differentiated"):
        (gx.sum() + gw.sum()).backward()


def test_saved_rows_changed_in_place_are_noticed(dev):
    x = torch.randn(4, 64, device=dev)
    w = torch.ones(64, device=dev, requires_grad=True)
    y, h = ops.layer_norm(x, w, residual=x)
    with torch.no_grad():
        h.mul_(2)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


def test_under_activation_checkpointing(dev):
    from torch.utils.checkpoint import checkpoint
    dat = data(20, 768, torch.bfloat16, torch.float32, dev, residual=True)
    x, w = dat["x"].requires_grad_(True), dat["w"].requires_grad_(True)
    f = lambda x: ops.layer_norm(x, w, dat["b"], residual=dat["res"])  # noqa: E731
    want = torch.autograd.grad(f(x), [x, w], [dat["dy"], dat["dh"]])
    for reentrant in (False, True):
        out = checkpoint(f, x, use_reentrant=reentrant)
        x.grad = w.grad = None
        torch.autograd.backward(out, [dat["dy"], dat["dh"]])
        assert torch.equal(x.grad, want[0]) and torch.equal(w.grad, want[1])


def test_gradients_add_up_over_uses(dev):
    """One weight in two norms and one x as both operands: what each use gives is added."""
    x = torch.randn(9, 96, device=dev, requires_grad=True)
    w = torch.ones(96, device=dev, requires_grad=True)
    y, h = ops.layer_norm(x, w, residual=x)
    g = torch.randn_like(x)
    (ops.layer_norm(y, w) * g).sum().backward()
    xd, wd = x.detach().double().requires_grad_(True), w.detach().double().requires_grad_(True)
    ln = torch.nn.functional.layer_norm
    (ln(ln(xd + xd, (96,), wd), (96,), wd) * g.double()).sum().backward()
    torch.testing.assert_close(x.grad.double(), xd.grad, rtol=1e-4, atol=1e-5)
    torch.testing.assert_close(w.grad.double(), wd.grad, rtol=1e-4, atol=1e-5)
