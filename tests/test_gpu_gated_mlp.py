"""GPU: the gated feed-forward block and its gradients against float64, over sizes, types, activations,
strides and the kernels that a size takes (few rows, small and large tiles, K in parts).

Tolerances: u = 2^-24, U_d half a step of the type.  A product of K terms is off by (K + 2) u of its
terms' absolute sum, whatever the order, and by its operands' errors times the other operand.  What
lies between the products is rounded to the type: h, and for the backward dg and du; u act'(g) and act(g)
are kept in 24 bits (2^-17 of their size; fp32: none lost).  act is within 8 u of its size (16-bit gelu: 1.5e-6, 25 u,
of its tail besides) and moves by at most 1.2 |dg|; act' moves by at most 1.2 |dg|."""
import math

import pytest
import torch

from haste_amd import ops
from haste_amd.gated_mlp import GatedMLP

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
UD = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 2.0 ** -126, torch.bfloat16: 2.0 ** -126, torch.float16: 2.0 ** -25}
TYPES = list(UD)
ACTS = ["silu", "gelu", "gelu_tanh"]


def act(name, g):
    """act(g) and act'(g) in float64."""
    if name == "silu":
        s = torch.sigmoid(g)
        return g * s, s * (1 + g * (1 - s))
    if name == "gelu":
        c = 0.5 * torch.erfc(-g / math.sqrt(2))
        return g * c, c + g * torch.exp(-g * g / 2) / math.sqrt(2 * math.pi)
    k = math.sqrt(2 / math.pi)
    t = torch.tanh(k * (g + 0.044715 * g ** 3))
    return 0.5 * g * (1 + t), 0.5 * (1 + t) + 0.5 * g * (1 - t * t) * k * (1 + 3 * 0.044715 * g * g)


def reference(x, wg, wu, wd, name, dy=None):
    """float64 results and error bounds."""
    dt = x.dtype
    ud, tiny = UD.get(dt, 0.0), TINY.get(dt, 0.0)
    X, G, Up, Dn = (t.double() for t in (x, wg, wu, wd))
    D, H = X.shape[1], G.shape[0]
    mm = lambda a, b: a @ b.contiguous()  # noqa: E731
    g, u = mm(X, G.t()), mm(X, Up.t())
    eg, eu = ((D + 2) * U * mm(X.abs(), w.abs().t()) for w in (G, Up))
    a, s = act(name, g)
    ka = 16 if dt is torch.float32 or name != "gelu" else 42
    ea = 1.2 * eg + ka * U * (a.abs() + g.abs() * 0.1)
    h = a * u
    eh = ea * (u.abs() + eu) + a.abs() * eu + ud * h.abs() + tiny
    y = mm(h, Dn.t())
    ey = mm(eh, Dn.abs().t()) + (H + 2) * U * mm(h.abs(), Dn.abs().t())
    out, tol = {"y": y}, {"y": ud * y.abs() + 1.05 * ey + tiny}
    if dy is not None:
        Y = dy.double()
        N, O = Y.shape
        dh = mm(Y, Dn)
        edh = (O + 2) * U * mm(Y.abs(), Dn.abs())
        ea, es = 1.2 * eg + ka * U * (a.abs() + 0.1 * g.abs()), 1.2 * eg + ka * U * (s.abs() + 0.1)
        kept = 0.0 if dt is torch.float32 else 2.0 ** -17
        eus = eu * s.abs() + u.abs() * es + eu * es
        eus, ea = 1.05 * eus + kept * (u * s).abs(), 1.05 * ea + kept * a.abs()
        dg, du = dh * u * s, dh * a
        edg = 1.05 * (edh * (u * s).abs() + dh.abs() * eus + edh * eus) + ud * dg.abs() + tiny
        edu = 1.05 * (edh * a.abs() + dh.abs() * ea + edh * ea) + ud * du.abs() + tiny

        def product(p, ep, q, eq, K):
            e = mm(ep, q.abs()) + (K + 2) * U * mm(p.abs(), q.abs())
            return mm(p, q), e if eq is None else e + mm(p.abs() + ep, eq)
        dx1, e1 = product(dg, edg, G, None, 2 * H)
        dx2, e2 = product(du, edu, Up, None, 2 * H)
        zero = torch.zeros_like
        res = {"dx": (dx1 + dx2, e1 + e2), "dwg": product(dg.t(), edg.t(), X, None, N),
               "dwu": product(du.t(), edu.t(), X, None, N),
               "dwd": product(Y.t(), zero(Y.t()), h, eh, N)}
        for k, (v, e) in res.items():
            out[k], tol[k] = v, ud * v.abs() + 1.05 * e + tiny
    return out, tol


def data(N, D, H, O, dt, dev, seed=0):
    g = torch.Generator(device=dev).manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, device=dev)  # noqa: E731
    return dict(x=r(N, D).to(dt), wg=(r(H, D) / D ** 0.5).to(dt), wu=(r(H, D) / D ** 0.5).to(dt),
                wd=(r(O, H) / H ** 0.5).to(dt), dy=r(N, O).to(dt))


def run(d, name="silu", need=("x", "wg", "wu", "wd")):
    t = {k: d[k].detach().requires_grad_(k in need) for k in ("x", "wg", "wu", "wd")}
    y = ops.gated_mlp(t["x"], t["wg"], t["wu"], t["wd"], activation=name)
    out = {"y": y.detach()}
    if d.get("dy") is not None and need:
        got = torch.autograd.grad([y], [t[k] for k in t if k in need], [d["dy"]])
        out |= dict(zip(["d" + k for k in t if k in need], got))
    return out


def close(got, want, tol):
    for k, v in got.items():
        assert v.shape == want[k].shape, k
        off = (v.double() - want[k]).abs() - tol[k]
        assert not ((off > 0) | off.isnan()).any(), (k, float(off.max()), int((off > 0).sum()))


def check(d, name="silu", need=("x", "wg", "wu", "wd")):
    got = run(d, name, need)
    close(got, *reference(d["x"], d["wg"], d["wu"], d["wd"], name, d["dy"]))
    return got


@pytest.mark.parametrize("N,D,H,O", [
    (1, 1, 1, 1), (1, 8, 8, 8), (2, 3, 5, 7), (16, 32, 16, 32), (17, 33, 31, 40), (33, 100, 60, 20),
    (64, 64, 64, 64), (65, 64, 64, 64), (65, 1, 2, 3), (100, 7, 300, 9), (127, 129, 65, 191),
    (128, 128, 128, 128), (129, 136, 120, 264), (200, 301, 103, 301), (257, 40, 1000, 24),
    (500, 768, 256, 96), (1000, 72, 72, 520), (700, 513, 255, 129)])
@pytest.mark.parametrize("dt", TYPES)
def test_sizes(dev, N, D, H, O, dt):
    check(data(N, D, H, O, dt, dev, seed=N + D), ACTS[(N + D) % 3])


@pytest.mark.parametrize("N", [1, 2, 15, 16, 17, 31, 32, 33, 48, 64, 65, 96])
@pytest.mark.parametrize("dt", TYPES)
def test_few_rows(dev, N, dt):
    d = data(N, 768, 1003, 768, dt, dev, seed=N)
    check(d, "silu", need=())
    check(data(N, 301, 136, 77, dt, dev, seed=N), "gelu")


@pytest.mark.parametrize("name", ACTS)
@pytest.mark.parametrize("dt", TYPES)
def test_activations(dev, name, dt):
    """Gates from far below zero to far above it."""
    d = data(300, 64, 96, 32, dt, dev)
    d["wg"] *= 4.0
    check(d, name)


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("sizes", [(8200, 1500, 4100, 1492), (8192, 1536, 4096, 1536)])
def test_large_tiles(dev, sizes, dt):
    check(data(*sizes, dt, dev), "silu")


@pytest.mark.parametrize("dt", TYPES)
def test_k_in_parts(dev, dt):
    """Few tiles and a long K: every product in parts, of uneven steps."""
    check(data(7001, 100, 72, 88, dt, dev), "silu")
    check(data(130, 2000, 2500, 136, dt, dev), "gelu_tanh")


@pytest.mark.parametrize("need", [("x",), ("wg",), ("wu",), ("wd",), ("x", "wd"), ("wg", "wu")])
def test_gradients_that_are_asked_for(dev, need):
    check(data(150, 72, 88, 56, torch.bfloat16, dev), "silu", need)


@pytest.mark.parametrize("kind", ["pitch", "odd_pitch", "offset", "transposed", "packed_weights",
                                  "one_row", "one_row_gradient", "shape", "vector"])
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("N", [40, 200])
def test_layouts(dev, kind, dt, N):
    d = data(N, 64, 96, 72, dt, dev)
    wide = lambda t, a, b: torch.cat([t, t, t], 1)[:, a: a + b]  # noqa: E731
    if kind == "pitch":
        d = {k: wide(v, 8 if k != "x" else 16, v.shape[1]) for k, v in d.items()}
    elif kind == "odd_pitch":
        d = {k: torch.cat([v, v[:, :3]], 1)[:, : v.shape[1]] for k, v in d.items()}
    elif kind == "offset":
        d = {k: wide(v, 3, v.shape[1]) for k, v in d.items()}
    elif kind == "transposed":
        d = {k: v.t().contiguous().t() for k, v in d.items()}
    elif kind == "packed_weights":
        both = torch.cat([d["wg"], d["wu"]])
        d["wg"], d["wu"] = both[:96], both[96:]
    elif kind == "one_row":
        d["x"] = d["x"][:1].expand(N, 64)
    elif kind == "one_row_gradient":
        d["dy"] = d["dy"][:1].expand(N, 72)
    if kind in ("shape", "vector"):
        flat = run(d)
        if kind == "shape":
            d["x"], d["dy"] = d["x"].view(4, N // 4, 64), d["dy"].view(4, N // 4, 72)
        else:
            d["x"], d["dy"] = d["x"][0], d["dy"][0]
            flat = {"y": run(dict(d, x=d["x"][None], dy=d["dy"][None]))["y"][0]}
        got = run(d)
        for k in flat:
            assert torch.equal(got[k].reshape(flat[k].shape), flat[k]), k
        return
    check(d)


@pytest.mark.parametrize("pads", [(0, 8), (8, 0), (16, 8), (0, 3), (3, 0), (5, 8), (8, 5)])
@pytest.mark.parametrize("N,H", [(40, 96), (200, 96), (600, 1001)])
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16, torch.float32])
def test_projections_of_two_pitches(dev, pads, N, H, dt):
    """w_gate and w_up with rows at different pitches: the bits of plain ones."""
    d = data(N, 64, H, 72, dt, dev, seed=1)
    want = run(d)
    for k, pad in zip(("wg", "wu"), pads):
        wide = torch.full((H, 64 + pad), float("nan"), dtype=dt, device=dev)
        wide[:, :64] = d[k]
        d[k] = wide[:, :64]
    got = run(d)
    for k in want:
        assert torch.equal(got[k], want[k]), k


def test_pitches_with_rubbish_between_rows(dev):
    """What lies between rows that are read in place is not taken for zeros."""
    for dt in (torch.bfloat16, torch.float16):
        d = data(300, 60, 100, 52, dt, dev)
        for k, v in d.items():
            wide = torch.full((v.shape[0], 112), float("nan"), dtype=dt, device=dev)
            wide[:, : v.shape[1]] = v
            d[k] = wide[:, : v.shape[1]]
        check(d)
        check(dict(d, x=d["x"][:20], dy=d["dy"][:20]))


def test_empty(dev):
    d = data(0, 24, 40, 16, torch.bfloat16, dev)
    got = run(d)
    assert got["y"].shape == (0, 16) and got["dx"].shape == (0, 24)
    assert not any(got[k].any() for k in ("dwg", "dwu", "dwd"))


def test_what_is_not_finite_stays_in_its_row(dev):
    d = data(300, 64, 96, 72, torch.bfloat16, dev)
    clean = run(d)
    d["x"][17, 3] = float("inf")
    d["x"][200, 5] = float("nan")
    d["dy"][17] = d["dy"][200] = 0
    got = run(d)
    keep = torch.ones(300, dtype=torch.bool, device=dev)
    keep[[17, 200]] = False
    assert torch.equal(got["y"][keep], clean["y"][keep]) and torch.equal(got["dx"][keep], clean["dx"][keep])
    assert not got["y"][~keep].isfinite().any()


def test_two_runs_give_the_same_bits(dev):
    for sizes in ((7001, 100, 72, 88), (500, 768, 256, 96), (20, 768, 1000, 768)):
        d = data(*sizes, torch.bfloat16, dev)
        a, b = run(d), run(d)
        assert all(torch.equal(a[k], b[k]) for k in a)


def test_gradient_against_differences(dev):
    d = data(70, 24, 40, 16, torch.float32, dev)
    got = run(d, "gelu")
    f = lambda **kw: (reference(*(kw.get(k, d[k]).double() for k in ("x", "wg", "wu", "wd")), "gelu",  # noqa: E731
                                None)[0]["y"] * d["dy"].double()).sum()
    for k in ("x", "wg", "wu", "wd"):
        step = torch.zeros_like(d[k], dtype=torch.float64)
        step[3, 7] = 1e-5
        slope = float(f(**{k: d[k].double() + step}) - f(**{k: d[k].double() - step})) / 2e-5
        # (the difference's own error: third derivatives times 1e-10, and 2^-52 of the sum over 1e-5)
        assert abs(slope - float(got["d" + k][3, 7])) < 1e-5 * (1 + abs(slope))


def test_module(dev):
    m = GatedMLP(48, 80, activation="gelu", device=dev, dtype=torch.bfloat16)
    x = torch.randn(3, 9, 48, device=dev, dtype=torch.bfloat16, requires_grad=True)
    y = m(x)
    assert y.shape == x.shape
    y.float().square().sum().backward()
    assert all(p.grad.shape == p.shape for p in m.parameters()) and x.grad.shape == x.shape
    assert list(m.state_dict()) == ["w_gate", "w_up", "w_down"]
    assert GatedMLP(48, 80, 20, device=dev)(torch.zeros(2, 48, device=dev)).shape == (2, 20)
    with pytest.raises(ValueError, match="activation"):
        GatedMLP(48, 80, activation="tanh")


def test_refusals(dev):
    d = data(4, 16, 24, 8, torch.float32, dev)
    f = lambda **kw: ops.gated_mlp(**dict(dict(x=d["x"], w_gate=d["wg"], w_up=d["wu"], w_down=d["wd"]), **kw))  # noqa: E731
    with pytest.raises(ValueError, match="activation"):
        f(activation="swish")
    for kw, match in ((dict(w_up=d["wu"][:20]), "one shape"), (dict(x=d["x"][:, :8]), "features"),
                      (dict(w_down=d["wd"][:, :8]), "features"), (dict(w_gate=d["wg"].half()), "must be"),
                      (dict(x=d["x"].cpu()), "HIP device"), (dict(w_up=d["wu"].cpu()), "HIP device"),
                      (dict(w_down=d["wd"][0]), "matrix"), (dict(x=d["x"].double()), "dtype")):
        with pytest.raises(RuntimeError, match=match):
            f(**kw)
    y = f(x=d["x"].clone().requires_grad_(True), w_gate=d["wg"].requires_grad_(True))
    g, = torch.autograd.grad([y], [d["wg"]], [d["dy"].requires_grad_(True)], create_graph=True)
    with pytest.raises(RuntimeError, match="cannot be differentiated"):
        g.sum().backward()


@pytest.mark.parametrize("sizes", [(300, 64, 96, 72), (7001, 100, 72, 88), (20, 64, 96, 72)])
def test_replays_of_a_graph(dev, sizes):
    d = data(*sizes, torch.bfloat16, dev)
    leaves = [d[k].requires_grad_(True) for k in ("x", "wg", "wu", "wd")]
    stream = torch.cuda.Stream(dev)
    stream.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(stream):
        for _ in range(2):
            torch.autograd.grad([ops.gated_mlp(*leaves)], leaves, [d["dy"]])
    torch.cuda.current_stream(dev).wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = ops.gated_mlp(*leaves)
        grads = torch.autograd.grad([y], leaves, [d["dy"]])
    for seed in range(4):
        fresh = data(*sizes, torch.bfloat16, dev, seed=seed + 3)
        with torch.no_grad():
            for k, v in fresh.items():
                d[k].copy_(v)
        graph.replay()
        torch.cuda.synchronize()
        kept = [t.detach().clone() for t in (y, *grads)]
        want = run(d)
        torch.cuda.synchronize()
        for a, b in zip(kept, want.values()):
            assert torch.equal(a, b)
