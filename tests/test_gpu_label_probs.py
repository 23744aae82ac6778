"""GPU: log probabilities of labels, entropy, likeliest labels and the logits' gradient against float64,
over sizes, types, strides, ties and rows that are masked or not finite.

Tolerances: u = 2^-24.  With d = z - m (one rounding) a term e^d is off by 4 u (1 + |d|) of itself: the
product with log2 e, its constant, and the exponential.  A thread sums n terms, and moves its sum to a new
maximum at most once a vector, which costs what the terms of the move's length cost; some 20
additions join the threads.  So s, and log s absolutely, is off by at most e_s = u (4 (1 + E|d|) + 4 R + 2 n
+ 40), R the finite logits' range, and so is t / s relative to E|d|, the mean under p."""
import math

import pytest
import torch

from haste_amd import ops

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
UD = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 2.0 ** -126, torch.bfloat16: 2.0 ** -126, torch.float16: 2.0 ** -25}
TYPES = list(UD)
INF = math.inf


def reference(z, labels=None, top=0, dlp=None, dent=None):
    """float64 results and error bounds (rows with a finite logit and no NaN or infinity)."""
    zd, O = z.double(), z.shape[1]
    m = zd.amax(1, keepdim=True)
    d = zd - m
    ok = zd > -INF
    p = d.exp()
    s = p.sum(1, keepdim=True)
    p = p / s
    d0 = torch.where(ok, d, 0.0)
    e = (p * d0.abs()).sum(1, keepdim=True)
    R = d0.abs().amax(1, keepdim=True)
    es = U * (4 * (1 + e) + 4 * torch.minimum(R, torch.full_like(R, 1000.0)) + 2 * (O / 256 + 8) + 40)
    lp = d - s.log()
    ent = s.log() - (p * d0).sum(1, keepdim=True)
    eent = es * (2 + e) + U * ent.abs()
    out, tol = {"entropy": ent[:, 0]}, {"entropy": eent[:, 0]}
    elp = lambda x: es + U * (2 * torch.where(x > -INF, x.abs(), 0.0) + s.log().abs())  # noqa: E731
    if labels is not None:
        given = (labels >= 0) & (labels < O)
        at = labels.long().clamp(0, O - 1)
        out["log_probs"] = torch.where(given, lp.gather(1, at), 0.0)
        tol["log_probs"] = elp(lp.gather(1, at))
    if top:
        order = torch.sort(zd, dim=1, descending=True, stable=True).indices[:, :top]
        out |= {"top_labels": order, "top_log_probs": lp.gather(1, order)}
        tol["top_log_probs"] = elp(out["top_log_probs"])
    if dlp is not None or dent is not None:
        g = torch.zeros_like(s) if dlp is None else (dlp.double() * given).sum(1, keepdim=True)
        ga = torch.zeros_like(s) if dlp is None else (dlp.double() * given).abs().sum(1, keepdim=True)
        h = torch.zeros_like(s) if dent is None else dent.double()[:, None]
        l0 = torch.where(ok, lp, 0.0)
        dz = p * (-g - h * (l0 + ent))
        size = p * (ga + h.abs() * (l0.abs() + ent.abs()))
        err = p * (h.abs() * (2 * es + eent)) + size * (es + U * (labels.shape[1] if labels is not None
                                                                  else 0) + U * (16 + 4 * d0.abs()))
        if dlp is not None:
            dz = dz.scatter_add(1, at, dlp.double() * given)
            err = err.scatter_add(1, at, 4 * U * labels.shape[1] * (dlp.double() * given).abs())
        out["dz"] = dz
        tol["dz"] = UD[z.dtype] * dz.abs() + 1.01 * err + TINY[z.dtype]
    return out, tol


def run(z, labels=None, top=0, dlp=None, dent=None):
    z = z.detach().requires_grad_(dlp is not None or dent is not None)
    r = ops.label_log_probs(z, labels, top=top)
    out = {k: v for k, v in r._asdict().items() if v is not None}
    if z.requires_grad:
        pairs = [(r.log_probs, dlp), (r.entropy, dent)]
        pairs = [(a, b) for a, b in pairs if b is not None]
        out["dz"], = torch.autograd.grad([a for a, _ in pairs], [z], [b for _, b in pairs])
    return {k: v.detach() for k, v in out.items()}


def check(z, labels=None, top=0, dlp=None, dent=None):
    got = run(z, labels, top, dlp, dent)
    want, tol = reference(z, labels, top, dlp, dent)
    assert got.keys() == want.keys()
    for k, v in got.items():
        assert v.shape == want[k].shape, k
        if k == "top_labels":
            assert torch.equal(v, want[k])
            continue
        off = (v.double() - want[k]).abs() - tol[k]
        both = (v == want[k])   # (-infinity)
        assert not ((off > 0) | off.isnan() & ~both).any(), (k, float(off[~both].max()))
    return got


def data(B, O, L, dt, dev, seed=0, pitch=0, spread=2.0, masked=0.01):
    g = torch.Generator(device=dev).manual_seed(seed)
    z = (torch.randn(B, O + pitch, generator=g, device=dev) * spread - 4).to(dt)[:, :O]
    z[torch.rand(B, O, generator=g, device=dev) < masked] = -INF
    z[:, 0] = 0.5
    labels = torch.randint(-1, O, (B, L), generator=g, device=dev)
    dlp = torch.randn(B, L, generator=g, device=dev)
    return z, labels, dlp, torch.randn(B, generator=g, device=dev)


@pytest.mark.parametrize("O", [1, 2, 3, 7, 8, 9, 15, 16, 17, 63, 64, 65, 100, 255, 511, 512, 513, 1000,
                               2047, 2048, 2049, 4099, 8193, 16391, 40001])
@pytest.mark.parametrize("dt", TYPES)
def test_sizes(dev, O, dt):
    z, labels, dlp, dent = data(9, O, 5, dt, dev, seed=O)
    for top in {0, 1, min(O, 5), min(O, 33), min(O, 128)}:
        check(z, labels, top, dlp, dent)


@pytest.mark.parametrize("B,O", [(1, 131073), (3, 131073), (1, 1000003), (70, 20011), (300, 5003), (2100, 700)])
@pytest.mark.parametrize("top", [0, 10, 100])
def test_few_and_many_rows(dev, B, O, top):
    z, labels, dlp, dent = data(B, O, 4, torch.bfloat16, dev, seed=B, pitch=3)
    check(z, labels, top, dlp, dent)


@pytest.mark.parametrize("B,O,dt", [(520, 70001, torch.bfloat16), (513, 40009, torch.float16),
                                    (260, 60013, torch.float32)])
@pytest.mark.parametrize("top", [1, 10, 100])
def test_long_parts(dev, B, O, dt, top):
    """Parts of many steps, whose likeliest labels are found again by windows of them."""
    z, _, _, _ = data(B, O, 1, dt, dev, seed=top, pitch=5)
    i = torch.arange(O, device=dev)
    z[3] = -1.5                                # all equal
    z[4], z[5] = (i / O).to(dt), (-i / O).to(dt)
    z[6] = (i * 7919 % 13).to(dt)              # many of each
    z[7], z[7, O - 3:] = -INF, 2.0             # three left, at the end
    z[8, O // 2 : O // 2 + 300] = 9.0          # side by side
    check(z, None, top)
    z[9, 12345] = z[9, O - 1] = math.nan
    z[10, 23456] = INF
    got = run(z, None, top)
    order = torch.sort(z[9:11].double(), dim=1, descending=True, stable=True).indices[:, :top]
    assert torch.equal(got["top_labels"][9:11], order)
    assert got["top_log_probs"][9:11].isnan().all()


@pytest.mark.parametrize("kind", ["equal", "ascending", "descending", "steps", "zeros", "two"])
@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("top", [1, 5, 32, 128])
def test_ties_and_orders(dev, kind, dt, top):
    """Equal logits in the labels' order, whatever the order in which they are met."""
    O = 30011
    i = torch.arange(O, device=dev, dtype=torch.float32)
    z = {"equal": torch.full_like(i, -3.0), "ascending": i / O, "descending": -i / O,
         "steps": (i * 7919 % 13).floor(), "zeros": torch.where(i % 2 == 0, -0.0, 0.0),
         "two": (i % 500 == 499).float()}[kind]
    check(torch.stack([z, z.roll(77), z.flip(0)]).to(dt), None, top)


@pytest.mark.parametrize("dt", TYPES)
def test_masks(dev, dt):
    z, labels, dlp, dent = data(6, 5003, 4, dt, dev)
    low = torch.finfo(dt).min
    z[0] = -INF
    z[0, 4321] = 1.0                    # one label left
    z[1, 7:] = -INF
    z[2, 100:] = low                    # the type's lowest value masks
    z[3, :4000] = low
    labels[0, 0], labels[1, 0], labels[2, 0] = 4321, 3, 5
    check(z, labels, 16, dlp, dent)
    # every label at the lowest value: as likely as one another
    z = torch.full((2, 700), low, device=dev, dtype=dt)
    check(z, labels[:2] % 700, 3, dlp[:2], dent[:2])


@pytest.mark.parametrize("dt", TYPES)
def test_rows_without_a_distribution(dev, dt):
    """All ruled out, NaN, +infinity: NaN in that row and in no other; the likeliest are still given."""
    z, labels, dlp, dent = data(8, 3001, 4, dt, dev)
    bad = [1, 3, 4, 6]
    clean = check(z, labels, 6, dlp, dent)     # (the same call: a row's bits go with its place)
    z[1] = -INF
    z[3, 2500] = math.nan
    z[3, 2900] = math.nan
    z[4, 17] = INF
    z[6] = math.nan
    labels[bad, 0], labels[bad, 1] = 5, -1
    got = run(z, labels, 6, dlp, dent)
    for k, v in got.items():
        assert torch.equal(v[[0, 2, 5, 7]], clean[k][[0, 2, 5, 7]]), k
    assert got["entropy"][bad].isnan().all() and got["log_probs"][bad, 0].isnan().all()
    assert (got["log_probs"][bad, 1] == 0).all() and got["dz"][bad].isnan().all()
    assert got["top_log_probs"][bad].isnan().all()
    assert got["top_labels"][1].tolist() == list(range(6))
    assert got["top_labels"][3, :2].tolist() == [2500, 2900]
    assert got["top_labels"][4, 0] == 17 and got["top_labels"][6].tolist() == list(range(6))


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("O", [1, 9, 700, 5003, 40001])
def test_infinity_is_the_likeliest(dev, dt, O):
    """One label at +infinity and no NaN, or one NaN: it is the first of any number of labels."""
    z, _, _, _ = data(6, O, 1, dt, dev)
    at = torch.tensor([0, O // 2, O - 1] * 2, device=dev)
    z[torch.arange(6, device=dev), at] = torch.tensor([INF] * 3 + [math.nan] * 3, device=dev, dtype=dt)
    for top in {1, min(2, O)}:
        assert torch.equal(run(z, None, top)["top_labels"][:, 0], at)


@pytest.mark.parametrize("scale", [1e-3, 30.0, 1e4, 1e38])
def test_logits_far_apart(dev, scale):
    g = torch.Generator(device=dev).manual_seed(3)
    z = (torch.rand(4, 3001, generator=g, device=dev) * 2 - 1) * scale
    labels = torch.randint(0, 3001, (4, 3), generator=g, device=dev)
    labels[:, 0] = z.argmax(1)
    check(z, labels, 7, torch.randn(4, 3, generator=g, device=dev), None)
    check(z + (5 * scale if scale < 1e37 else 0), labels, 7, None,
          torch.randn(4, generator=g, device=dev))


def test_labels_twice_and_outside(dev):
    z, labels, dlp, dent = data(20, 300, 9, torch.float32, dev)
    labels[:, 3] = labels[:, 1]
    labels[:, 8] = labels[:, 1]
    labels[5] = -1
    labels[6] = 300
    labels[7, :4] = torch.tensor([2 ** 40, -2 ** 40, 299, 299], device=dev)
    check(z, labels, 0, dlp, dent)
    got = check(z, labels, 0, dlp, None)
    assert not got["dz"][5].any() and not got["dz"][6].any()
    # every label asked for, without a gradient, and as many as may have one
    z, _, _, _ = data(3, 9000, 1, torch.float32, dev)
    check(z, torch.arange(9000, device=dev).expand(3, 9000))
    z, labels, dlp, dent = data(3, 5000, 4096, torch.float32, dev)
    check(z, labels, 0, dlp, dent)
    # many labels, more than threads
    z, labels, dlp, dent = data(3, 900, 700, torch.float32, dev)
    check(z, labels, 0, dlp, dent)


@pytest.mark.parametrize("kind", ["pitch1", "pitch3", "pitch8", "one_row", "strided", "shape3", "vector",
                                  "int32", "strided_labels", "offset"])
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32])
def test_layouts(dev, kind, dt):
    pitch = {"pitch1": 1, "pitch3": 3, "pitch8": 8}.get(kind, 0)
    z, labels, dlp, dent = data(12, 2053, 4, dt, dev, pitch=pitch)
    if kind == "one_row":
        z = z[:1].expand(12, 2053)
    elif kind == "strided":
        z = z.t().contiguous().t()
    elif kind == "int32":
        labels = labels.int()
    elif kind == "strided_labels":
        labels = labels.t().contiguous().t()
    elif kind == "offset":
        z = torch.cat([z, z], 1)[:, 5: 5 + 2053]
    if kind in ("shape3", "vector"):
        flat = check(z, labels, 5, dlp, dent)
        if kind == "shape3":
            got = run(z.view(3, 4, -1), labels.view(3, 4, -1), 5, dlp.view(3, 4, -1), dent.view(3, 4))
        else:
            got = run(z[0], labels[0], 5, dlp[0], dent[0])
        for k, v in got.items():
            assert torch.equal(v, flat[k].view(v.shape) if kind == "shape3" else flat[k][0]), k
        return
    check(z, labels, 5, dlp, dent)


def test_empty(dev):
    r = ops.label_log_probs(torch.zeros(0, 5, device=dev), torch.zeros(0, 2, dtype=torch.int64, device=dev),
                            top=3)
    assert r.log_probs.shape == (0, 2) and r.entropy.shape == (0,) and r.top_labels.shape == (0, 3)
    z, _, _, dent = data(4, 50, 0, torch.float32, dev)
    none = torch.zeros(4, 0, dtype=torch.int64, device=dev)
    assert check(z, none, 0, None, dent)["log_probs"].shape == (4, 0)
    check(z, None, 0, None, dent)


def test_gradients_that_do_not_arrive(dev):
    """Only one output is used: what the other would add is left out."""
    z, labels, dlp, dent = data(7, 600, 3, torch.float32, dev)
    check(z, labels, 0, dlp, None)
    check(z, labels, 2, None, dent)
    z = z.requires_grad_(True)
    r = ops.label_log_probs(z, labels, top=4)
    assert not r.top_log_probs.requires_grad and not r.top_labels.requires_grad
    (-r.log_probs.mean()).backward()          # (a gradient of one element for all)
    want, tol = reference(z.detach(), labels, 0, torch.full_like(dlp, -1 / 21), None)
    assert ((z.grad.double() - want["dz"]).abs() <= tol["dz"] + 1e-7 * want["dz"].abs()).all()


def test_loss_is_torchs(dev):
    z, _, _, _ = data(64, 1000, 1, torch.float32, dev, masked=0.0)
    labels = torch.randint(0, 1000, (64, 1), device=dev)
    a, b = z.clone().requires_grad_(True), z.clone().requires_grad_(True)
    la = -ops.label_log_probs(a, labels).log_probs.mean()
    lb = torch.nn.functional.cross_entropy(b, labels[:, 0])
    la.backward()
    lb.backward()
    assert abs(float(la) - float(lb)) < 1e-5
    # (two fp32 forms of p, each within 2^-19 of it, over 64 rows)
    assert (a.grad - b.grad).abs().max() < 2 * 2.0 ** -19 / 64


def test_gradient_against_differences(dev):
    z, labels, dlp, dent = data(3, 40, 2, torch.float32, dev, masked=0.0)
    dz = run(z, labels, 0, dlp, dent)["dz"]

    def f(z):
        want, _ = reference(z, labels)
        return (want["log_probs"] * dlp.double()).sum() + (want["entropy"] * dent.double()).sum()
    for i, j in ((0, 0), (1, 17), (2, 39), (0, int(labels[0].max()))):
        step = torch.zeros_like(z, dtype=torch.float64)
        step[i, j] = 1e-4
        slope = (f(z.double() + step) - f(z.double() - step)) / 2e-4
        # (third derivatives are below 40: 40 h^2 / 6, and fp32's p)
        assert abs(float(slope) - float(dz[i, j])) < 1e-6 + 40 * 1e-8 / 6 + 1e-5 * abs(float(slope))


def test_past_2_31_logits(dev):
    """1024 rows of 3,000,000: offsets past 32 bits, with a gradient; whole rows are known."""
    B, O = 1024, 3_000_000
    torch.cuda.empty_cache()
    if torch.cuda.mem_get_info(dev)[0] < 40 << 30:
        pytest.skip("needs 40 GiB")
    z = torch.full((B, O), -2.0, dtype=torch.bfloat16, device=dev)
    hot = (torch.arange(B, device=dev) * 2929) % O
    z.scatter_(1, hot[:, None], 14.0)
    labels = torch.stack([hot, (hot + 1) % O], 1)
    z.requires_grad_(True)
    r = ops.label_log_probs(z, labels, top=2)
    s = 1 + (O - 1) * math.exp(-16.0)
    assert (r.log_probs[:, 0] + math.log(s)).abs().max() < 1e-4
    assert (r.log_probs[:, 1] + 16 + math.log(s)).abs().max() < 1e-4
    ent = math.log(s) + (O - 1) * math.exp(-16.0) * 16 / s
    assert (r.entropy - ent).abs().max() < 1e-3
    assert torch.equal(r.top_labels[:, 0], hot)
    assert torch.equal(r.top_labels[:, 1], (hot == 0).long())
    dz, = torch.autograd.grad([r.log_probs], [z], [torch.tensor([1.0, 0.0], device=dev).expand(B, 2)])
    low = torch.tensor(-math.exp(-16.0) / s, device=dev).to(torch.bfloat16)
    for i in range(0, B, 64):
        part = dz[i: i + 64].clone()
        top = part.gather(1, hot[i: i + 64, None])
        assert (top.float() - (1 - 1 / s)).abs().max() < 2.0 ** -8
        part.scatter_(1, hot[i: i + 64, None], low.item())
        assert ((part.float() - low.float()).abs() <= 2.0 ** -7 * low.float().abs()).all()


def test_refusals(dev):
    z, labels, dlp, _ = data(4, 50, 2, torch.float32, dev)
    for bad, match in ((labels.float(), "int64 or int32"), (labels.cpu(), "HIP device"),
                       (labels[:3], r"\[..., L\]"), (labels[0], r"\[..., L\]")):
        with pytest.raises(RuntimeError, match=match):
            ops.label_log_probs(z, bad)
    for top in (-1, 51, 129):
        with pytest.raises(RuntimeError, match="top must be"):
            ops.label_log_probs(z, labels, top=top)
    with pytest.raises(RuntimeError, match="dtype"):
        ops.label_log_probs(z.double(), labels)
    with pytest.raises(RuntimeError, match="last axis"):
        ops.label_log_probs(z[:, :0], None)
    z = z.clone().requires_grad_(True)
    with pytest.raises(RuntimeError, match="4096 labels"):
        ops.label_log_probs(z, labels.repeat(1, 2049))
    r = ops.label_log_probs(z, labels)
    g, = torch.autograd.grad([r.log_probs], [z], [dlp.requires_grad_(True)], create_graph=True)
    with pytest.raises(RuntimeError, match="cannot be differentiated"):
        g.sum().backward()
    r = ops.label_log_probs(z * 1, labels)
    y = z * 1
    r = ops.label_log_probs(y, labels)
    y.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        r.log_probs.sum().backward()


def test_replays_of_a_graph(dev):
    z, labels, dlp, dent = data(40, 9001, 4, torch.bfloat16, dev)
    z.requires_grad_(True)
    stream = torch.cuda.Stream(dev)
    stream.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(stream):
        for _ in range(2):
            run(z, labels, 8, dlp, dent)
    torch.cuda.current_stream(dev).wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        r = ops.label_log_probs(z, labels, top=8)
        dz, = torch.autograd.grad([r.log_probs, r.entropy], [z], [dlp, dent])
    for seed in range(4):
        fresh = data(40, 9001, 4, torch.bfloat16, dev, seed=seed + 5)
        with torch.no_grad():
            for a, b in zip((z, labels, dlp, dent), fresh):
                a.copy_(b)
        graph.replay()
        torch.cuda.synchronize()
        kept = {k: v.clone() for k, v in r._asdict().items()} | {"dz": dz.clone()}
        want = check(z.detach(), labels, 8, dlp, dent)
        torch.cuda.synchronize()
        for k, v in want.items():
            assert torch.equal(kept[k], v), k
