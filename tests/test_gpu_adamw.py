"""GPU: AdamW's step with 32- and 8-bit states, and the gradients' norm, against float64.

Every step is compared with the reference's step from the state the library had before it.  fp32
arithmetic is off by at most a few u = 2^-24 of the terms: m by 3 u (|b1 m| + |(1 - b1) g|), v
alike, the update by 16 u of itself, w by 4 u |w| more; to that comes the rounding to w's type.
A value rounded by drawn bits may land on the other neighbour where what is cut off is
that close to the draw: one spacing, rarely."""
import copy

import numpy as np
import pytest
import torch

import adamw_reference as ref
from haste_amd.optim_adamw import STATE_BLOCK, AdamW, grad_norm

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
MANT = {torch.bfloat16: (7, -126), torch.float16: (10, -14)}
UD = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
SIZES = [1, 3, 8, 127, 128, 129, 1000, 4101, 70001]
HYPER = dict(lr=1e-2, betas=(0.9, 0.99), eps=1e-8, weight_decay=0.1)


def f64(t):
    return t.detach().float().cpu().numpy().astype(np.float64).reshape(-1)


def make(dev, sizes, wt, gt, seed=0, gscale=1e-2, **kw):
    g = torch.Generator(device=dev).manual_seed(seed)
    ps = [torch.nn.Parameter((torch.randn(n, generator=g, device=dev) * 0.1).to(wt)) for n in sizes]
    opt = AdamW(ps, **(HYPER | kw))
    return ps, opt, g


def new_grads(ps, gt, g, gscale=1e-2):
    for p in ps:
        spread = torch.exp(2 * torch.randn(p.shape, generator=g, device=p.device))
        grad = (torch.randn(p.shape, generator=g, device=p.device) * spread * gscale).to(gt)
        if gt is not p.dtype:
            p.grad_dtype = gt
        p.grad = grad


def moments(opt, p):
    """(m, v) as the state holds them, [n] float64."""
    s, n = opt.state[p], p.numel()
    if not s:
        return np.zeros(n), np.zeros(n)
    if "exp_avg_sq" in s:
        return f64(s["exp_avg"]), f64(s["exp_avg_sq"])
    m, u = (np.repeat(f64(s[k + "_scale"]), STATE_BLOCK) * f64(s[k]) for k in ("exp_avg", "rms"))
    return m[:n], u[:n] ** 2


def pad(x):
    return np.concatenate([x, np.zeros(-len(x) % ref.BLOCK)])


def check_step(opt, ps, before, seed, factor=1.0):
    """The state and parameters of every p with a gradient, from what they were before."""
    group = opt.param_groups[0]
    bits, sr = group["state_bits"], group["stochastic_rounding"]
    flips = total = 0
    for i, p in enumerate(ps):
        w0, m0, v0, t0 = before[i]
        if p.grad is None:
            assert np.array_equal(f64(p), w0, equal_nan=True)
            continue
        t, g = t0 + 1, f64(p.grad) * factor
        assert opt.state[p]["step"] == t
        (b1, b2), lr, wd = group["betas"], group["lr"], group["weight_decay"]
        w, m, v = ref.step(w0, g, m0, v0, t, lr, b1, b2, group["eps"], wd)
        em = 4 * U * (np.abs(b1 * m0) + np.abs((1 - b1) * g))
        ev = 6 * U * v
        upd = np.abs(w - w0 * (1 - lr * wd))
        ew = 4 * U * np.abs(w0) + 16 * U * upd + upd * np.where(m != 0, em / np.maximum(np.abs(m), 1e-300), 0)
        got_m, got_v = moments(opt, p)
        r, rm, ru = ref.draws(np.arange(len(pad(w))), bits, i, seed) if sr or bits == 8 else (None,) * 3
        if bits == 32:
            assert (np.abs(got_m - m) <= em + 1e-45).all() and (np.abs(got_v - v) <= ev + 1e-45).all()
        else:
            for got, x, rr, keep in ((got_m, m, rm, False), (np.sqrt(got_v), np.sqrt(v), ru, True)):
                want, unit = (a[: len(x)] for a in ref.quantise(pad(x), rr, keep))
                assert (np.abs(got - want) <= 1.01 * unit).all()
                flips += int((np.abs(got - want) > 1e-6 * unit).sum())
                total += len(x)
            assert ((got_v > 0) == (v > 0)).all()
        got = f64(p)
        if sr and p.dtype != torch.float32:
            up = r[: len(w)] / 65536.0 if p.dtype == torch.bfloat16 else (r[: len(w)] >> 3) / 8192.0
            want, unit = ref.cut(w, up, *MANT[p.dtype])
            assert (np.abs(got - want) <= ew + 1.01 * unit).all()
            flips += int((np.abs(got - want) > 1e-6 * unit).sum())
            total += len(w)
        else:
            sub = 2.0 ** -25 if p.dtype == torch.float16 else 0.0
            assert (np.abs(got - w) <= ew + UD[p.dtype] * np.abs(w) * 1.01 + sub).all()
    # fp32 is off by some 10 u of a value, 2^13 (fp16, 2^-13 draws) to 2^20 (e4m3) times less
    # than its spacing
    assert flips <= 5 + total / 100, (flips, total)


def snapshot(opt, ps):
    return [(f64(p).copy(), *moments(opt, p), opt.state[p].get("step", 0)) for p in ps]


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("sr", [True, False])
@pytest.mark.parametrize("wt", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("gt", [torch.bfloat16, torch.float16, torch.float32])
def test_steps(dev, bits, sr, wt, gt):
    ps, opt, g = make(dev, SIZES, wt, gt, seed=bits, state_bits=bits, stochastic_rounding=sr)
    for k in range(3):
        new_grads(ps, gt, g)
        before, seed = snapshot(opt, ps), opt.param_groups[0]["seed"]
        opt.step()
        check_step(opt, ps, before, seed)
        assert opt.param_groups[0]["seed"] == seed + 1


@pytest.mark.parametrize("bits", [32, 8])
def test_many_tensors_some_without_gradients(dev, bits):
    sizes = [1 + (37 * k) % 700 for k in range(150)]
    ps, opt, g = make(dev, sizes, torch.bfloat16, torch.bfloat16, state_bits=bits)
    for k in range(3):
        new_grads(ps, torch.bfloat16, g)
        for i in range(k, len(ps), 5):
            ps[i].grad = None
        if k == 2:
            ps[7].grad_dtype = torch.float32
            ps[7].grad = torch.randn(ps[7].shape, device=dev)
        before, seed = snapshot(opt, ps), opt.param_groups[0]["seed"]
        versions = [p._version for p in ps]
        opt.step()
        check_step(opt, ps, before, seed)
        for p, ver in zip(ps, versions):
            assert (p._version > ver) == (p.grad is not None)


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32])
def test_layouts_and_alignment(dev, bits, dt):
    """Views at odd starts, transposed parameters and gradients, negated gradients: the bits of
    the plain tensors' step, and nothing beside them written."""
    g = torch.Generator(device=dev).manual_seed(5)
    base = [(torch.randn(37, 53, generator=g, device=dev) * 0.1).to(dt) for _ in range(4)]
    grads = [torch.randn(37, 53, generator=g, device=dev).to(dt) for _ in range(4)]
    plain = [torch.nn.Parameter(b.clone()) for b in base]
    flat = torch.full((4 * 37 * 53 + 10,), 7.0, dtype=dt, device=dev)
    odd = []
    for k, b in enumerate(base):
        v = flat[1 + k * 37 * 53: 1 + (k + 1) * 37 * 53].view(37, 53)
        v.copy_(b)
        odd.append(v)
    t = base[3].t().contiguous().t()                 # not contiguous
    odd = [torch.nn.Parameter(v) for v in odd[:3]] + [torch.nn.Parameter(t)]
    assert not odd[3].is_contiguous()
    gflat = torch.empty(37 * 53 + 1, dtype=dt, device=dev)
    gflat[1:].copy_(grads[1].view(-1))
    ograds = [grads[0].t().contiguous().t(), gflat[1:].view(37, 53), torch._neg_view(-grads[2]), grads[3]]
    a, b = (AdamW(p, **HYPER, state_bits=bits) for p in (plain, odd))
    for _ in range(2):
        for p, q, x, y in zip(plain, odd, grads, ograds):
            p.grad, q.grad = x, y
        a.step()
        b.step()
        for p, q in zip(plain, odd):
            assert torch.equal(p, q)
    assert flat[0] == 7 and (flat[1 + 4 * 37 * 53:] == 7).all()


@pytest.mark.parametrize("bits", [32, 8])
def test_grad_scale(dev, bits):
    ps, opt, g = make(dev, SIZES, torch.bfloat16, torch.float32, state_bits=bits)
    for k, scale in enumerate((0.25, 3.0, 0.0)):
        new_grads(ps, torch.float32, g)
        before, seed = snapshot(opt, ps), opt.param_groups[0]["seed"]
        opt.step(grad_scale=torch.tensor([scale], device=dev))
        check_step(opt, ps, before, seed, factor=scale)
    kept = [p.detach().clone() for p in ps]
    states = [{k: v.clone() for k, v in opt.state[p].items() if k != "step"} for p in ps]
    opt.step(grad_scale=torch.full((), float("nan"), device=dev))
    for p, w, s in zip(ps, kept, states):
        assert torch.equal(p, w) and opt.state[p]["step"] == 4
        for k, v in s.items():
            assert torch.equal(v.view(torch.uint8), opt.state[p][k].view(torch.uint8)), k


@pytest.mark.parametrize("bits", [32, 8])
def test_zero_gradients_and_what_is_not_finite(dev, bits):
    ps, opt, g = make(dev, [1000], torch.bfloat16, torch.bfloat16, state_bits=bits, weight_decay=0.0)
    w0 = ps[0].detach().clone()
    ps[0].grad = torch.zeros_like(w0)
    opt.step()
    assert torch.equal(ps[0], w0) and not moments(opt, ps[0])[0].any()
    new_grads(ps, torch.bfloat16, g)
    other, clean = make(dev, [1000], torch.bfloat16, torch.bfloat16, state_bits=bits, weight_decay=0.0)[:2]
    with torch.no_grad():
        other[0].copy_(w0)
    other[0].grad = torch.zeros_like(w0)
    clean.step()
    other[0].grad = ps[0].grad.clone()
    at = torch.tensor([0, 5, 130, 131, 999], device=dev)
    ps[0].grad[at] = torch.tensor([float("nan"), float("inf"), -float("inf"), float("nan"), float("inf")],
                                  device=dev, dtype=torch.bfloat16)
    for o in (opt, clean):
        o.step()
    keep = torch.ones(1000, dtype=torch.bool, device=dev)
    keep[at] = False
    assert torch.isnan(ps[0][at]).all()
    if bits == 32:
        assert torch.equal(ps[0][keep], other[0][keep])
    m, v = moments(opt, ps[0])
    k = keep.cpu().numpy()
    assert np.isfinite(m[k]).all() and np.isfinite(v[k]).all() and not np.isfinite(m[~k]).any()
    # the other elements' states, up to the scale that the left-out maximum may have set
    if bits == 8:
        m2, v2 = moments(clean, other[0])
        assert (np.abs(m - m2)[k] <= 0.13 * np.abs(m2[k]) + 2.0 ** -9 * np.abs(m2).max()).all()
    new_grads(ps, torch.bfloat16, g)
    opt.step()                                     # such states stay, the others go on
    m, v = moments(opt, ps[0])
    assert np.isfinite(m[k]).all() and not np.isfinite(m[~k]).any()


def test_huge_gradients_overflow_to_their_own_element(dev):
    """g^2 past fp32: v is infinite, m is not; with 8 bits the root is NaN, m keeps its code."""
    ps, opt, g = make(dev, [256], torch.float32, torch.float32, state_bits=8)
    new_grads(ps, torch.float32, g)
    ps[0].grad[3] = 1e30
    opt.step()
    m, v = moments(opt, ps[0])
    assert np.isnan(v[3]) and np.isfinite(np.delete(v, 3)).all() and np.isfinite(m).all()


def test_small_roots_are_kept_above_zero(dev):
    """One large and many small gradients in a block: the small ones' roots, far under the
    codes' range, stay above zero, so that a later step does not divide by eps."""
    ps, opt, g = make(dev, [128], torch.float32, torch.float32, state_bits=8, weight_decay=0.0)
    ps[0].grad = torch.full((128,), 1e-7, device=dev)
    ps[0].grad[0] = 10.0
    opt.step()
    m, v = moments(opt, ps[0])
    assert (v > 0).all()
    w = ps[0].detach().clone()
    ps[0].grad = torch.zeros(128, device=dev)
    opt.step()
    assert (ps[0] - w).abs().max() < 3 * HYPER["lr"]


@pytest.mark.parametrize("bits", [32, 8])
def test_vanishing_gradients(dev, bits):
    """Gradients whose squares underflow: m / eps stays far below a weight's spacing."""
    ps, opt, _ = make(dev, [700], torch.float32, torch.float32, state_bits=bits, weight_decay=0.0)
    w = ps[0].detach().clone()
    ps[0].grad = torch.logspace(-44, -17, 700, device=dev)
    for _ in range(3):
        opt.step()
    assert torch.equal(ps[0], w)
    m, v = moments(opt, ps[0])
    assert np.isfinite(m).all() and np.isfinite(v).all()


@pytest.mark.parametrize("wt", [torch.bfloat16, torch.float16])
def test_rounding_is_unbiased(dev, wt):
    """Over 2000 seeds the mean of w' and of the 8-bit moments is the exact value: the mean's
    deviation is at most half a spacing / sqrt(2000) = 0.011; 6 of those."""
    n, K = 256, 2000
    g = torch.Generator(device=dev).manual_seed(1)
    w = (torch.randn(n, generator=g, device=dev) * 0.1).to(wt)
    grad = torch.randn(n, generator=g, device=dev) * 1e-2
    ps = [torch.nn.Parameter(w.clone()) for _ in range(K)]
    for p in ps:
        p.grad_dtype = torch.float32
        p.grad = grad
    opt = AdamW(ps, **HYPER, state_bits=8)
    opt.step()                                     # K streams of one seed
    w1, m1, v1 = ref.step(f64(w), f64(grad), np.zeros(n), np.zeros(n), 1, HYPER["lr"],
                          *HYPER["betas"], HYPER["eps"], HYPER["weight_decay"])
    _, unit = ref.cut(w1, 0.0, *MANT[wt])
    got = np.mean([f64(p) for p in ps], 0)
    assert (np.abs(got - w1) <= 0.07 * unit).all()
    for j, (x, keep) in enumerate(((m1, False), (np.sqrt(v1), True))):
        _, unit = ref.quantise(x, np.zeros(n), keep)
        got = np.mean([moments(opt, p)[j] if j == 0 else np.sqrt(moments(opt, p)[1]) for p in ps], 0)
        normal = np.abs(x) >= 2.0 ** -9 * np.abs(x).max()   # the smallest roots are kept up
        assert (np.abs(got - x) <= 0.07 * unit)[normal].all()


@pytest.mark.parametrize("bits", [32, 8])
def test_draws_round_the_exact_difference(dev, bits):
    """bf16 weights of 1/2 to 2 against draws added to the float64 result.  The change, 1e-6, is off
    by some 16 u of itself, 2^-32 of a weight's spacing: of 2^22 weights none in a thousand runs
    rounds the other way.  Were w - t first rounded to the nearest fp32, one in 2^18 would, some 16."""
    n = 1 << 22
    g = torch.Generator(device=dev).manual_seed(11)
    w = torch.rand(n, generator=g, device=dev) * 1.5 + 0.5
    w = torch.where(torch.rand(n, generator=g, device=dev) < 0.5, -w, w).bfloat16()
    p = torch.nn.Parameter(w)
    opt = AdamW([p], lr=1e-6, weight_decay=0.01, state_bits=bits, seed=77)
    p.grad = torch.randn(n, generator=g, device=dev, dtype=torch.bfloat16)
    w0, zero = f64(p).copy(), np.zeros(n)
    opt.step()
    want = ref.step(w0, f64(p.grad), zero, zero, 1, 1e-6, 0.9, 0.999, 1e-8, 0.01)[0]
    want, _ = ref.cut(want, ref.draws(np.arange(n), bits, 0, 77)[0] / 65536.0, *MANT[torch.bfloat16])
    assert (want != w0).any()
    assert (f64(p) != want).sum() <= 1


def test_against_torch_adamw(dev):
    """fp32, ten steps of the same gradients: both round each step's few operations."""
    g = torch.Generator(device=dev).manual_seed(2)
    ours = [torch.nn.Parameter(torch.randn(s, generator=g, device=dev)) for s in ((300, 70), (70,))]
    theirs = [torch.nn.Parameter(p.detach().clone()) for p in ours]
    a, b = AdamW(ours, **HYPER), torch.optim.AdamW(theirs, **HYPER)
    for _ in range(10):
        for p, q in zip(ours, theirs):
            p.grad = torch.randn(p.shape, generator=g, device=dev)
            q.grad = p.grad.clone()
        a.step()
        b.step()
    for p, q in zip(ours, theirs):
        assert (p - q).abs().max() <= 10 * (16 * U * 2 * HYPER["lr"] * 10 + 4 * U * p.abs().max())


@pytest.mark.parametrize("bits", [32, 8])
def test_checkpoint_resumes_bit_identically(dev, bits):
    ps, opt, g = make(dev, [500, 129], torch.bfloat16, torch.bfloat16, state_bits=bits)
    new_grads(ps, torch.bfloat16, g)
    opt.step()
    saved = copy.deepcopy(opt.state_dict())
    qs = [torch.nn.Parameter(p.detach().clone()) for p in ps]
    opt2 = AdamW(qs, lr=1.0, state_bits=bits, seed=9)
    opt2.load_state_dict(saved)
    for p, q in zip(ps, qs):
        for k, v in opt.state[p].items():
            if k != "step":
                assert opt2.state[q][k].dtype == v.dtype
    new_grads(ps, torch.bfloat16, g)
    for p, q in zip(ps, qs):
        q.grad = p.grad.clone()
    opt.step()
    opt2.step()
    for p, q in zip(ps, qs):
        assert torch.equal(p, q)
    other = AdamW([torch.nn.Parameter(p.detach().clone()) for p in ps], state_bits=40 - bits)
    saved["param_groups"][0]["state_bits"] = 40 - bits
    with pytest.raises(ValueError, match="does not fit"):
        other.load_state_dict(saved)


def test_eight_bit_states_train_like_32(dev):
    """A regression with bf16 weights: the loss falls as far as with torch's AdamW on fp32
    weights, and with 8-bit states as far as with 32."""
    def train(dt, make):
        g = torch.Generator(device=dev).manual_seed(4)
        x = torch.randn(2048, 256, generator=g, device=dev)
        y = x @ torch.randn(256, 32, generator=g, device=dev)
        w = torch.nn.Parameter(torch.zeros(256, 32, device=dev, dtype=dt))
        opt = make([w], lr=2e-2, weight_decay=0.0)
        for k in range(400):
            opt.param_groups[0]["lr"] = 2e-2 * (1 - k / 400)
            loss = (x @ w.float() - y).square().mean()
            opt.zero_grad()
            loss.backward()
            if make is torch.optim.AdamW:
                torch.nn.utils.clip_grad_norm_([w], 10.0)
                opt.step()
            else:
                opt.step(grad_scale=grad_norm([w.grad], 10.0)[1])
        return float(loss.detach())
    start, lt = 256.0, train(torch.float32, torch.optim.AdamW)
    l32, l8 = (train(torch.bfloat16, lambda p, **kw: AdamW(p, state_bits=b, **kw)) for b in (32, 8))
    assert l32 < 2 * lt + 1e-3 * start and l8 < 2 * l32 + 1e-3 * start


def test_offsets_past_2_31_elements(dev):
    n = 2 ** 31 + 2 ** 20 + 77
    p = torch.nn.Parameter(torch.full((n,), 0.5, dtype=torch.bfloat16, device=dev))
    p.grad = torch.full((n,), 1e-3, dtype=torch.bfloat16, device=dev)
    tail = 4173
    g = torch.Generator(device=dev).manual_seed(8)
    p.grad[-tail:] = (torch.randn(tail, generator=g, device=dev) * 1e-2).to(torch.bfloat16)
    opt = AdamW([p], **HYPER, state_bits=8)
    opt.step()
    w, m, v = ref.step(np.full(tail, 0.5), f64(p.grad[-tail:]), np.zeros(tail), np.zeros(tail), 1,
                       HYPER["lr"], *HYPER["betas"], HYPER["eps"], HYPER["weight_decay"])
    r, rm, ru = ref.draws(np.arange(n - tail, n), 8, 0, 123)
    want, unit = ref.cut(w, r / 65536.0, 7, -126)
    got = f64(p[-tail:])
    assert (np.abs(got - want) <= 1.01 * unit).all() and (got != want).mean() < 0.01
    s = opt.state[p]
    blocks = -(-n // 128)
    first = (n - tail + 127) // 128                # whole blocks of the tail
    scale = f64(s["exp_avg_scale"][first:])
    codes = f64(s["exp_avg"][first * 128:]) * np.repeat(scale, 128)
    off = first * 128 - (n - tail)
    want, unit = ref.quantise(pad(m[off:]), np.concatenate([rm[off:], np.zeros(blocks * 128 - n, int)]), False)
    assert (np.abs(codes - want) <= 1.01 * unit).all() and (codes != want).mean() < 0.01
    norm, _ = grad_norm([p.grad])
    exact = ((n - tail) * float(p.grad[0]) ** 2 + float((f64(p.grad[-tail:]) ** 2).sum())) ** 0.5
    assert abs(float(norm) - exact) <= 1e-5 * exact


# ------------------------------------------------------------- grad_norm ----
@pytest.mark.parametrize("sizes", [[1], [7, 0, 300], [16384, 16385, 5], [3] * 200, [1 << 22, 77]])
@pytest.mark.parametrize("dts", [(torch.bfloat16,), (torch.float32,),
                                 (torch.float16, torch.float32, torch.bfloat16)])
def test_norm(dev, sizes, dts):
    """Each thread's fp32 sum has at most a few hundred additions; the norm is half as far off."""
    g = torch.Generator(device=dev).manual_seed(len(sizes))
    ts = [torch.randn(n + 1, generator=g, device=dev).to(dts[k % len(dts)])[1:] for k, n in enumerate(sizes)]
    before = [t.clone() for t in ts]
    exact = sum(float(t.double().square().sum()) for t in ts) ** 0.5
    for max_norm in (exact / 2, exact * 2, float("inf"), 0.0):
        norm, coef = grad_norm(ts, max_norm)
        assert abs(float(norm) - exact) <= 1e-5 * exact and norm.shape == coef.shape == ()
        want = min(1.0, max_norm / (exact + 1e-6))
        assert abs(float(coef) - want) <= 2e-5 * want
    a, b = grad_norm(ts, 1.0), grad_norm(ts, 1.0)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    for t, u in zip(ts, before):
        assert torch.equal(t, u)


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_norm_that_is_not_finite_skips_the_step(dev, bad):
    ps, opt, g = make(dev, [300, 20], torch.bfloat16, torch.bfloat16, state_bits=8)
    new_grads(ps, torch.bfloat16, g)
    ps[1].grad[3] = bad
    kept = [p.detach().clone() for p in ps]
    norm, coef = grad_norm([p.grad for p in ps], 1.0)
    assert not torch.isfinite(norm) and torch.isnan(coef)
    opt.step(grad_scale=coef)
    for p, w in zip(ps, kept):
        assert torch.equal(p, w)


def test_norm_layouts(dev):
    t = torch.randn(60, 40, device=dev)
    want = grad_norm([t])[0]
    for v in (t.t(), torch._neg_view(t)):
        assert abs(float(grad_norm([v])[0] - want)) <= 1e-5 * float(want)
    wide = torch.randn(60, 80, device=dev)
    assert abs(float(grad_norm([wide[:, ::2]])[0]) - float(wide[:, ::2].double().norm())) < 1e-3
    assert float(grad_norm([torch.zeros(0, device=dev)])[0]) == 0.0


def test_clipped_step_is_that_of_clipped_gradients(dev):
    ps, opt, g = make(dev, SIZES, torch.float32, torch.float32)
    new_grads(ps, torch.float32, g, gscale=1.0)
    norm, coef = grad_norm([p.grad for p in ps], 1.0)
    before, seed = snapshot(opt, ps), opt.param_groups[0]["seed"]
    opt.step(grad_scale=coef)
    check_step(opt, ps, before, seed, factor=float(coef))


# ------------------------------------------------- the optimizer's manners ----
def test_hooks_closure_and_groups(dev):
    calls = []
    a, b = (torch.nn.Parameter(torch.ones(10, device=dev)) for _ in range(2))
    opt = AdamW([dict(params=[a], lr=0.1), dict(params=[b], state_bits=8, seed=5)], lr=0.01)
    opt.register_step_pre_hook(lambda o, args, kw: calls.append(("pre", sorted(kw))))
    opt.register_step_post_hook(lambda o, args, kw: calls.append("post"))

    def closure():
        calls.append(torch.is_grad_enabled())
        a.grad, b.grad = torch.ones_like(a), torch.ones_like(b)
        return 3.5
    assert opt.step(closure, grad_scale=torch.ones(1, device=dev)) == 3.5
    assert calls == [("pre", ["grad_scale"]), True, "post"]
    assert set(opt.state[a]) == {"step", "exp_avg", "exp_avg_sq"}
    assert set(opt.state[b]) == {"step", "exp_avg", "rms", "exp_avg_scale", "rms_scale"}
    assert abs(float(a[0]) - 0.9 * 1.0) < 2e-3 and abs(float(b[0]) - 0.99) < 2e-3


@pytest.mark.parametrize("bits", [32, 8])
def test_empty_parameters_schedulers_and_saved_files(dev, bits, tmp_path):
    a = torch.nn.Parameter(torch.ones(300, device=dev, dtype=torch.bfloat16))
    b = torch.nn.Parameter(torch.ones(0, 4, device=dev, dtype=torch.bfloat16))
    opt = AdamW([a, b], lr=1e-2, state_bits=bits)
    sched = torch.optim.lr_scheduler.LambdaLR(opt, lambda k: 0.5 ** k)
    for _ in range(2):
        a.grad, b.grad = torch.ones_like(a), torch.ones_like(b)
        norm, coef = grad_norm([a.grad, b.grad], 1.0)
        opt.step(grad_scale=coef)
        sched.step()
    assert opt.state[b]["step"] == 2 and abs(opt.param_groups[0]["lr"] - 2.5e-3) < 1e-9
    torch.save(opt.state_dict(), tmp_path / "opt.pt")
    c = torch.nn.Parameter(a.detach().clone())
    opt2 = AdamW([c, torch.nn.Parameter(b.detach().clone())], state_bits=bits)
    opt2.load_state_dict(torch.load(tmp_path / "opt.pt", weights_only=True))
    for o, p in ((opt, a), (opt2, c)):
        p.grad = torch.full_like(p, 0.3)
        o.step()
    assert torch.equal(a, c) and opt2.param_groups[0]["seed"] == opt.param_groups[0]["seed"]


def test_other_stream_than_the_tensors_own(dev):
    ps, opt, g = make(dev, [100000], torch.bfloat16, torch.bfloat16, state_bits=8)
    qs, opt2, _ = make(dev, [100000], torch.bfloat16, torch.bfloat16, state_bits=8)
    new_grads(ps, torch.bfloat16, g)
    qs[0].grad = ps[0].grad.clone()
    s = torch.cuda.Stream(dev)
    s.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(s):
        opt2.step(grad_scale=grad_norm([qs[0].grad], 1.0)[1])
    torch.cuda.current_stream(dev).wait_stream(s)
    opt.step(grad_scale=grad_norm([ps[0].grad], 1.0)[1])
    assert torch.equal(ps[0], qs[0])


def test_refusals(dev):
    p = torch.nn.Parameter(torch.ones(4, device=dev))
    opt = AdamW([p])
    p.grad = torch.ones_like(p)
    for bad in (torch.ones(2, device=dev), torch.ones(1), torch.ones(1, device=dev, dtype=torch.float64)):
        with pytest.raises(RuntimeError):
            opt.step(grad_scale=bad)
    opt.step()
    opt.state[p]["exp_avg"] = torch.zeros(3, device=dev)
    with pytest.raises(RuntimeError, match="does not fit"):
        opt.step()
    q = torch.nn.Parameter(torch.ones(4, device=dev, dtype=torch.float64))
    q.grad = torch.ones_like(q)
    with pytest.raises(RuntimeError, match="unsupported dtype"):
        AdamW([q]).step()
    r = torch.nn.Parameter(torch.ones(4, 2, device=dev))
    r.grad = torch.ones(4, 2, device=dev).to_sparse()
    with pytest.raises(RuntimeError, match="dense"):
        AdamW([r]).step()
    with pytest.raises(RuntimeError, match="no tensors"):
        grad_norm([])
    with pytest.raises(RuntimeError, match="HIP device"):
        grad_norm([torch.ones(3)])
    with pytest.raises(RuntimeError, match="max_norm"):
        grad_norm([p.grad], -1.0)
    w = torch.nn.Parameter(torch.ones(4, device=dev))
    w.grad = torch.ones_like(w)
    opt = AdamW([w])
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match="captured"):
        with torch.cuda.graph(graph):
            opt.step()
    opt.step()
