"""GPU: calls of AdamW and of the gradients' norm whose answers the other tests do not reach."""
import numpy as np
import pytest
import torch

import adamw_reference as ref
from haste_amd.optim_adamw import AdamW, grad_norm

pytestmark = pytest.mark.gpu
INF = float("inf")


def counts(opt, ps):
    return [(opt.state[p].get("step"), p._version, p.detach().clone()) for p in ps], \
        [g["seed"] for g in opt.param_groups]


def unchanged(opt, ps, before):
    now = counts(opt, ps)
    assert now[1] == before[1]
    for a, b in zip(now[0], before[0]):
        assert a[:2] == b[:2] and torch.equal(a[2], b[2])


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("plain", [True, False])
def test_a_refused_step_moves_no_count(dev, bits, plain):
    """Settings that the library refuses, for parameters of either path: the count of steps, the
    version and the seed stay, and the step after it is that of an optimizer that was never refused."""
    def make():
        w = torch.arange(600, device=dev, dtype=torch.bfloat16).view(20, 30) / 600
        p = torch.nn.Parameter(w if plain else w.t())
        p.grad = torch.ones_like(p) if plain else torch.ones(20, 30, device=dev, dtype=p.dtype).t()
        opt = AdamW([p], lr=1e-2, state_bits=bits)
        opt.step()
        return p, opt
    (p, opt), (q, other) = make(), make()
    before = counts(opt, [p])
    opt.param_groups[0]["betas"] = (1.5, 0.9)
    for _ in range(3):
        with pytest.raises(RuntimeError, match="betas"):
            opt.step()
        unchanged(opt, [p], before)
    opt.param_groups[0]["betas"] = (0.9, 0.999)
    opt.step()
    other.step()
    assert torch.equal(p, q) and opt.state[p]["step"] == 2


def test_a_refused_tensor_stops_the_others_of_its_group(dev):
    """States that start off 16 bytes (views of an unpadded buffer) are refused before any tensor of
    the group is stepped, whatever its dtypes."""
    ps = [torch.nn.Parameter(torch.ones(64, device=dev, dtype=d)) for d in (torch.bfloat16, torch.float32)]
    opt = AdamW(ps, lr=1e-2)
    for p in ps:
        p.grad = torch.ones_like(p)
    opt.step()
    flat = torch.zeros(65, device=dev)
    good = opt.state[ps[1]]["exp_avg"]
    opt.state[ps[1]]["exp_avg"] = flat[1:]
    before = counts(opt, ps)
    for _ in range(2):
        with pytest.raises(RuntimeError, match="exp_avg .*16 bytes"):
            opt.step()
        unchanged(opt, ps, before)
    opt.state[ps[1]]["exp_avg"] = good
    opt.step()
    assert [opt.state[p]["step"] for p in ps] == [2, 2]


@pytest.mark.skipif(torch.cuda.device_count() < 2, reason="needs two devices")
@pytest.mark.parametrize("bits", [32, 8])
def test_steps_on_a_device_that_is_not_the_current_one(dev, bits):
    ps = [torch.nn.Parameter(torch.linspace(-1, 1, 5000, device=f"cuda:{k}")) for k in (0, 1)]
    for p in ps:
        opt = AdamW([p], lr=1e-2, state_bits=bits)
        for _ in range(2):
            p.grad = torch.cos(p.detach() * 7)
            opt.step(grad_scale=grad_norm([p.grad.view(50, 100).t()], 1.0)[1])
    assert torch.equal(ps[0].cpu(), ps[1].cpu())


@pytest.mark.parametrize("wt", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("bits", [32, 8])
def test_a_negated_grad_scale(dev, wt, bits):
    """A lazily negated factor counts with its sign, for plain parameters and for others."""
    scale = torch.full((1,), 0.5, device=dev)
    for shape in ((40, 30), (30, 40)):
        w = torch.randn(40, 30, device=dev).to(wt)
        grad = torch.randn(40, 30, device=dev).to(wt)
        got = []
        for s in (-scale, torch._neg_view(scale)):
            p = torch.nn.Parameter(w.clone() if shape == (40, 30) else w.clone().t())
            opt = AdamW([p], lr=1e-2, state_bits=bits)
            for _ in range(2):
                p.grad = grad.clone() if shape == (40, 30) else grad.t()
                opt.step(grad_scale=s)
            got.append(p.detach().clone())
        assert torch.equal(*got)


def test_a_negated_state_is_refused(dev):
    p = torch.nn.Parameter(torch.ones(64, device=dev))
    opt = AdamW([p])
    for _ in range(2):
        p.grad = torch.ones_like(p)
        opt.step()
        kept = p.detach().clone()
        opt.state[p]["exp_avg"] = torch._neg_view(opt.state[p]["exp_avg"])
        with pytest.raises(RuntimeError, match="does not fit"):
            opt.step()
        assert torch.equal(p, kept)
        opt.state[p]["exp_avg"] = torch._neg_view(opt.state[p]["exp_avg"])


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("sr", [True, False])
@pytest.mark.parametrize("wt", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("wd", [0.0, 0.1])
def test_infinite_weights_stay_so(dev, bits, sr, wt, wd):
    """w (1 - lr wd) less a finite update; NaN stays NaN, and their neighbours are not touched."""
    g = torch.Generator(device=dev).manual_seed(3)
    w = (torch.randn(300, generator=g, device=dev) * 0.1).to(wt)
    grad = torch.randn(300, generator=g, device=dev).to(wt)
    a, b = (torch.nn.Parameter(w.clone()) for _ in range(2))
    at = torch.tensor([0, 17, 130, 299], device=dev)
    with torch.no_grad():
        a[at] = torch.tensor([INF, -INF, float("nan"), INF], device=dev, dtype=wt)
    for p in (a, b):
        opt = AdamW([p], lr=1e-2, weight_decay=wd, state_bits=bits, stochastic_rounding=sr)
        for _ in range(2):
            p.grad = grad
            opt.step()
    got = a.detach()[at].float().cpu().numpy()
    assert np.array_equal(got, np.float32([INF, -INF, np.nan, INF]), equal_nan=True)
    keep = torch.ones(300, dtype=torch.bool, device=dev)
    keep[at] = False
    assert torch.equal(a[keep], b[keep])


@pytest.mark.parametrize("value", [1e-22, 1e-30, 3e-19, 4e18, 1.7e19, 3e38])
@pytest.mark.parametrize("n", [1, 64, 20000, 70000])
@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
def test_norms_whose_squares_leave_fp32(dev, value, n, dt):
    """The norm of n equal gradients is |g| sqrt(n), here below fp32's largest value unless that
    is passed: squares from 1e-60 to 9e76 are sums of fp64, off by a few 1e-16, and the rest by
    fp32's sums of 64 squares and the norm's own rounding, under 70 2^-24."""
    t = torch.full((n,), value, device=dev).to(dt)
    t[::3] *= -1
    exact = float(t[0].double().abs()) * n ** 0.5
    norm, coef = grad_norm([t, torch.zeros(5000, device=dev)], 1.0)
    if exact > 3.4028235e38:
        assert float(norm) == INF and bool(torch.isnan(coef))
        return
    assert abs(float(norm) - exact) <= 70 * 2.0 ** -24 * exact
    want = min(1.0, 1.0 / (exact + 1e-6))
    assert abs(float(coef) - want) <= 80 * 2.0 ** -24 * want


def test_norms_of_small_beside_large(dev):
    """One workgroup's share of each kind: what is small is not lost and not counted twice."""
    small, large = torch.full((40000,), 1e-22, device=dev), torch.full((40000,), 2e-22, device=dev)
    zero = torch.zeros(40000, device=dev)
    exact = (40000 * (float(small[0].double()) ** 2 + float(large[0].double()) ** 2)) ** 0.5
    norm, _ = grad_norm([small, zero, -zero, large])
    assert abs(float(norm) - exact) <= 70 * 2.0 ** -24 * exact
    one = torch.ones(1, device=dev)
    assert float(grad_norm([small, one])[0]) == 1.0
    bad = small.clone()
    bad[777] = float("nan")
    assert bool(torch.isnan(grad_norm([bad, one])[0]))
    assert float(grad_norm([zero])[0]) == 0.0


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("plain", [True, False])
def test_groups_draw_for_themselves(dev, bits, plain):
    """The same 4000 weights and gradients twice in one group and in two others of its seed: no two
    are rounded by the same draws."""
    g = torch.Generator(device=dev).manual_seed(6)
    w = torch.randn(40, 100, generator=g, device=dev).to(torch.bfloat16)
    grad = torch.randn(40, 100, generator=g, device=dev).to(torch.bfloat16)
    ps = [torch.nn.Parameter(w.clone() if plain else w.t().contiguous().t()) for _ in range(4)]
    opt = AdamW([dict(params=ps[:2]), dict(params=ps[2:3]), dict(params=ps[3:])], lr=1e-3, state_bits=bits)
    for k in range(2):
        for p in ps:
            p.grad = grad.clone()
        opt.step()
        for i in range(4):
            for j in range(i):
                assert not torch.equal(ps[i], ps[j]), (k, i, j)


def test_2_35_elements(dev):
    """More than the 2^32 threads of one launch, 8 elements to each: the weights where the second
    launch begins and at the end.  (Gradients are the weights' own memory, to have room.)"""
    n = 2 ** 35 + 4173
    torch.cuda.empty_cache()
    if torch.cuda.mem_get_info(dev)[0] < 160 * 2 ** 30:
        pytest.skip("needs 160 GiB")
    p = torch.nn.Parameter(torch.full((n,), 0.5, dtype=torch.bfloat16, device=dev))
    p.grad = p.detach()
    opt = AdamW([p], lr=1e-2, state_bits=8, seed=31)
    opt.step()
    zero = np.zeros(6000)
    for at in (0, (2 ** 24 - 1) * 2048 - 3000, n - 6000):
        w = ref.step(zero + 0.5, zero + 0.5, zero, zero, 1, 1e-2, 0.9, 0.999, 1e-8, 0.01)[0]
        i = np.arange(at, at + 6000)
        want, unit = ref.cut(w, ref.draws(i, 8, 0, 31)[0] / 65536.0, 7, -126)
        got = p.detach()[at: at + 6000].double().cpu().numpy()
        # fp32 is off by some 20 u of the change, 2^-16 of a spacing: a draw in 2^16 at most differs
        assert (np.abs(got - want) <= 1.01 * unit).all() and (got != want).sum() <= 6, at
    codes = opt.state[p]["exp_avg"].view(torch.uint8)
    assert all((c != 0).all() for c in (codes[:n][-10 ** 6:], codes[: 10 ** 6])) and not codes[n:].any()
    del p.grad
