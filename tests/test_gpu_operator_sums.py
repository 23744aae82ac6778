"""GPU: layer norm's sums over rows where they are exact, and the codes of 8-bit AdamW states
against their own draws: a row or a draw too many or too few shows as such."""
import numpy as np
import pytest
import torch

import adamw_reference as ref
from haste_amd import _lib
from haste_amd.optim_adamw import AdamW
from test_gpu_layer_norm import UD, U

pytestmark = pytest.mark.gpu
CODE = {torch.bfloat16: _lib.DTYPE_BF16, torch.float16: _lib.DTYPE_F16, torch.float32: _lib.DTYPE_F32}


# (rows of 768 in 16 bits: 8192 a turn of all workgroups; 24: 65,536; 1537: 2048; 4096 and up: 512)
@pytest.mark.parametrize("N,D", [
    (N, D) for N in (1, 511, 513, 1025, 2049, 8191, 8192, 8193, 16385, 20011, 65537)
    for D in (5, 24, 768, 1537, 4096, 12000, 20000) if N * D <= 2 ** 25])
@pytest.mark.parametrize("dt", list(CODE))
def test_row_sums_that_are_exact(dev, N, D, dt):
    """Rows of -1 and 1, dy of -2 to 2, weights of 1, mean 0 and rstd 1 given: dw and db are whole
    numbers below 2^24, and dx = a - c1 - n c2 + dh is off by its roundings."""
    g = torch.Generator(device=dev).manual_seed(N + D)
    h = (torch.randint(0, 2, (N, D), generator=g, device=dev) * 2 - 1).to(dt)
    dy = torch.randint(-2, 3, (N, D), generator=g, device=dev).to(dt)
    dh = torch.randint(-2, 3, (N, D), generator=g, device=dev).to(dt) if N % 2 else None
    w = torch.ones(D, device=dev)
    stats = torch.tensor([0.0, 1.0], device=dev).repeat(N, 1)
    dx, dw, db = torch.empty_like(h), torch.empty_like(w), torch.empty_like(w)
    size = _lib.lib().haste_layer_norm_bwd_workspace_size(N, D)
    ws = torch.empty(size, dtype=torch.uint8, device=dev)
    _lib.call("haste_layer_norm_bwd", dy.data_ptr(), D, None if dh is None else dh.data_ptr(), D,
              h.data_ptr(), D, w.data_ptr(), stats.data_ptr(), dx.data_ptr(), dw.data_ptr(),
              db.data_ptr(), ws.data_ptr(), size, N, D, CODE[dt], _lib.DTYPE_F32,
              torch.cuda.current_stream(dev).cuda_stream)
    assert torch.equal(db, dy.float().sum(0)) and torch.equal(dw, (dy.float() * h.float()).sum(0))
    a, n = dy.double(), h.double()
    want = a - a.mean(1, keepdim=True) - n * (a * n).mean(1, keepdim=True)
    if dh is not None:
        want += dh.double()
    assert ((dx.double() - want).abs() <= UD[dt] * want.abs() + 16 * U).all()


def test_codes_are_rounded_by_their_draws(dev):
    """Three steps of 2^20 weights.  m is off by 3 u (|b1 m| + |c1 g|) and u by 4 u of itself (three
    roundings of v halved, the root's 1 ulp), so a code may go the other way where what is cut off
    is that close to its draw: over all elements as many as these errors in units of the codes'
    spacing, twice (both sides of the draw); four times that and 20 are not passed by chance."""
    n = 1 << 20
    u24 = 2.0 ** -24
    g = torch.Generator(device=dev).manual_seed(21)
    p = torch.nn.Parameter(torch.randn(n, generator=g, device=dev))
    opt = AdamW([p], lr=1e-3, betas=(0.9, 0.99), state_bits=8, seed=5)
    m = v = np.zeros(n)
    for t in range(3):
        spread = torch.exp(2 * torch.randn(n, generator=g, device=dev))
        p.grad = torch.randn(n, generator=g, device=dev) * spread
        grad = p.grad.double().cpu().numpy()
        opt.step()
        _, rm, ru = ref.draws(np.arange(n), 8, 0, 5 + t)
        err_m = 3 * u24 * (0.9 * np.abs(m) + 0.1 * np.abs(grad))
        m, v = 0.9 * m + 0.1 * grad, 0.99 * v + 0.01 * grad * grad
        held = []
        for x, err, r, keep, key in ((m, err_m, rm, False, "exp_avg"),
                                     (np.sqrt(v), 4 * u24 * np.sqrt(v), ru, True, "rms")):
            want, unit = ref.quantise(x, r, keep)
            scale = opt.state[p][key + "_scale"].double().cpu().numpy()
            top = np.abs(x).reshape(-1, ref.BLOCK).max(1)
            assert np.array_equal(scale, np.exp2(ref.scale_exponent(top).astype(np.float64)))
            got = opt.state[p][key].double().cpu().numpy() * np.repeat(scale, ref.BLOCK)
            flips, chance = int((got != want).sum()), float((2 * err / unit).sum())
            assert (np.abs(got - want) <= 1.01 * unit).all() and flips <= 20 + 4 * chance, (flips, chance)
            held.append(got)
        m, v = held[0], held[1] ** 2
