"""GPU: calls of layer norm that could end in a wrong answer without an error."""
import pytest
import torch
import torch.autograd.forward_ad as fwAD

from haste_amd import _lib, ops
from test_gpu_layer_norm import U, UD, close, data, reference, run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("which", ["x", "weight", "bias", "residual"])
@pytest.mark.parametrize("grad", [False, True])
def test_forward_mode_is_refused(dev, which, grad):
    """A tangent that the kernels would drop, with and without a backward to record."""
    t = {k: torch.randn(s, device=dev) for k, s in
         dict(x=(4, 64), weight=(64,), bias=(64,), residual=(4, 64)).items()}
    if grad:
        t["x" if which != "x" else "weight"].requires_grad_(True)
    with fwAD.dual_level():
        t[which] = fwAD.make_dual(t[which], torch.ones_like(t[which]))
        with pytest.raises(NotImplementedError, match="forward-mode"):
            ops.layer_norm(t["x"], t["weight"], t["bias"], residual=t["residual"])


def free_gib(dev):
    torch.cuda.empty_cache()
    return torch.cuda.mem_get_info(dev)[0] / 2 ** 30


@pytest.mark.parametrize("dt,D", [(torch.bfloat16, 4), (torch.float32, 3)])
def test_2_24_narrow_rows(dev, dt, D):
    """Rows of a workgroup each, past the 2^32 threads of one launch.  dy of -1, 0 and 1: db is a whole
    number, of which every partial sum is exact."""
    N = 2 ** 24 + 3
    if free_gib(dev) < 32:
        pytest.skip("needs 32 GiB")
    dat = data(N, D, dt, torch.float32, dev, seed=1)
    dat["dy"] = torch.randint(-1, 2, (N, D), device=dev).to(dt)
    got = run(dat)
    want, tol = reference(dat["x"], dat["w"], dat["b"], dat["dy"])
    for k in ("y", "dx"):
        close(k, got[k], want[k], tol[k])
    assert torch.equal(got["db"].double(), want["db"])
    # dw: 16,384 rows to a thread one after another, then some 100 sums
    terms = ((got["y"].double() - dat["b"].double()) / dat["w"].double() * dat["dy"].double()).abs().sum(0)
    assert ((got["dw"].double() - want["dw"]).abs() <= (N / 1024 + 200) * U * terms).all()


def test_2_32_threads_of_rows_in_registers(dev):
    """2^28 rows of 65, 16 threads to each: all are one row, read where it lies."""
    N, D = 2 ** 28 + 5, 65
    if free_gib(dev) < 48:
        pytest.skip("needs 48 GiB")
    x = torch.randn(1, D, device=dev).to(torch.bfloat16)
    w = torch.randn(D, device=dev).to(torch.bfloat16)
    want = ops.layer_norm(x, w)
    y = ops.layer_norm(x.expand(N, D), w)
    for part in y.split(2 ** 25):
        assert (part == want).all()


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32])
def test_rows_of_2_28_elements(dev, dt):
    """dw and db over more columns than a launch has threads for.  Rows of -1 and 1 with mean 0 and
    rstd 1 given, dy of -2 to 2 and weights of 1: all sums are exact, and dx = a - c1 - n c2 is off
    by its three roundings and its own."""
    N, D = 2, 2 ** 28 + 7
    if free_gib(dev) < 48:
        pytest.skip("needs 48 GiB")
    g = torch.Generator(device=dev).manual_seed(2)
    h = (torch.randint(0, 2, (N, D), generator=g, device=dev, dtype=torch.int8) * 2 - 1).to(dt)
    dy = torch.randint(-2, 3, (N, D), generator=g, device=dev, dtype=torch.int8).to(dt)
    w = torch.ones(D, device=dev)
    stats = torch.tensor([[0.0, 1.0]] * N, device=dev)
    dx, dw, db = torch.empty_like(h), torch.empty_like(w), torch.empty_like(w)
    size = _lib.lib().haste_layer_norm_bwd_workspace_size(N, D)
    ws = torch.empty(size, dtype=torch.uint8, device=dev)
    p = [t.data_ptr() for t in (dy, h, w, stats, dx, dw, db, ws)]
    _lib.call("haste_layer_norm_bwd", p[0], D, None, 0, p[1], D, p[2], p[3], p[4], p[5], p[6], p[7], size,
              N, D, _lib.DTYPE_BF16 if dt is torch.bfloat16 else _lib.DTYPE_F32, _lib.DTYPE_F32,
              torch.cuda.current_stream(dev).cuda_stream)
    assert torch.equal(db, dy.float().sum(0)) and torch.equal(dw, (dy.float() * h.float()).sum(0))
    for r in range(N):
        a, n = dy[r].double(), h[r].double()
        want = a - a.mean() - n * (a * n).mean()
        assert ((dx[r].double() - want).abs() <= UD[dt] * want.abs() + 8 * U).all()
