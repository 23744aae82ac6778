"""CPU: the argument checks of layer norm, AdamW and the gradients' norm (they return before any
HIP call), and the reference's random bits against published vectors."""
import numpy as np
import pytest
import torch

import adamw_reference as ref
from haste_amd import _lib, ops
from haste_amd.layer_norm import LayerNorm
from haste_amd.optim_adamw import AdamW, grad_norm

OK, BAD, WS = _lib.HASTE_OK, _lib.HASTE_ERR_INVALID_ARG, _lib.HASTE_ERR_WORKSPACE
BF16, F16, F32 = _lib.DTYPE_BF16, _lib.DTYPE_F16, _lib.DTYPE_F32


def test_philox_known_answers():
    """Random123's known answers of Philox4x32-10 for counter and key of zeros."""
    assert ref.philox([0], 0, 0, 0)[0].tolist() == [0x6627e8d5, 0xe169c58d, 0xbc57ac4c, 0x9b00dbd8]


def test_reference_rounds_up_by_its_draw():
    x = np.array([1.0 + 2 ** -8, -(1.0 + 2 ** -8), 0.0])
    assert ref.cut(x, 0.49, 7, -126)[0].tolist() == [1.0, -1.0, 0.0]
    assert ref.cut(x, 0.51, 7, -126)[0].tolist() == [1.0 + 2 ** -7, -(1.0 + 2 ** -7), 0.0]


def _ln(**kw):
    a = dict(x=64, ldx=768, res=None, ldres=0, w=128, b=None, y=192, h=None, stats=None, N=4, D=768,
             eps=1e-5, dtype=BF16, w_dtype=BF16, stream=None)
    return _lib.lib().haste_layer_norm(*(a | kw).values())


@pytest.mark.parametrize("kw,word", [
    (dict(N=-1), "sizes"), (dict(D=0), "sizes"), (dict(eps=-1.0), "eps"),
    (dict(eps=float("nan")), "eps"), (dict(dtype=7), "rows must be"),
    (dict(w_dtype=F16), "weights must be"), (dict(x=None), "x is NULL"), (dict(x=65), "aligned"),
    (dict(ldx=700), "row pitch"), (dict(ldx=-768), "row pitch"), (dict(w=None), "w is NULL"),
    (dict(y=None), "y is NULL"), (dict(res=256, ldres=768), "h is NULL"),
    (dict(w_dtype=F32, w=130), "aligned"), (dict(b=129), "aligned"), (dict(D=1 << 31), "too large"),
    (dict(stats=130), "stats")])
def test_layer_norm_rejects(kw, word):
    assert _ln(**kw) == BAD and word in _lib.last_error()


def _lnb(**kw):
    a = dict(dy=64, lddy=768, dh=None, lddh=0, h=128, ldh=768, w=192, stats=256, dx=320, dw=384,
             db=448, ws=512, ws_bytes=1 << 30, N=4, D=768, dtype=BF16, w_dtype=BF16, stream=None)
    return _lib.lib().haste_layer_norm_bwd(*(a | kw).values())


@pytest.mark.parametrize("kw,rc,word", [
    (dict(N=-1), BAD, "sizes"), (dict(D=0), BAD, "sizes"), (dict(dy=None), BAD, "dy is NULL"),
    (dict(h=None), BAD, "h is NULL"), (dict(stats=None), BAD, "stats"), (dict(lddy=5), BAD, "pitch"),
    (dict(dh=64, lddh=5), BAD, "pitch"), (dict(dx=321), BAD, "aligned"), (dict(dw=385), BAD, "aligned"),
    (dict(ws=None), BAD, "workspace"), (dict(ws=520), BAD, "workspace"), (dict(ws_bytes=0), WS, "too small"),
    (dict(dtype=9), BAD, "rows must be"), (dict(w_dtype=F16), BAD, "weights must be")])
def test_layer_norm_bwd_rejects(kw, rc, word):
    assert _lnb(**kw) == rc and word in _lib.last_error()


def test_layer_norm_workspace_size():
    f = _lib.lib().haste_layer_norm_bwd_workspace_size
    assert f(-1, 8) < 0 and f(8, -1) < 0
    for N, D in ((0, 1), (1, 1), (256, 4096), (10 ** 9, 768), (5, 10 ** 8)):
        assert 0 < f(N, D) < 2 ** 40


def _adamw(ts, **kw):
    a = dict(w_dtype=BF16, g_dtype=BF16, bits=8, lr=1e-3, b1=0.9, b2=0.999, eps=1e-8, wd=0.0, step=1,
             sr=1, seed=1, scale=None, stream=None)
    arr = (_lib.AdamwTensor * max(1, len(ts)))(*ts)
    return _lib.lib().haste_adamw_step(arr, len(ts), *(a | kw).values())


GOOD = (64, 128, 192, 256, 320, 384, 10, 0)


@pytest.mark.parametrize("ts,kw,word", [
    ([GOOD], dict(w_dtype=4), "must be bf16"), ([GOOD], dict(g_dtype=-1), "must be bf16"),
    ([GOOD], dict(bits=16), "8 or 32 bits"), ([GOOD], dict(b1=1.0), "betas"), ([GOOD], dict(b2=-0.1), "betas"),
    ([GOOD], dict(eps=-1.0), "eps"), ([GOOD], dict(step=0), "step"), ([GOOD], dict(scale=2), "grad_scale"),
    ([GOOD, (64, 128, 192, 256, 320, 384, -1, 0)], {}, "tensor 1: n"),
    ([(None,) + GOOD[1:]], {}, "null pointer"), ([(64, None) + GOOD[2:]], {}, "null pointer"),
    ([GOOD[:4] + (None, 384, 10, 0)], {}, "null pointer"), ([(65,) + GOOD[1:]], {}, "misaligned"),
    ([(64, 128, 196, 256, 320, 384, 10, 0)], {}, "misaligned"),
    ([(64, 128, 200, 256, None, None, 10, 0)], dict(bits=32), "misaligned")])
def test_adamw_rejects(ts, kw, word):
    assert _adamw(ts, **kw) == BAD and word in _lib.last_error()


def test_adamw_without_elements_is_a_success():
    assert _adamw([]) == OK
    assert _adamw([(None, None, None, None, None, None, 0, 0)] * 70) == OK


def test_grad_norm_rejects():
    L = _lib.lib()
    assert L.haste_grad_norm_workspace_size(-1) < 0
    size = L.haste_grad_norm_workspace_size(1)
    assert L.haste_grad_norm_workspace_size(500) > size > 0
    call = lambda t, n=1, mx=1.0, out=64, ws=128, b=size: L.haste_grad_norm(  # noqa: E731
        (_lib.GradTensor * 1)(t), n, mx, out, ws, b, None)
    for rc, kw, t, word in ((BAD, {}, (64, -1, BF16), "n must be"), (BAD, {}, (64, 5, 9), "must be bf16"),
                            (BAD, {}, (None, 5, BF16), "NULL"), (BAD, {}, (66, 5, F32), "misaligned"),
                            (BAD, dict(out=None), (64, 5, BF16), "out"), (BAD, dict(ws=None), (64, 5, BF16), "workspace"),
                            (BAD, dict(mx=-1.0), (64, 5, BF16), "max_norm"), (BAD, dict(n=-1), (64, 5, BF16), "list"),
                            (BAD, dict(mx=float("nan")), (64, 5, BF16), "max_norm"),
                            (WS, dict(b=size - 1), (64, 5, BF16), "too small")):
        assert call(t, **kw) == rc and word in _lib.last_error(), word


def test_python_refuses_cpu_tensors_and_bad_settings():
    w = torch.nn.Parameter(torch.ones(8))
    w.grad = torch.ones(8)
    with pytest.raises(RuntimeError, match="HIP device"):
        AdamW([w]).step()
    with pytest.raises(RuntimeError, match="HIP device"):
        grad_norm([w.grad])
    with pytest.raises(RuntimeError, match="HIP device"):
        ops.layer_norm(torch.ones(2, 8), w)
    with pytest.raises(RuntimeError, match="HIP device"):
        LayerNorm(8)(torch.ones(2, 8))
    for kw in (dict(lr=-1.0), dict(eps=-1.0), dict(betas=(1.0, 0.9)), dict(betas=(0.9, -0.1)),
               dict(weight_decay=-1.0), dict(state_bits=16)):
        with pytest.raises(ValueError):
            AdamW([w], **kw)


def test_state_that_does_not_fit_is_not_loaded():
    w = torch.nn.Parameter(torch.ones(200))
    opt = AdamW([w], state_bits=8)
    opt._new_state(w, 8)
    saved = opt.state_dict()
    assert saved["state"][0]["exp_avg"].numel() == 256 and saved["state"][0]["rms_scale"].numel() == 2
    again = AdamW([w], state_bits=8)
    again.load_state_dict(saved)
    assert again.state[w]["rms"].dtype == torch.float8_e4m3fn
    saved["param_groups"][0]["state_bits"] = 32
    with pytest.raises(ValueError, match="does not fit"):
        AdamW([w]).load_state_dict(saved)
