"""The C entry points of the embedding, the gated block and the label log probabilities reject bad
arguments on the host (these calls return before any HIP call), and the Python functions CPU tensors."""
import pytest
import torch

from haste_amd import _lib, ops

OK, BAD, WS = _lib.HASTE_OK, _lib.HASTE_ERR_INVALID_ARG, _lib.HASTE_ERR_WORKSPACE
BF16, F16, F32 = _lib.DTYPE_BF16, _lib.DTYPE_F16, _lib.DTYPE_F32


def _call(name, args, **kw):
    return getattr(_lib.lib(), name)(*dict(args, **kw).values())


EMB = dict(tokens=64, bits=64, w=64, ldw=8, y=64, N=4, V=10, D=8, scale=1.0, dtype=BF16, stream=None)
EMB_BWD = dict(tokens=64, bits=64, dy=64, lddy=8, dw=64, N=4, V=10, D=8, scale=1.0, padding=-1, dtype=BF16,
               ws=256, ws_bytes=1 << 40, stream=None)


@pytest.mark.parametrize("kw", [dict(bits=16), dict(tokens=None), dict(tokens=68), dict(w=None), dict(w=65),
                                dict(ldw=7), dict(ldw=-8), dict(y=None), dict(N=-1), dict(V=0), dict(D=0),
                                dict(N=1 << 31), dict(V=1 << 31), dict(D=1 << 31), dict(dtype=3),
                                dict(dtype=F32, w=66)])
def test_embedding_rejects(kw):
    assert _call("haste_embedding", EMB, **kw) == BAD and "haste_embedding" in _lib.last_error()


@pytest.mark.parametrize("kw", [dict(bits=8), dict(tokens=None), dict(dy=None), dict(lddy=5), dict(dw=None),
                                dict(dw=65), dict(V=0), dict(N=-1), dict(dtype=9), dict(ws=None), dict(ws=8)])
def test_embedding_bwd_rejects(kw):
    assert _call("haste_embedding_bwd", EMB_BWD, **kw) == BAD


def test_embedding_sizes():
    size = _lib.lib().haste_embedding_bwd_workspace_size
    assert size(-1, 1, 1) < 0 and size(1, 0, 1) < 0 and size(1, 1, 1 << 31) < 0
    last = 0
    for N in (0, 1, 2048, 2049, 65536, 65537, 10 ** 6, 2 ** 31 - 1):
        got = size(N, 32000, 768)
        assert got >= 16 * N and got >= last
        last = got
    assert _call("haste_embedding_bwd", EMB_BWD, ws_bytes=size(4, 10, 8) - 1) == WS
    assert "workspace too small" in _lib.last_error()
    assert _call("haste_embedding", EMB, N=0) == OK


MLP = dict(x=64, ldx=8, wg=64, ldg=8, wu=64, ldu=8, wd=64, ldd=16, y=64, kept=None, h=64, N=100, D=8, H=16,
           O=8, act=0, dtype=BF16, ws=256, ws_bytes=1 << 40, stream=None)
MLP_BWD = dict(x=64, ldx=8, wg=64, ldg=8, wu=64, ldu=8, wd=64, ldd=16, dy=64, lddy=8, kept=64, h=64, dx=64,
               dwg=64, dwu=64, dwd=64, N=100, D=8, H=16, O=8, dtype=BF16, ws=256, ws_bytes=1 << 40,
               stream=None)


@pytest.mark.parametrize("kw", [dict(act=3), dict(act=-1), dict(dtype=3), dict(N=-1), dict(D=0), dict(H=0),
                                dict(O=0), dict(N=1 << 30), dict(D=(1 << 20) + 1), dict(N=1 << 29, D=64, ldx=64), dict(x=None), dict(x=65),
                                dict(ldx=7), dict(ldx=0), dict(ldx=1 << 23), dict(wg=None), dict(wu=None),
                                dict(wd=None), dict(ldd=15), dict(y=None), dict(h=None), dict(h=72),
                                dict(kept=72), dict(dtype=F32, x=66)])
def test_gated_mlp_rejects(kw):
    assert _call("haste_gated_mlp", MLP, **kw) == BAD and "haste_gated_mlp" in _lib.last_error()


@pytest.mark.parametrize("kw", [dict(dtype=7), dict(N=-1), dict(dy=None), dict(lddy=0), dict(kept=None),
                                dict(h=None), dict(dwg=None), dict(dwu=None), dict(dx=65), dict(ws=None),
                                dict(ws=8), dict(x=None)])
def test_gated_mlp_bwd_rejects(kw):
    assert _call("haste_gated_mlp_bwd", MLP_BWD, **kw) == BAD


def test_gated_mlp_sizes():
    L = _lib.lib()
    size, kept = L.haste_gated_mlp_workspace_size, L.haste_gated_mlp_kept_size
    assert size(100, 0, 16, 8, BF16, 0, 0) < 0 and size(100, 8, 16, 8, 5, 0, 0) < 0
    assert kept(-1, 8, BF16) < 0 and kept(0, 8, BF16) == 0
    assert kept(17, 65, BF16) == 2 * 2 * 2 * 16 * 64 * 3 and kept(17, 65, F32) == 2 * 2 * 2 * 16 * 64 * 4
    for dt in (BF16, F16, F32):
        for backward in (0, 1):
            for s in ((1, 1, 1, 1), (100, 8, 16, 8), (65, 301, 1003, 301), (65536, 768, 2048, 768),
                      (16384, 4096, 8192, 4096)):
                a, b = size(*s, dt, backward, 1), size(*s, dt, backward, 0)
                assert 0 <= a <= b or dt == F32 and a == b
    # odd rows are copied: more than aligned ones take
    need = size(100, 8, 16, 8, BF16, 1, 0)
    assert _call("haste_gated_mlp_bwd", MLP_BWD, x=66, dy=66, wg=66, wu=66, wd=66, ws_bytes=need - 1) == WS
    assert _call("haste_gated_mlp", MLP, N=0) == OK
    # two pitches of the projections: both are copied
    assert _call("haste_gated_mlp", MLP, ldu=16, ws_bytes=size(100, 8, 16, 8, BF16, 0, 1)) == WS
    assert _call("haste_gated_mlp_bwd", MLP_BWD, ldg=16, ws_bytes=size(100, 8, 16, 8, BF16, 1, 1)) == WS


LP = dict(z=64, ldz=50, labels=64, bits=64, L=2, stats=None, lp=64, ent=64, top=64, top_labels=64, B=4, O=50,
          K=3, dtype=BF16, ws=None, ws_bytes=0, stream=None)
LP_BWD = dict(z=64, ldz=50, labels=64, bits=64, L=2, stats=64, ent=64, dlp=64, dent=64, dz=64, lddz=50, B=4,
              O=50, dtype=BF16, stream=None)


@pytest.mark.parametrize("kw", [dict(z=None), dict(z=65), dict(ldz=49), dict(labels=None), dict(labels=68),
                                dict(bits=16), dict(L=-1), dict(B=-1), dict(O=0), dict(O=1 << 31),
                                dict(B=1 << 31), dict(K=-1), dict(K=51), dict(K=129, O=1000, ldz=1000),
                                dict(lp=None), dict(top=None), dict(top_labels=None), dict(top_labels=68),
                                dict(ent=66), dict(stats=66), dict(dtype=3)])
def test_label_log_probs_rejects(kw):
    assert _call("haste_label_log_probs", LP, **kw) == BAD
    assert "haste_label_log_probs" in _lib.last_error()


@pytest.mark.parametrize("kw", [dict(z=None), dict(stats=None), dict(ent=None), dict(dlp=66), dict(dent=66),
                                dict(dz=None), dict(dz=65), dict(lddz=49), dict(labels=None), dict(bits=0),
                                dict(L=4097)])
def test_label_log_probs_bwd_rejects(kw):
    assert _call("haste_label_log_probs_bwd", LP_BWD, **kw) == BAD


def test_label_log_probs_sizes():
    size = _lib.lib().haste_label_log_probs_workspace_size
    assert size(-1, 5, 0) < 0 and size(1, 0, 0) < 0 and size(1, 5, 129) < 0 and size(1, 1 << 31, 0) < 0
    assert size(0, 5, 0) >= 0 and size(512, 1000, 10) == 0       # (rows that are not cut)
    need = size(1, 131073, LP["K"])
    assert 0 < size(1, 131073, 0) < need < size(1, 131073, 10)
    assert _call("haste_label_log_probs", LP, B=1, O=131073, ldz=131073, ws=64, ws_bytes=need - 1) == WS
    assert _call("haste_label_log_probs", LP, B=1, O=131073, ldz=131073, ws=64, ws_bytes=0) == WS
    assert _call("haste_label_log_probs", LP, B=1, O=131073, ldz=131073) == BAD   # no workspace
    assert _call("haste_label_log_probs", LP, B=0) == OK and _call("haste_label_log_probs_bwd", LP_BWD, B=0) == OK


def test_python_functions_reject_cpu_tensors():
    x = torch.randn(4, 8)
    t = torch.zeros(4, dtype=torch.int64)
    for f in (lambda: ops.embedding(t, x), lambda: ops.gated_mlp(x, x, x, x), lambda: ops.label_log_probs(x),
              lambda: ops.embedding(t, None), lambda: ops.label_log_probs([1.0]),
              lambda: ops.gated_mlp(x, None, x, x)):
        with pytest.raises(RuntimeError, match="HIP device"):
            f()
    with pytest.raises(ValueError, match="activation"):
        ops.gated_mlp(x, x, x, x, activation="relu")
