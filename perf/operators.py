"""Performance cases of the operators that train the encoder in front of an FFI layer.

Two kinds of pass:
  "ln"     ops.layer_norm: of rows [N, D], with a residual added to them first or without,
           forward alone (serving) or with its backward (all gradients);
  "adamw"  optim_adamw.AdamW.step over the tensors of an encoder, with optimizer states
           in 32 or in 8 bits, after the gradients' norm and clip factor
           (optim_adamw.grad_norm) or without.
Where ``own`` is false both are computed from elementary torch operations in 32 bits.

The tensors of an "adamw" case are views of one flat buffer, each starting at a multiple of
128 elements, so that a pass returns a few whole tensors however many parameters there are.
8-bit states are float8 codes with one power of two for each 128 elements; they are returned
as both (codes, scales).
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
LN_EPS = 1e-5
LR, BETAS, ADAM_EPS, WD = 1e-3, (0.9, 0.999), 1e-8, 0.01
STEP0, SEED0 = 99, 123        # steps that the states have behind them; the first pass's seed
MAX_NORM = 1.0
BLOCK = 128                   # elements of an 8-bit state that share a scale


def listed():
    return [
        # one short text's tokens in serving: the call's latency is all there is
        dict(name="ln_serve", kind="ln", N=32, D=768, dtype="bf16", wdtype="bf16", residual=False,
             train=False, pitch=0),
        # serving a batch of texts with the residual joined in
        dict(name="ln_serve_batch", kind="ln", N=16384, D=768, dtype="bf16", wdtype="bf16",
             residual=True, train=False, pitch=0),
        # an encoder layer's norm in training: 512 texts of 128 tokens, mixed precision
        dict(name="ln_train", kind="ln", N=65536, D=768, dtype="bf16", wdtype="f32",
             residual=True, train=True, pitch=0),
        # the wide penultimate layer's norm: few rows, many columns
        dict(name="ln_train_wide", kind="ln", N=256, D=4096, dtype="bf16", wdtype="bf16",
             residual=False, train=True, pitch=0),
        # fp32 training at odd sizes, rows cut out of a wider buffer
        dict(name="ln_train_odd", kind="ln", N=8191, D=769, dtype="f32", wdtype="f32",
             residual=False, train=True, pitch=3),
        # a long batch of a wide encoder
        dict(name="ln_train_large", kind="ln", N=65536, D=4096, dtype="bf16", wdtype="bf16",
             residual=True, train=True, pitch=0),
        # a projection with its norm: the smallest step, host time counts
        dict(name="adamw_small", kind="adamw", layers=0, width=768, ffn=0, vocab=512, dtype="bf16",
             gdtype="bf16", bits=32, sr=True, clip=False),
        # fp32 weights of a 6-layer encoder under mixed precision, clipped
        dict(name="adamw_f32", kind="adamw", layers=6, width=768, ffn=2048, vocab=32000,
             dtype="f32", gdtype="f32", bits=32, sr=False, clip=True),
        # bf16 weights stepped with stochastic rounding, 12 layers (195 tensors), clipped
        dict(name="adamw_bf16", kind="adamw", layers=12, width=768, ffn=2048, vocab=32000,
             dtype="bf16", gdtype="bf16", bits=32, sr=True, clip=True),
        # the same with states in 8 bits
        dict(name="adamw8_bf16", kind="adamw", layers=12, width=768, ffn=2048, vocab=32000,
             dtype="bf16", gdtype="bf16", bits=8, sr=True, clip=True),
        # ragged tensors in fp16 with fp32 gradients: every tensor ends inside a block
        dict(name="adamw8_odd", kind="adamw", layers=3, width=301, ffn=1003, vocab=20011,
             dtype="f16", gdtype="f32", bits=8, sr=True, clip=False),
        # a wide encoder's 670 M weights
        dict(name="adamw8_large", kind="adamw", layers=4, width=4096, ffn=8192, vocab=32000,
             dtype="bf16", gdtype="bf16", bits=8, sr=True, clip=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case of either kind: sizes spread over their ranges' logarithm."""
    if rng.random() < 0.5:
        while True:
            c = dict(kind="ln", N=_log(rng, 1, 131072), D=_log(rng, 8, 12000))
            if rng.random() < 0.5:
                c["D"] = max(64, c["D"] // 64 * 64)       # most widths are round
            if c["N"] * c["D"] <= 2 ** 27 and 3072 not in (c["N"], c["D"]):
                break
        c["dtype"] = rng.choice(["bf16", "bf16", "f16", "f32"])
        c["wdtype"] = rng.choice([c["dtype"], "f32"])
        c["residual"], c["train"] = rng.random() < 0.5, rng.random() < 0.7
        c["pitch"] = rng.choice([0, 0, 8, 5])
        return c
    while True:
        width = _log(rng, 64, 2048)
        if rng.random() < 0.6:
            width = max(64, width // 64 * 64)
        c = dict(kind="adamw", layers=rng.randint(0, 12), width=width,
                 ffn=width * rng.choice([1, 2, 4]) + rng.choice([0, 0, 3]), vocab=_log(rng, 100, 60000))
        if sum(math.prod(s) for s in _shapes(c)) <= 2 ** 27 and 3072 not in c.values():
            break
    c["dtype"] = rng.choice(["bf16", "bf16", "f16", "f32"])
    c["gdtype"] = rng.choice([c["dtype"], "f32"])
    c["bits"] = rng.choice([8, 32])
    c["sr"] = c["dtype"] != "f32" and rng.random() < 0.8
    c["clip"] = rng.random() < 0.5
    return c


def _shapes(c):
    """The parameters of an encoder: embedding with its norm, then layers of four square
    projections, two of the feed-forward, and two norms."""
    w, f = c["width"], c["ffn"]
    layer = [(w, w), (w,)] * 4 + [(f, w), (f,), (w, f), (w,)] + [(w,)] * 4
    return [(c["vocab"], w), (w,), (w,)] + layer * c["layers"]


def _layout(c):
    """(shape, first element, elements) of every tensor in the flat buffer, and its length."""
    out, at = [], 0
    for s in _shapes(c):
        n = math.prod(s)
        out.append((s, at, n))
        at += -(-n // BLOCK) * BLOCK
    return out, at


def work(case):
    c = case
    if c["kind"] == "ln":
        s, e = DTYPES[c["dtype"]].itemsize, c["N"] * c["D"]
        moved = (4 if c["residual"] else 2) + ((4 if c["residual"] else 3) if c["train"] else 0)
        ws = DTYPES[c["wdtype"]].itemsize * c["D"] * (5 if c["train"] else 2)
        return {"bytes": e * s * moved + ws + (16 * c["N"] if c["train"] else 0),
                "flops": e * (8 + (14 if c["train"] else 0))}
    n = sum(m for _, _, m in _layout(c)[0])
    state = 16 if c["bits"] == 32 else 4 + 4 / BLOCK
    return {"bytes": int(n * (2 * DTYPES[c["dtype"]].itemsize + DTYPES[c["gdtype"]].itemsize + state)),
            "flops": n * (16 + (2 if c["clip"] else 0))}


# ---------------------------------------------------------------- inputs ----
def prepare(case, seed):
    c = case
    g = torch.Generator(device="cuda").manual_seed(seed)
    rand = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    if c["kind"] == "ln":
        N, D, dt, wt = c["N"], c["D"], DTYPES[c["dtype"]], DTYPES[c["wdtype"]]
        # activations with a mean and a spread of their own in every row, some columns far out
        x = rand(N, D + c["pitch"]).mul_(torch.exp(rand(N, 1) * 0.5)).add_(rand(N, 1) * 0.3)
        x[:, :: 97] *= 6.0
        st = dict(c=c, x=x.to(dt)[:, :D], res=rand(N, D).to(dt) if c["residual"] else None,
                  w=(1 + 0.1 * rand(D)).to(wt), b=(0.1 * rand(D)).to(wt), dy=None, dh=None)
        if c["train"]:
            st["dy"] = (rand(N, D) * 0.1).to(dt)
            st["dh"] = (rand(N, D) * 0.1).to(dt) if c["residual"] else None
            st["leaves"] = [t for t in (st["x"], st["res"], st["w"], st["b"]) if t is not None]
            for t in st["leaves"]:
                t.requires_grad_(True)
        return st
    lay, n = _layout(c)
    dt, gt = DTYPES[c["dtype"]], DTYPES[c["gdtype"]]
    live = torch.zeros(n, dtype=torch.bool, device="cuda")
    for _, at, m in lay:
        live[at: at + m] = True
    # gradients spread over the tensors' blocks, about twice as long as MAX_NORM in all
    scale = torch.exp(rand(n // BLOCK) * 1.5).mul_(0.2 / math.sqrt(n)).repeat_interleave(BLOCK)
    st = dict(c=c, lay=lay, live=live, P=(rand(n) * 0.02 * live).to(dt),
              G=(rand(n) * scale * live).to(gt), t=STEP0, seed=SEED0)
    m = rand(n).mul_(scale).mul_(0.3).mul_(live)
    u = rand(n).mul_(0.3).exp_().mul_(scale).mul_(live)
    del scale
    if c["bits"] == 32:
        st["M"], st["V"] = m, u.square_()
    else:
        st["M"], st["MS"] = _to8(m)
        st["U"], st["US"] = _to8(u)
    if own:
        from haste_amd.optim_adamw import AdamW
        params = [torch.nn.Parameter(st["P"][at: at + k].view(s)) for s, at, k in lay]
        opt = AdamW(params, lr=LR, betas=BETAS, eps=ADAM_EPS, weight_decay=WD,
                    state_bits=c["bits"], stochastic_rounding=c["sr"], seed=SEED0)
        for p, (s, at, k) in zip(params, lay):
            p.grad_dtype = gt        # the gradients may be wider than the weights
            p.grad = st["G"][at: at + k].view(s)
            if c["bits"] == 32:
                state = dict(exp_avg=st["M"][at: at + k].view(s), exp_avg_sq=st["V"][at: at + k].view(s))
            else:
                end = at + -(-k // BLOCK) * BLOCK
                blk = slice(at // BLOCK, end // BLOCK)
                state = dict(exp_avg=st["M"][at:end], exp_avg_scale=st["MS"][blk],
                             rms=st["U"][at:end], rms_scale=st["US"][blk])
            opt.state[p] = dict(step=STEP0, **state)
        st["opt"], st["grads"] = opt, [p.grad for p in params]
    return st


def _to8(x):
    """Codes and scales of x, rounded to nearest: states as an earlier step left them."""
    x = x.view(-1, BLOCK)
    code = _scale_code(x.abs().amax(1))
    codes = x.mul(_pow2(127 - code)[:, None]).to(torch.float8_e4m3fn)
    return codes.view(-1), code.to(torch.uint8).view(torch.float8_e8m0fnu)


def _exponent(x):
    """Biased exponent of x >= 0."""
    return x.view(torch.int32) >> 23


def _pow2(e):
    return ((e + 127) << 23).view(torch.float32)


def _scale_code(most):
    return (_exponent(most) - 7).clamp_(min=1)


# ------------------------------------------------------------------ passes ----
def run(state):
    c = state["c"]
    if c["kind"] == "ln":
        return _ln_own(state) if own else _ln_plain(state)
    out = _adamw_own(state) if own else _adamw_plain(state)
    return out | ({"p": state["P"], "m": state["M"], "v": state["V"]} if c["bits"] == 32 else
                  {"p": state["P"], "m": state["M"], "m_scale": state["MS"], "u": state["U"],
                   "u_scale": state["US"]})


def _ln_own(st):
    from haste_amd import ops
    c = st["c"]
    if not c["residual"]:
        y = ops.layer_norm(st["x"], st["w"], st["b"], eps=LN_EPS)
        out, grads = {"y": y}, [st["dy"]]
    else:
        y, h = ops.layer_norm(st["x"], st["w"], st["b"], eps=LN_EPS, residual=st["res"])
        out, grads = {"y": y, "h": h}, [st["dy"], st["dh"]]
    if c["train"]:
        got = torch.autograd.grad(list(out.values()), st["leaves"], grads)
        names = ["dx", "dres", "dw", "db"] if c["residual"] else ["dx", "dw", "db"]
        out = {k: v.detach() for k, v in out.items()} | dict(zip(names, got))
    return out


@torch.no_grad()
def _ln_plain(st):
    c, D, dt = st["c"], st["c"]["D"], st["x"].dtype
    w, b = st["w"].float(), st["b"].float()
    h = st["x"] if st["res"] is None else (st["x"].float() + st["res"].float()).to(dt)
    xh = h.float()
    xh = xh - xh.sum(1, keepdim=True) / D
    r = 1 / torch.sqrt((xh * xh).sum(1, keepdim=True) / D + LN_EPS)
    xh = xh * r
    out = {"y": (xh * w + b).to(dt)}
    if c["residual"]:
        out["h"] = h
    if c["train"]:
        dy = st["dy"].float()
        a = dy * w
        dx = r * (a - a.sum(1, keepdim=True) / D - xh * ((a * xh).sum(1, keepdim=True) / D))
        if c["residual"]:
            dx = dx + st["dh"].float()
        out["dx"] = dx.to(dt)
        if c["residual"]:
            out["dres"] = out["dx"]
        out["dw"] = (dy * xh).sum(0).to(st["w"].dtype)
        out["db"] = dy.sum(0).to(st["b"].dtype)
    return out


def _adamw_own(st):
    if not st["c"]["clip"]:
        st["opt"].step()
        return {}
    from haste_amd.optim_adamw import grad_norm
    norm, coef = grad_norm(st["grads"], MAX_NORM)
    st["opt"].step(grad_scale=coef)
    return {"norm": norm, "coef": coef}


@torch.no_grad()
def _adamw_plain(st):
    c, out = st["c"], {}
    P, b1, b2 = st["P"], *BETAS
    st["t"], seed = st["t"] + 1, st["seed"]
    st["seed"] += 1
    g = st["G"].float()
    if c["clip"]:
        norm = torch.sqrt((g * g).sum())
        coef = (MAX_NORM / (norm + 1e-6)).clamp(max=1.0)
        out = {"norm": norm, "coef": coef}
        g = g * coef
    if c["bits"] == 32:
        m, v = st["M"], st["V"]
        m.copy_(m * b1 + g * (1 - b1))
        v.copy_(v * b2 + g * g * (1 - b2))
        u = torch.sqrt(v)
    else:
        m = _from8(st["M"], st["MS"]) * b1 + g * (1 - b1)
        u = _from8(st["U"], st["US"])
        u = torch.sqrt(u * u * b2 + g * g * (1 - b2))
    del g
    step = m / (u * (1 / math.sqrt(1 - b2 ** st["t"])) + ADAM_EPS) * (LR / (1 - b1 ** st["t"]))
    w = P.float() * (1 - LR * WD) - step
    del step
    words = _words(st, seed, 8 if c["bits"] == 32 else 4) if c["sr"] or c["bits"] == 8 else None
    if c["bits"] == 8:
        hi = words >> 16
        st["M"][:], st["MS"][:] = _round8(m, hi, False)
        st["U"][:], st["US"][:] = _round8(u, torch.roll(hi, -1, 1), True)
        words = words & 0xFFFF
    elif c["sr"]:
        words = torch.stack([words & 0xFFFF, words >> 16], 2)
    P.copy_(_round16(w, words.view(-1), P.dtype) if c["sr"] else w)
    return out


def _from8(codes, scales):
    return (codes.float().view(-1, BLOCK) * scales.float()[:, None]).view(-1)


def _round8(x, r, keep):
    """x to e4m3 under one power of two for each block, up with the probability of what is cut
    off; `keep`: what is above zero stays above it."""
    x = x.view(-1, BLOCK)
    a = x.abs()
    code = _scale_code(a.amax(1))
    a = a * _pow2(127 - code)[:, None]
    q = _exponent(a).clamp(min=127 - 6) - 127 - 3
    t = torch.floor(a * _pow2(-q) + r.view(-1, BLOCK).float() * 2.0 ** -16)
    if keep:
        t = torch.where(a > 0, t.clamp(min=1), t)
    t = torch.copysign(t * _pow2(q), x)
    return t.to(torch.float8_e4m3fn).view(-1), code.to(torch.uint8).view(torch.float8_e8m0fnu)


def _round16(w, r, dtype):
    """w to 16 bits, up with the probability of what is cut off."""
    r = r.to(torch.int32)
    if dtype == torch.bfloat16:
        return ((w.view(torch.int32) + r) & -65536).view(torch.float32).to(dtype)
    a = w.abs()
    q = _exponent(a).clamp(min=127 - 14) - 127 - 10
    t = torch.floor(a * _pow2(-q) + (r >> 3).float() * 2.0 ** -13)
    return torch.copysign(t * _pow2(q), w).to(dtype)


def _words(st, seed, per):
    """Philox4x32-10 words [elements / per, 4]: key `seed`, counter (element / per within its
    tensor: low, high word; the tensor's index; 0)."""
    size = torch.tensor([-(-n // BLOCK) for _, _, n in st["lay"]], device=st["P"].device)
    index = torch.arange(len(size), device=size.device).repeat_interleave(size)
    first = (size.cumsum(0) - size).repeat_interleave(size)
    block = torch.arange(index.numel(), device=size.device) - first
    k = BLOCK // per
    at = (block[:, None] * k + torch.arange(k, device=size.device)).view(-1)
    low = 0xFFFFFFFF
    c0, c1, c2, c3 = at & low, at >> 32, index.repeat_interleave(k), torch.zeros_like(at)
    k0, k1 = seed & low, seed >> 32 & low
    for _ in range(10):
        p0, p1 = c0 * 0xD2511F53, c2 * 0xCD9E8D57
        c0, c1, c2, c3 = ((p1 >> 32) & low) ^ c1 ^ k0, p1 & low, ((p0 >> 32) & low) ^ c3 ^ k1, p0 & low
        k0, k1 = (k0 + 0x9E3779B9) & low, (k1 + 0xBB67AE85) & low
    return torch.stack([c0, c1, c2, c3], 1)


# ----------------------------------------------------------- in 64 bits ----
@torch.no_grad()
def exact(case, seed):
    """What a first pass returns, in double precision from the definitions: what is rounded to
    nearest is left unrounded, what is rounded by drawn bits is rounded by them."""
    st = prepare(case, seed)
    return _ln_exact(st) if case["kind"] == "ln" else _adamw_exact(st)


def _ln_exact(st):
    c = st["c"]
    h = st["x"].double()
    if c["residual"]:
        h = (h + st["res"].double()).to(st["x"].dtype).double()
    var, mean = torch.var_mean(h, 1, correction=0, keepdim=True)
    sd = (var + LN_EPS).sqrt()
    n = (h - mean) / sd
    w = st["w"].double()
    out = {"y": torch.addcmul(st["b"].double(), n, w)}
    if c["residual"]:
        out["h"] = h
    if c["train"]:
        dy = st["dy"].double()
        dn = dy * w
        # the gradient with respect to h is dn less its parts along 1 and along n
        dh = (dn - dn.mean(1, keepdim=True) - n * (dn * n).mean(1, keepdim=True)) / sd
        if c["residual"]:
            dh += st["dh"].double()
            out["dres"] = dh
        out["dx"] = dh
        out["dw"] = torch.linalg.vecdot(dy, n, dim=0)
        out["db"] = dy.sum(0)
    return out


def _adamw_exact(st):
    c, (b1, b2), t = st["c"], BETAS, STEP0 + 1
    out, parts = {}, []
    factor = 1.0
    if c["clip"]:
        norm = math.sqrt(sum(float(x.double().square().sum()) for x in st["G"].split(1 << 26)))
        factor = min(1.0, MAX_NORM / (norm + 1e-6))
        out = {"norm": torch.tensor(norm, dtype=torch.float64), "coef": torch.tensor(factor, dtype=torch.float64)}
    for i, (_, at, n) in enumerate(st["lay"]):
        end = at + -(-n // BLOCK) * BLOCK
        cut, blk = slice(at, end), slice(at // BLOCK, end // BLOCK)
        g = st["G"][cut].double() * factor
        if c["bits"] == 32:
            m, v = st["M"][cut].double(), st["V"][cut].double()
        else:
            m, v = (st[k][cut].double().view(-1, BLOCK) * st[s][blk].float().double()[:, None]
                    for k, s in (("M", "MS"), ("U", "US")))
            m, v = m.view(-1), v.view(-1) ** 2
        m, v = torch.lerp(g, m, b1), torch.lerp(g * g, v, b2)
        w = st["P"][cut].double() * (1 - LR * WD)
        w -= LR * (m / (1 - b1 ** t)) / ((v / (1 - b2 ** t)).sqrt() + ADAM_EPS)
        bits = _draws(i, end - at, 4 if c["bits"] == 8 else 8, w.device) if c["sr"] or c["bits"] == 8 else None
        if c["bits"] == 8:
            m, ms = _cut8(m, bits >> 16)
            u, us = _cut8(v.sqrt(), (bits >> 16).view(-1, 4)[:, [1, 2, 3, 0]].reshape(-1))
            u = torch.where((v > 0) & (u == 0), torch.full_like(u, 2.0 ** -9), u)
            bits = bits % 65536
        if c["sr"]:
            mant, low, most = (7, -126, 16) if c["dtype"] == "bf16" else (10, -14, 13)
            w = _cut(w, bits / 2.0 ** 16 if most == 16 else torch.floor(bits / 8) / 2.0 ** 13, mant, low)
        parts.append((w, m, v) if c["bits"] == 32 else (w, m, ms, u, us))
    names = ("p", "m", "v") if c["bits"] == 32 else ("p", "m", "m_scale", "u", "u_scale")
    return out | {k: torch.cat([p[j] for p in parts]) for j, k in enumerate(names)}


def _cut(x, up, mantissa, low):
    """x to multiples of its spacing, up if what is cut off and `up` make a whole one."""
    e = (torch.frexp(x.abs()).exponent - 1).clamp(min=low) - mantissa
    unit = torch.exp2(e.double())
    return torch.sign(x) * torch.floor(x.abs() / unit + up) * unit


def _cut8(x, bits):
    x = x.view(-1, BLOCK)
    top = x.abs().amax(1)
    e = torch.where(top > 0, torch.frexp(top).exponent - 1 - 7, -126).clamp(min=-126).double()
    codes = _cut(x / torch.exp2(e)[:, None], bits.view(-1, BLOCK) / 2.0 ** 16, 3, -6)
    return codes.view(-1), torch.exp2(e)


def _draws(index, n, per, device):
    """The drawn bits of a tensor's elements, 32 each (per = 4) or 16 (per = 8): Philox4x32-10
    with products put together from 16-bit halves."""
    def mul(a, k):
        a0, a1, k0, k1 = a & 65535, a >> 16, k & 65535, k >> 16
        mid = a1 * k0 + (a0 * k0 >> 16)
        mid2 = a0 * k1 + (mid & 65535)
        return a1 * k1 + (mid >> 16) + (mid2 >> 16), (mid2 & 65535) << 16 | (a0 * k0 & 65535)
    j = torch.arange(n // per, device=device)
    x = [j % 2 ** 32, j // 2 ** 32, torch.full_like(j, index), torch.zeros_like(j)]
    for r in range(10):
        (h0, l0), (h1, l1) = mul(x[0], 0xD2511F53), mul(x[2], 0xCD9E8D57)
        x = [h1 ^ x[1] ^ (SEED0 + r * 0x9E3779B9) % 2 ** 32, l1, h0 ^ x[3] ^ (r * 0xBB67AE85) % 2 ** 32, l0]
    if per == 4:
        return torch.stack(x, 1).view(-1)
    return torch.stack([h for w in x for h in (w % 65536, w >> 16)], 1).view(-1)
