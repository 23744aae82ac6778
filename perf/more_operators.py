"""Performance cases of what an encoder and its output layer answer with, beside the layer itself.

Three kinds of pass:
  "emb"  ops.embedding: rows of a table by tokens, scaled, forward alone (serving) or with the
         table's gradient;
  "mlp"  ops.gated_mlp: the gated feed-forward block (act(x Wg^T) * (x Wu^T)) Wd^T, forward alone or
         with all gradients;
  "lp"   ops.label_log_probs: log probabilities of given labels under rows of logits, their entropy
         and the likeliest labels, forward alone or with the logits' gradient.
Where ``own`` is false all are computed from elementary torch operations in 32 bits.
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def listed():
    return [
        # one short text's tokens in serving: the call's latency is all there is
        dict(name="emb_serve", kind="emb", N=32, D=768, V=32000, dtype="bf16", train=False, scale=1.0),
        # 512 texts of 128 tokens in training, rows scaled by the root of their width
        dict(name="emb_train", kind="emb", N=65536, D=768, V=32000, dtype="bf16", train=True,
             scale=768 ** 0.5),
        # ragged texts, odd widths, fp32 tables
        dict(name="emb_train_odd", kind="emb", N=8191, D=301, V=20011, dtype="f32", train=True,
             scale=0.5),
        # one text's vector through a block of the encoder: its weights are read for one row
        dict(name="mlp_serve", kind="mlp", N=1, D=768, H=2048, dtype="bf16", act="silu", train=False),
        # a request's tokens in serving
        dict(name="mlp_serve_batch", kind="mlp", N=509, D=768, H=2048, dtype="bf16", act="gelu",
             train=False),
        # a block of the encoder in training: 512 texts of 128 tokens
        dict(name="mlp_train", kind="mlp", N=65536, D=768, H=2048, dtype="bf16", act="silu", train=True),
        # odd sizes in fp16: no row starts on 16 bytes
        dict(name="mlp_train_odd", kind="mlp", N=4001, D=301, H=1003, dtype="f16", act="gelu_tanh",
             train=True),
        # a wide encoder's block
        dict(name="mlp_train_large", kind="mlp", N=16384, D=4096, H=8192, dtype="bf16", act="silu",
             train=True),
        # one text's answers among 131,073 labels
        dict(name="lp_serve", kind="lp", B=1, O=131073, L=0, top=5, dtype="bf16", train=False, pitch=0),
        # evaluating a batch: its labels' probabilities, the entropy, and the ten likeliest labels
        dict(name="lp_eval", kind="lp", B=512, O=131073, L=8, top=10, dtype="bf16", train=False,
             pitch=63),
        # the softmax loss of a batch over 670,091 labels
        dict(name="lp_train", kind="lp", B=512, O=670091, L=8, top=0, dtype="bf16", train=True,
             pitch=21),
        # a small label set in fp32, rows cut out of a wider buffer
        dict(name="lp_train_odd", kind="lp", B=301, O=4099, L=3, top=3, dtype="f32", train=True,
             pitch=5),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case of any kind: sizes spread over their ranges' logarithm."""
    kind = rng.choice(["emb", "mlp", "lp"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    train = rng.random() < 0.6
    if kind == "emb":
        while True:
            c = dict(kind=kind, N=_log(rng, 1, 262144), D=_log(rng, 8, 4096), V=_log(rng, 64, 200000))
            if rng.random() < 0.5:
                c["D"] = max(64, c["D"] // 64 * 64)       # most widths are round
            if max(c["N"], c["V"]) * c["D"] <= 2 ** 27:
                break
        scale = rng.choice([1.0, c["D"] ** 0.5, 0.5])
        return dict(c, dtype=dtype, train=train, scale=scale)
    if kind == "mlp":
        while True:
            c = dict(kind=kind, N=_log(rng, 1, 65536), D=_log(rng, 32, 4096), H=_log(rng, 32, 8192))
            if rng.random() < 0.6:
                c["D"], c["H"] = (max(64, c[k] // 64 * 64) for k in "DH")
            if c["N"] * c["D"] * c["H"] <= 2 ** (36 if dtype == "f32" else 38):
                break
        return dict(c, dtype=dtype, act=rng.choice(["silu", "gelu", "gelu_tanh"]), train=train)
    while True:
        c = dict(kind=kind, B=_log(rng, 1, 4096), O=_log(rng, 100, 3000000))
        if c["B"] * c["O"] <= 2 ** 28:
            break
    return dict(c, L=rng.randint(1, 12), top=rng.choice([0, 1, 5, 10, 100]), dtype=dtype, train=train,
                pitch=rng.choice([0, 0, 8, 5]))


def work(case):
    c, s = case, DTYPES[case["dtype"]].itemsize
    if c["kind"] == "emb":
        rows = c["N"] * c["D"]
        read = min(c["N"], c["V"]) * c["D"]
        moved = (read + rows) * s + 8 * c["N"]
        if c["train"]:
            moved += (rows + c["V"] * c["D"]) * s
        return {"bytes": moved, "flops": rows * (2 if c["train"] else 1)}
    if c["kind"] == "mlp":
        N, D, H = c["N"], c["D"], c["H"]
        return {"bytes": s * ((4 if c["train"] else 2) * N * D + (6 if c["train"] else 3) * D * H),
                "flops": (18 if c["train"] else 6) * N * D * H}
    e = c["B"] * c["O"]
    return {"bytes": e * s * (3 if c["train"] else 1) + c["B"] * (12 * c["L"] + 12 * c["top"] + 4),
            "flops": e * (8 + (6 if c["train"] else 0))}


# ---------------------------------------------------------------- inputs ----
def prepare(case, seed):
    c = case
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = DTYPES[c["dtype"]]
    rand = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    rand01 = lambda *s: torch.rand(*s, generator=g, device="cuda")  # noqa: E731
    if c["kind"] == "emb":
        N, D, V = c["N"], c["D"], c["V"]
        # tokens by the inverse of their rank, in an order of their own; a fifth is padding
        names = torch.randperm(V, generator=g, device="cuda")
        tokens = names[(torch.exp(rand01(N).double() * math.log(V)) - 1).long().clamp_(0, V - 1)]
        tokens = torch.where(rand01(N) < 0.2, torch.zeros_like(tokens), tokens)
        st = dict(c=c, tokens=tokens, w=(rand(V, D) * 0.02).to(dt))
        if c["train"]:
            st["dy"] = (rand(N, D) * 0.1).to(dt)
            st["leaves"] = [st["w"].requires_grad_(True)]
        return st
    if c["kind"] == "mlp":
        N, D, H = c["N"], c["D"], c["H"]
        st = dict(c=c, x=rand(N, D).to(dt), wg=(rand(H, D) / D ** 0.5).to(dt),
                  wu=(rand(H, D) / D ** 0.5).to(dt), wd=(rand(D, H) / H ** 0.5).to(dt))
        if c["train"]:
            st["dy"] = (rand(N, D) * 0.1).to(dt)
            st["leaves"] = [st[k].requires_grad_(True) for k in ("x", "wg", "wu", "wd")]
        return st
    B, O, L = c["B"], c["O"], c["L"]
    # logits around -4 with a spread of 2; one label in a hundred is not to be answered
    z = torch.empty(B, O + c["pitch"], device="cuda", dtype=dt)
    for at in range(0, B, 64):
        z[at: at + 64] = rand(min(64, B - at), O + c["pitch"]).mul_(2.0).sub_(4.0)
    z[:, :O].masked_fill_(rand01(O) < 0.01, -math.inf)
    # up to L labels a row, the rest of the list is empty (-1)
    labels = torch.randint(0, O, (B, L), generator=g, device="cuda")
    labels = torch.where(rand01(B, L) < 0.3, torch.full_like(labels, -1), labels)
    if L:
        at = labels.clamp(min=0)
        z[:, :O].scatter_(1, at, (2 + 0.25 * (at % 13)).to(dt))    # (a label twice: one value)
    st = dict(c=c, z=z[:, :O], labels=labels if L else None)
    if c["train"]:
        st["dlp"] = rand01(B, L).add_(0.5).mul_(-1.0 / max(L, 1))
        st["dent"] = rand(B) * 0.01
        st["leaves"] = [st["z"].requires_grad_(True)]
    return st


# ------------------------------------------------------------------ passes ----
def run(state):
    kind = state["c"]["kind"]
    if own:
        return {"emb": _emb_own, "mlp": _mlp_own, "lp": _lp_own}[kind](state)
    return {"emb": _emb_plain, "mlp": _mlp_plain, "lp": _lp_plain}[kind](state)


def _emb_own(st):
    from haste_amd import ops
    c = st["c"]
    y = ops.embedding(st["tokens"], st["w"], scale=c["scale"], padding_idx=0)
    if not c["train"]:
        return {"y": y}
    dw, = torch.autograd.grad([y], st["leaves"], [st["dy"]])
    return {"y": y.detach(), "dw": dw}


@torch.no_grad()
def _emb_plain(st):
    c, w = st["c"], st["w"]
    out = {"y": (w[st["tokens"]].float() * c["scale"]).to(w.dtype)}
    if c["train"]:
        live = st["tokens"] != 0
        # (in 64 bits: a frequent token's sum is long)
        dw = torch.zeros(w.shape, dtype=torch.float64, device=w.device)
        dw.index_add_(0, st["tokens"], st["dy"].double() * live[:, None])
        out["dw"] = (dw * c["scale"]).to(w.dtype)
    return out


def _mlp_own(st):
    from haste_amd import ops
    c = st["c"]
    y = ops.gated_mlp(st["x"], st["wg"], st["wu"], st["wd"], activation=c["act"])
    if not c["train"]:
        return {"y": y}
    got = torch.autograd.grad([y], st["leaves"], [st["dy"]])
    return {"y": y.detach()} | dict(zip(["dx", "dwg", "dwu", "dwd"], got))


@torch.no_grad()
def _mlp_plain(st):
    c, dt = st["c"], st["x"].dtype
    x, wg, wu, wd = (st[k].float() for k in ("x", "wg", "wu", "wd"))
    g, u = x @ wg.t(), x @ wu.t()
    if c["act"] == "silu":
        s = 1 / (1 + torch.exp(-g))
        a, slope = g * s, s * (1 + g * (1 - s))
    elif c["act"] == "gelu":
        cdf = 0.5 * (1 + torch.erf(g * 0.5 ** 0.5))
        a, slope = g * cdf, cdf + g * torch.exp(-0.5 * g * g) * (1 / math.sqrt(2 * math.pi))
    else:
        k, k3 = math.sqrt(2 / math.pi), 0.044715
        t = torch.tanh(k * (g + k3 * g * g * g))
        a = 0.5 * g * (1 + t)
        slope = 0.5 * (1 + t) + 0.5 * g * (1 - t * t) * k * (1 + 3 * k3 * g * g)
    h = a * u
    out = {"y": (h @ wd.t()).to(dt)}
    if c["train"]:
        dy = st["dy"].float()
        dh = dy @ wd
        dg, du = dh * u * slope, dh * a
        out |= {"dx": (dg @ wg + du @ wu).to(dt), "dwg": (dg.t() @ x).to(dt), "dwu": (du.t() @ x).to(dt),
                "dwd": (dy.t() @ h).to(dt)}
    return out


def _lp_own(st):
    from haste_amd import ops
    c = st["c"]
    r = ops.label_log_probs(st["z"], st["labels"], top=c["top"])
    out = {"entropy": r.entropy}
    if c["L"]:
        out["log_probs"] = r.log_probs
    if c["top"]:
        out |= {"top_log_probs": r.top_log_probs, "top_labels": r.top_labels}
    if c["train"]:
        dz, = torch.autograd.grad([r.log_probs, r.entropy], st["leaves"], [st["dlp"], st["dent"]])
        out = {k: v.detach() for k, v in out.items()} | {"dz": dz}
    return out


@torch.no_grad()
def _lp_plain(st):
    c, z = st["c"], st["z"].float()
    m = z.amax(1, keepdim=True)
    t = z - m
    e = torch.exp(t)
    s = e.sum(1, keepdim=True)
    log_s = torch.log(s)
    t = torch.where(e > 0, t, torch.zeros_like(t))       # (what is left out counts for nothing)
    ent = log_s - (e * t).sum(1, keepdim=True) / s
    out = {"entropy": ent[:, 0]}
    if c["L"]:
        given = st["labels"] >= 0
        label = st["labels"].clamp(min=0)
        out["log_probs"] = torch.where(given, z.gather(1, label) - m - log_s, torch.zeros_like(m))
    if c["top"]:
        # the float's order as a whole number's, then the lowest label first
        bits = torch.where(z == 0, torch.zeros_like(z), z).view(torch.int32)
        bits = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits).long()
        key = (bits << 32) + (0xFFFFFFFF - torch.arange(c["O"], device=z.device))
        at = 0xFFFFFFFF - (key.topk(c["top"], 1).values & 0xFFFFFFFF)
        out |= {"top_log_probs": z.gather(1, at) - m - log_s, "top_labels": at}
    if c["train"]:
        p = e / s
        dz = p * (-(st["dlp"] * given).sum(1, keepdim=True) - st["dent"][:, None] * (t - log_s + ent))
        dz.scatter_add_(1, label, st["dlp"] * given)
        out["dz"] = dz.to(st["z"].dtype)
    return out


# ----------------------------------------------------------- in 64 bits ----
@torch.no_grad()
def exact(case, seed):
    """What a pass returns, in double precision from the definitions, unrounded."""
    st = prepare(case, seed)
    return {"emb": _emb_exact, "mlp": _mlp_exact, "lp": _lp_exact}[case["kind"]](st)


def _emb_exact(st):
    c = st["c"]
    out = {"y": st["w"].double()[st["tokens"]] * c["scale"]}
    if c["train"]:
        # running sums over the tokens in order, less those up to the token before
        keep = st["tokens"] != 0
        tokens, order = st["tokens"][keep].sort()
        run_sum = torch.cumsum(st["dy"][keep][order].double(), 0)
        run_sum = torch.cat([run_sum.new_zeros(1, c["D"]), run_sum])
        end = torch.searchsorted(tokens, torch.arange(c["V"], device=tokens.device), right=True)
        begin = torch.cat([end.new_zeros(1), end[:-1]])
        out["dw"] = (run_sum[end] - run_sum[begin]) * c["scale"]
    return out


def _mlp_exact(st):
    c = st["c"]
    names = ("x", "wg", "wu", "wd")
    x, wg, wu, wd = leaves = [st[k].detach().double().requires_grad_(c["train"]) for k in names]
    with torch.enable_grad():
        g = torch.mm(x, wg.T)
        if c["act"] == "silu":
            a = torch.nn.functional.silu(g)
        else:
            a = torch.nn.functional.gelu(g, approximate="tanh" if c["act"] == "gelu_tanh" else "none")
        y = torch.mm(a * torch.mm(x, wu.T), wd.T)
    out = {"y": y.detach()}
    if c["train"]:
        out |= dict(zip(["dx", "dwg", "dwu", "dwd"], torch.autograd.grad(y, leaves, st["dy"].double())))
    return out


def _lp_exact(st):
    c, parts = st["c"], []
    for i in range(0, c["B"], 64):
        rows = slice(i, i + 64)
        z = st["z"][rows].double()
        logp = torch.log_softmax(z, 1)
        p = logp.exp()
        ent = -torch.xlogy(p, p).sum(1)
        part = {"entropy": ent}
        if c["L"]:
            labels = st["labels"][rows]
            none = labels < 0
            part["log_probs"] = logp.gather(1, labels.masked_fill(none, 0)).masked_fill(none, 0.0)
        if c["top"]:
            order = torch.sort(z, dim=1, descending=True, stable=True).indices[:, : c["top"]]
            part |= {"top_log_probs": logp.gather(1, order), "top_labels": order}
        if c["train"]:
            dlp = st["dlp"][rows].double().masked_fill(none, 0.0)
            # d lp_l / dz = [l] - p,  d entropy / dz = -p (log p + entropy)
            dz = torch.xlogy(p, p).add_(p * ent[:, None]).mul_(-st["dent"][rows].double()[:, None])
            dz -= p * dlp.sum(1, keepdim=True)
            part["dz"] = dz.scatter_add(1, labels.masked_fill(none, 0), dlp)
        parts.append(part)
    return {k: torch.cat([q[k] for q in parts]) for k in parts[0]}
