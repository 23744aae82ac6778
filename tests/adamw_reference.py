"""AdamW's step and its random bits in float64 and integers (numpy), apart from the library."""
import numpy as np

BLOCK = 128


def philox(c0, c1, c2, key):
    """Philox4x32-10 words [n, 4] of counters (c0, c1, c2, 0), uint64 arithmetic."""
    m32 = np.uint64(0xFFFFFFFF)
    x = [np.asarray(v, dtype=np.uint64) * np.ones_like(np.asarray(c0, dtype=np.uint64))
         for v in (c0, c1, c2, 0)]
    k0, k1 = key & 0xFFFFFFFF, key >> 32
    for _ in range(10):
        p0, p1 = x[0] * np.uint64(0xD2511F53), x[2] * np.uint64(0xCD9E8D57)
        x = [(p1 >> np.uint64(32)) ^ x[1] ^ np.uint64(k0), p1 & m32,
             (p0 >> np.uint64(32)) ^ x[3] ^ np.uint64(k1), p0 & m32]
        k0, k1 = (k0 + 0x9E3779B9) & 0xFFFFFFFF, (k1 + 0xBB67AE85) & 0xFFFFFFFF
    return np.stack(x, 1).astype(np.int64)


def draws(i, bits, stream, seed):
    """(r, r_m, r_u): 16-bit draws of elements i for w, m and u."""
    i = np.asarray(i, dtype=np.int64)
    k = i // (4 if bits == 8 else 8)
    q = philox(k & 0xFFFFFFFF, k >> 32, stream, seed)
    at = np.arange(len(i))
    if bits == 32:
        return (q[at, (i & 7) >> 1] >> (16 * (i & 1))) & 0xFFFF, None, None
    return q[at, i & 3] & 0xFFFF, q[at, i & 3] >> 16, q[at, (i + 1) & 3] >> 16


def cut(x, up, mant, low):
    """(x rounded to its spacing with `up` in [0, 1), that spacing)."""
    with np.errstate(all="ignore"):
        unit = np.exp2(np.maximum(np.frexp(np.abs(x))[1] - 1, low).astype(np.float64) - mant)
        return np.copysign(np.floor(np.abs(x) / unit + up) * unit, x), unit


def scale_exponent(top):
    """Exponent of the power of two that puts `top` in [128, 256)."""
    return np.where(top > 0, np.maximum(np.frexp(top)[1] - 1 - 7, -126), -126)


def quantise(x, r, keep):
    """(values, spacing) of x as 8-bit codes hold it, x padded to whole blocks."""
    b = x.reshape(-1, BLOCK)
    fin = np.where(np.isfinite(b), np.abs(b), 0.0)
    s = np.exp2(scale_exponent(fin.max(1)).astype(np.float64))[:, None]
    v, unit = cut(b / s, r.reshape(-1, BLOCK) / 65536.0, 3, -6)
    if keep:
        v = np.where((b > 0) & (v == 0), 2.0 ** -9, v)
    v = np.where(np.isfinite(b), v, np.nan)
    return (v * s).reshape(-1), (unit * s).reshape(-1)


def step(w, g, m, v, t, lr, b1, b2, eps, wd):
    """(w', m', v') of float64 arrays."""
    with np.errstate(all="ignore"):
        m = b1 * m + (1 - b1) * g
        v = b2 * v + (1 - b2) * g * g
        w = w * (1 - lr * wd) - lr / (1 - b1 ** t) * m / (np.sqrt(v / (1 - b2 ** t)) + eps)
    return w, m, v
