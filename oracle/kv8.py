"""CPU statement of the paged 8-bit KV cache (test infrastructure only).

The stored format is defined in fp32 with every operation rounded by itself, so
these functions give its bits; attention is in fp64.
"""

from __future__ import annotations

import numpy as np

from .kv4 import head_norm, rotate  # noqa: F401  (the same norm and rotation)

F32 = np.float32
BLOCK = 16


def scale(x):
    """The scale of a run of tokens x (n, D): the least power of two s >= 2^-126 with |x| < 128 s."""
    if not np.isfinite(x).all():
        return F32(np.nan)
    top = float(np.abs(x).max()) if x.size else 0.0
    if top == 0.0:
        return F32(0)
    e = -126
    while top >= 128 * 2.0 ** e:
        e += 1
    return F32(2.0 ** e)


def codes(x, s):
    """floor(x / s); zeros where s is 0 or no number."""
    if not s > 0:
        return np.zeros(x.shape, np.int8)
    return np.floor(x.astype(np.float64) / float(s)).astype(np.int8)


def quantise(x):
    """fp32 (n, Hk, D) from a run's first position on -> codes int8 (n, Hk, D), scales fp32 (runs, Hk)."""
    n, Hk, D = x.shape
    c = np.zeros(x.shape, np.int8)
    s = np.zeros((-(-n // BLOCK), Hk), F32)
    for r in range(len(s)):
        at = slice(r * BLOCK, (r + 1) * BLOCK)
        for h in range(Hk):
            s[r, h] = scale(x[at, h])
            c[at, h] = codes(x[at, h], s[r, h])
    return c, s


def values(c, s):
    """What codes (n, Hk, D) with scales (runs, Hk) stand for, fp32."""
    f = np.repeat(s, BLOCK, 0)[: len(c), :, None]
    with np.errstate(invalid="ignore"):
        return (c.astype(F32) + F32(0.5)) * f


def attention(q, k, v, scale):
    """fp64: q (S, Hq, D) the last S of the tokens, k and v (n, Hk, D) -> (out, log-sums)."""
    S, Hq, D = q.shape
    n, Hk = k.shape[:2]
    out, lse = np.zeros((S, Hq, D)), np.full((S, Hq), -np.inf)
    for i in range(S):
        m = n - (S - 1 - i)
        if m <= 0:
            continue
        for h in range(Hq):
            s = k[:m, h // (Hq // Hk)].astype(np.float64) @ q[i, h].astype(np.float64) * scale
            p = np.exp(s - s.max())
            out[i, h] = p @ v[:m, h // (Hq // Hk)].astype(np.float64) / p.sum()
            lse[i, h] = s.max() + np.log(p.sum())
    return out, lse
