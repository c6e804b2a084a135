"""CPU statement of the paged 4-bit KV cache (test infrastructure only).

The stored format is defined in fp32 with every operation rounded by itself, so
these functions give its bits; attention and scores are in fp64.
"""

from __future__ import annotations

import math

import numpy as np

F32 = np.float32


def quantise(x):
    """fp32 (..., D) -> codes int8 (..., D), scales fp16 (..., D // 32)."""
    g = np.asarray(x, F32).reshape(*x.shape[:-1], x.shape[-1] // 32, 32)
    bad = ~np.isfinite(g).all(-1)
    amax = np.abs(np.where(np.isfinite(g), g, 0)).max(-1)
    s = np.minimum(amax * F32(1.0 / 7.0), F32(65504)).astype(np.float16)
    f = s.astype(F32)[..., None]
    with np.errstate(all="ignore"):
        t = np.where(f > 0, g / np.where(f > 0, f, F32(1)), F32(0))
    codes = np.clip(np.rint(np.where(bad[..., None], F32(0), t)), -7, 7).astype(np.int8)
    return codes.reshape(x.shape), np.where(bad, np.float16(np.nan), s)


def values(codes, scales):
    """fp32 code * scale."""
    g = codes.astype(F32).reshape(*codes.shape[:-1], codes.shape[-1] // 32, 32)
    return (g * scales.astype(F32)[..., None]).reshape(codes.shape)


def head_norm(x, w, eps):
    """fp32 x (..., D) * r * w, the sum of squares as a tree over neighbours."""
    s = (x * x).astype(F32)
    while s.shape[-1] > 1:
        if s.shape[-1] % 2:
            s = np.concatenate([s, np.zeros_like(s[..., :1])], -1)
        s = s[..., 0::2] + s[..., 1::2]
    r = F32(1) / np.sqrt(s * F32(1.0 / x.shape[-1]) + F32(eps))
    return x * r * w.astype(F32)


def rotate(x, cs, interleaved):
    """fp32 x (n, H, D); cs (n, R) cosines then sines of each token."""
    R = cs.shape[-1]
    c, s = cs[:, None, : R // 2], cs[:, None, R // 2:]
    y = x.copy()
    i = (slice(0, R, 2), slice(1, R, 2)) if interleaved else (slice(0, R // 2), slice(R // 2, R))
    a, b = x[..., i[0]], x[..., i[1]]
    y[..., i[0]] = a * c - b * s
    y[..., i[1]] = b * c + a * s
    return y


def exponent(amax, least):
    """Smallest integer e >= least with amax <= 127 * 2^e."""
    e = least
    if amax > 0:
        e = max(least, math.frexp(float(amax))[1] - 8)
    while float(amax) > 127 * 2.0 ** e:
        e += 1
    return e


def bounds(held):
    """fp32 keys (n, D) of a page and head -> int8 (2, D), exponent."""
    lo, hi = held.min(0).astype(np.float64), held.max(0).astype(np.float64)
    e = exponent(np.abs(held).max(), -40)
    return np.stack([np.floor(lo * 2.0 ** -e), np.ceil(hi * 2.0 ** -e)]).astype(np.int8), e


def attend(q, k, v, seen=None, scale=None):
    """q (G, D), k and v (n, D): the softmax attention and the log of its sum; `seen`
    (n) bool or the number of leading keys."""
    n, D = k.shape
    at = np.arange(n)
    on = np.ones(n, bool) if seen is None else at < seen if np.ndim(seen) == 0 else seen
    if not on.any():
        return np.zeros(q.shape), np.full(len(q), -np.inf)
    a = (q.astype(np.float64) @ k[on].astype(np.float64).T) * (D ** -0.5 if scale is None else scale)
    top = a.max(-1, keepdims=True)
    p = np.exp(a - top)
    return p @ v[on].astype(np.float64) / p.sum(-1, keepdims=True), np.log(p.sum(-1)) + top[:, 0]


def select(q, bound, exps, count, sink, recent):
    """q (G, D), bound (n, 2, D) int8, exps (n): the chosen pages, ascending."""
    n = len(exps)
    if n <= count:
        return list(range(n))
    G, D = q.shape
    e = exponent(np.abs(q).max(), -100) + max(0, math.ceil(math.log2(G * D / 1024)))
    z = np.rint(q.astype(np.float64) * 2.0 ** -e)[:, None]
    score = np.maximum(z * bound[:, 0], z * bound[:, 1]).sum((0, 2)) * 2.0 ** np.asarray(exps, float)
    stay = [p < sink or p >= n - recent for p in range(n)]
    order = sorted(range(n), key=lambda p: (not stay[p], -score[p], p))
    return sorted(order[:count])
