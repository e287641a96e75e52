"""Numpy restatement in 64 bits of the paged 4-bit cache's operators (``starkv.h``,
``starkv_kv4_*``).  Steps that the specification takes in fp32 are taken in 64 bits
and rounded to fp32 (the same result for sums, products and quotients of fp32
numbers); attention is 64-bit throughout."""

from __future__ import annotations

import numpy as np

D, GROUP = 128, 32


def _r32(x):
    return np.asarray(x, np.float64).astype(np.float32).astype(np.float64)


def _r16(x):
    return np.asarray(x, np.float64).astype(np.float32).astype(np.float16).astype(np.float64)


def quantise(x):
    """x (..., 128) -> codes in [-8, 7], s and m per group (..., 4)."""
    x = np.clip(np.asarray(x, np.float64), -65504.0, 65504.0).reshape(*np.shape(x)[:-1], D // GROUP, GROUP)
    lo, hi = x.min(-1), x.max(-1)
    s = _r16(_r32(_r32(hi - lo) / 15.0))
    m = _r16(_r32(lo + 8.0 * s))
    inv = np.where(s > 0, _r32(1.0 / np.where(s > 0, s, 1.0)), 0.0)
    c = np.clip(np.rint(_r32(_r32(x - m[..., None]) * inv[..., None])), -8, 7)
    return c, s, m


def values(x):
    """What x (..., 128) reads back as, in fp32 steps."""
    c, s, m = quantise(x)
    return _r32(s[..., None] * c + m[..., None]).reshape(np.shape(x))


def bounds(page):
    """page (n, 128) of stored key values -> (up, lo, t) of the full page."""
    hi, lo = page.max(0), page.min(0)
    t = _r32(max(np.abs(hi).max(), np.abs(lo).max()) / 127.0)
    if t == 0:
        return np.zeros(D), np.zeros(D), t
    return np.minimum(np.ceil(_r32(hi / t)), 127), np.maximum(np.floor(_r32(lo / t)), -127), t


def select(q, keys, page_size, keep, first=1, last=1):
    """q (columns, 128), keys (n, 128) stored values of one KV head -> page ordinals kept, ascending."""
    n = len(keys)
    pages = -(-n // page_size)
    if pages <= keep:
        return list(range(pages))
    u = _r32(np.abs(q).max(-1) / 127.0)
    a = np.where(u[:, None] > 0, np.rint(_r32(q / np.where(u > 0, u, 1.0)[:, None])), 0.0)
    scores = {}
    for p in range(first, pages - last):
        up, lo, t = bounds(keys[p * page_size:(p + 1) * page_size])
        dot = (np.where(a > 0, a * up, a * lo)).sum(-1)
        scores[p] = float(_r32(_r32(dot * u).max() * t))
    best = sorted(scores, key=lambda p: (-scores[p], p))[:keep - first - last]
    return sorted(list(range(first)) + list(range(pages - last, pages)) + best)


def attend(q, k, v, scaling, keep=None, mask=None):
    """q (Q, G, 128) newest queries of one KV head over stored k / v (n, 128); keep:
    bool (n,) positions of the selected pages.  Returns out (Q, G, 128), lse (Q, G) and
    the softmax weights (Q, G, n)."""
    Q, G, _ = q.shape
    n = len(k)
    out, lse, w = np.zeros((Q, G, D)), np.full((Q, G), -np.inf), np.zeros((Q, G, n))
    for i in range(Q):
        ok = np.arange(n) < n - Q + 1 + i
        if keep is not None:
            ok &= keep
        add = np.zeros(n) if mask is None else np.asarray(mask, np.float64)[:n]
        ok &= add > -np.inf
        if not ok.any():
            continue
        x = q[i] @ k[ok].T * scaling + add[ok]
        top = x.max(-1, keepdims=True)
        e = np.exp(x - top)
        z = e.sum(-1, keepdims=True)
        w[i][:, ok] = e / z
        out[i] = (e / z) @ v[ok]
        lse[i] = (top + np.log(z))[:, 0]
    return out, lse, w
