"""The 4-bit paged cache in plain numpy and 64 bits, written from its
definition: the quantizer (with the fp32 and fp16 roundings the definition
names), the record, the page bounds, the page choice and the attention."""
from __future__ import annotations

import numpy as np

PAGE, GROUP = 64, 32
F32, F16 = np.float32, np.float16


def quantize(x):
    """(codes, scale, min) of ``x`` [..., D]: codes [..., D] int, scale/min fp16
    [..., D / 32]; a group that does not fit is (0, nan, nan)."""
    x = np.asarray(x, np.float64)
    g = x.reshape(*x.shape[:-1], x.shape[-1] // GROUP, GROUP)
    with np.errstate(all="ignore"):
        lo, hi = g.min(-1), g.max(-1)
        s = ((hi - lo).astype(F32).astype(np.float64) * float(F32(1.0 / 15.0))).astype(F32).astype(F16)
        z = lo.astype(F32).astype(F16)
        bad = ~(np.isfinite(s) & np.isfinite(z))
        s64, z64 = s.astype(np.float64), z.astype(np.float64)
        r = np.where(s64 > 0, (1.0 / np.where(s64 > 0, s64, 1.0)).astype(F32).astype(np.float64), 0.0)
        c = ((g - z64[..., None]).astype(F32).astype(np.float64) * r[..., None]).astype(F32)
        c = np.clip(np.rint(np.where(np.isfinite(c), c, 0)), 0, 15).astype(np.int64)
    c[bad] = 0
    s[bad] = np.nan
    z[bad] = np.nan
    return c.reshape(x.shape), s, z


def stored(x):
    """fp32 values the cache holds for ``x``."""
    c, s, z = quantize(x)
    with np.errstate(all="ignore"):
        v = c.reshape(*c.shape[:-1], c.shape[-1] // GROUP, GROUP) * s.astype(np.float64)[..., None] + z.astype(np.float64)[..., None]
        return v.reshape(c.shape).astype(F32)


def record_values(rec, D):
    """(key, value) fp32 [64, D] of one record (int32 [20 D]), nibble by nibble."""
    w = np.asarray(rec).astype(np.int64) & 0xFFFFFFFF
    key, value = np.zeros((PAGE, D), F32), np.zeros((PAGE, D), F32)

    def param(base, k, G):
        p = int(w[base + k * (D // 32) + G])
        return (float(np.array(p & 0xFFFF, np.uint16).view(F16)), float(np.array(p >> 16, np.uint16).view(F16)))

    for k in range(PAGE):
        for d in range(D):
            G, t, n = d // 32, d % 32 // 8, d % 8
            c = (int(w[k * (D // 8) + t * (D // 32) + G]) >> (4 * n)) & 15
            s, z = param(8 * D, k, G)
            key[k, d] = F32(c * s + z)
            ww, u, g, n = d // 64, d % 64 // 32, d % 32 // 4, d % 4
            c = (int(w[10 * D + k // 8 * D + g * (D // 8) + k % 8 // 2 * (D // 32) + k % 2 * (D // 64) + ww])
                 >> (4 * (4 * u + n))) & 15
            s, z = param(18 * D, k, G)
            value[k, d] = F32(c * s + z)
    return key, value


def exponent(most):
    """Smallest e >= -40 with most <= 127 * 2^e."""
    e = -40
    while most > 127.0 * 2.0 ** e:
        e += 1
    return e


def page_bounds(key):
    """(upper, lower, e) whole numbers of a page's stored Key [64, D]."""
    v = np.where(np.isfinite(key), key, 0).astype(np.float64)
    e = exponent(np.abs(v).max())
    return (np.ceil(v.max(0) / 2.0 ** e).astype(np.int64), np.floor(v.min(0) / 2.0 ** e).astype(np.int64), e)


def choose(q, key, seen, top, sink, recent):
    """Logical pages of one KV head for its queries ``q`` [heads, D] over stored
    Key [tokens, D], of which ``seen`` are visible."""
    n = -(-seen // PAGE)
    slots = sink + recent + top
    if n <= slots:
        return list(range(n)) + [-1] * (slots - n)
    q = np.where(np.isfinite(q), np.asarray(q, np.float64), 0.0)
    f = exponent(np.abs(q).max())
    Q = np.rint(q / 2.0 ** f)
    plus, minus = np.maximum(Q, 0).sum(0), np.minimum(Q, 0).sum(0)
    scores = []
    for p in range(sink, n - recent):
        up, low, e = page_bounds(key[p * PAGE:(p + 1) * PAGE])
        scores.append(F32(float((up * plus + low * minus).sum())) * F32(2.0 ** e))
    order = np.argsort(-np.array(scores, np.float64), kind="stable")[:top]
    return sorted(list(range(sink)) + [sink + int(i) for i in order] + list(range(n - recent, n)))


def attention(q, key, value, scaling, keep):
    """(out, weight) [heads, D] of queries ``q`` [heads, D] over the tokens where
    ``keep``; weight = sum of p |value|, the scale of a rounding of p."""
    q = np.asarray(q, np.float64)
    if not keep.any():
        return np.zeros(q.shape), np.zeros(q.shape)
    k, v = key[keep].astype(np.float64), value[keep].astype(np.float64)
    logits = q @ k.T * scaling
    p = np.exp(logits - logits.max(-1, keepdims=True))
    p /= p.sum(-1, keepdims=True)
    return p @ v, p @ np.abs(v)
