"""float64 numpy restatement of attention under a sliding window with sinks, and
of the 4-bit paged cache it may read.

Test infrastructure only.  The query at position p sees t <= p where
t > p - window (window 0: every one) or t < sinks.  A query that sees nothing is 0
with lse -inf.  Of the 4-bit cache's format: ``pagelora_amd/kv4.py``.
"""

from __future__ import annotations

import numpy as np

from .paged_decode import _f64

LEVELS = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])


def quantize(x):
    """x [..., D] float64 -> (codes [..., D] uint8, scale bytes [..., D / 32] uint8)."""
    g = _f64(x).reshape(*x.shape[:-1], -1, 32)
    top = np.abs(g).max(-1)
    held = np.isfinite(top)
    with np.errstate(divide="ignore", invalid="ignore"):
        e = np.where(held & (top > 0), np.ceil(np.log2(np.where(held, top, 1.0) / 6.0)), 0.0)
    e = np.clip(e, -125, 125)
    y = np.where(held[..., None], g, 0.0) / np.exp2(e)[..., None]
    a = np.minimum(np.abs(y), 6.0)
    step = np.where(a < 2, 0.5, np.where(a < 4, 1.0, 2.0))
    level = np.minimum(np.round(a / step) * step, 6.0)
    codes = np.searchsorted(LEVELS, level).astype(np.uint8) + 8 * (np.signbit(y) & held[..., None]).astype(np.uint8)
    scales = np.where(held, e + 127, 255).astype(np.uint8)
    return codes.reshape(x.shape), scales


def values(codes, scales):
    """What codes [..., D] and scale bytes [..., D / 32] stand for."""
    v = LEVELS[codes & 7] * np.where(codes & 8, -1.0, 1.0)
    power = np.where(scales == 255, np.nan, np.exp2(scales.astype(np.float64) - 127))
    return (v.reshape(*v.shape[:-1], -1, 32) * power[..., None]).reshape(v.shape)


def pack_pages(kc, ks, vc, vs):
    """Codes [P, page, Hkv, D] and scales [P, page, Hkv, D / 32] of K and V -> a layer uint8 [P, 2, Hkv, bytes]."""
    p, page, hkv, d = kc.shape
    pair = lambda c: (c[..., 0::2] | (c[..., 1::2] << 4)).astype(np.uint8)  # noqa: E731
    k = np.concatenate([pair(kc).transpose(0, 2, 1, 3).reshape(p, hkv, -1), ks.transpose(0, 2, 1, 3).reshape(p, hkv, -1)], 2)
    v = pair(vc).reshape(p, page // 4, 4, hkv, d // 8, 4).transpose(0, 3, 1, 4, 2, 5).reshape(p, hkv, -1)
    s = vs.reshape(p, page // 4, 4, hkv, d // 32).transpose(0, 3, 1, 4, 2).reshape(p, hkv, -1)
    return np.stack([k, np.concatenate([v, s], 2)], 1)


def sees(p, n, window, sinks):
    """The positions of n that the query at p sees."""
    t = np.arange(n)
    seen = t <= p
    if window:
        seen &= (t > p - window) | (t < sinks)
    return np.flatnonzero(seen)


def attend(q, k, v, window, sinks, sm_scale):
    """q [n, Hq, D], the last n positions of k and v [kv_len, Hkv, D].  Returns (o [n, Hq, D], lse [n, Hq], spread
    [n, Hq, D]: the weighted mean of |v|, reach [n, Hq]: the largest sum |q||k| s of a score)."""
    q, k, v = _f64(q), _f64(k), _f64(v)
    n, hq, d = q.shape
    kv_len, hkv, _ = k.shape
    g = hq // hkv
    o, lse = np.zeros((n, hq, d)), np.full((n, hq), -np.inf)
    spread, reach = np.zeros((n, hq, d)), np.zeros((n, hq))
    for i in range(n):
        at = sees(kv_len - n + i, kv_len, window, sinks)  # the others do not enter, whatever they hold
        if at.size == 0:
            continue
        for h in range(hq):
            kk, vv = k[at, h // g], v[at, h // g]
            s = kk @ q[i, h] * sm_scale
            m = s.max()
            p = np.exp(s - m)
            odd = ~np.isfinite(vv)
            with np.errstate(invalid="ignore"):
                o[i, h] = p @ np.where(odd, 0.0, vv) / p.sum() + np.where(odd, vv, 0.0).sum(0)
                lse[i, h] = m + np.log(p.sum())
                spread[i, h] = p @ np.where(odd, 0.0, np.abs(vv)) / p.sum()
                reach[i, h] = (np.abs(kk) @ np.abs(q[i, h])).max() * abs(sm_scale)
    return o, lse, spread, reach
