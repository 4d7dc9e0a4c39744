"""Position rotation, paged-cache append and paged attention restated in float64 — TEST
INFRASTRUCTURE (see ``oracle/__init__.py``; the reference tree has none of these operators, so
the definitions are the ones include/lvb.h states)."""
from __future__ import annotations

import numpy as np


def rotate(x, pos, freqs, sections=None, layout="halves", inverse=False):
    """x [..., D] with pos [axes, ...] (x's leading dimensions, broadcastable) -> float64."""
    x = np.asarray(x, dtype=np.float64)
    freqs = np.asarray(freqs, dtype=np.float64)
    n = len(freqs)
    axis = np.repeat(np.arange(len(sections or [n])), sections or [n])
    y = x.copy()
    for i in range(n):
        a = pos[axis[i]].astype(np.float64) * freqs[i]
        c, s = np.cos(a), np.sin(-a if inverse else a)
        j, k = (i, i + n) if layout == "halves" else (2 * i, 2 * i + 1)
        y[..., j] = x[..., j] * c - x[..., k] * s
        y[..., k] = x[..., k] * c + x[..., j] * s
    return y


def attention_one(q, k, v, lens, qlens, prefix, causal, scale):
    """One sequence and KV head. q [qlen, group, D]; k, v [prefix + len, D] -> O, lse float64."""
    q, k, v = (np.asarray(a, dtype=np.float64) for a in (q, k, v))
    s = np.einsum("qgd,ld->qgl", q, k) * scale
    i = np.arange(qlens)[:, None]
    j = np.arange(prefix + lens)[None, :]
    seen = (j < prefix) | ((j - prefix <= lens - qlens + i) if causal else np.ones_like(j, dtype=bool))
    s = np.where(seen[:, None, :], s, -np.inf)
    if s.shape[-1] == 0:
        return np.zeros_like(q), np.full(q.shape[:2], -np.inf)
    m = s.max(-1, keepdims=True)
    p = np.exp(s - np.where(np.isfinite(m), m, 0.0))
    l = p.sum(-1, keepdims=True)
    O = np.where(l > 0, np.einsum("qgl,ld->qgd", p, v) / np.where(l > 0, l, 1), 0.0)
    lse = np.where(l > 0, np.where(np.isfinite(m), m, 0.0) + np.log(np.where(l > 0, l, 1)), -np.inf)
    return O, lse[..., 0]
