"""Float64 restatement of a recurrent block's parts: the gated linear recurrence and the gated feed-forward layer.

Plain numpy on the definitions, step by step; with each result the magnitudes its error bound is made of.
"""
from __future__ import annotations

import math

import numpy as np


def _sigmoid(x):
    e = np.exp(-np.abs(x))
    return np.where(x >= 0, 1 / (1 + e), e / (1 + e))


def gated_scan(gate, value, state=None, activation="none", reset=None, lengths=None, dh=None, dlast=None):
    """dict of ``h``, ``last``, ``dgate``, ``dvalue``, ``dstate`` for upstream gradients (default zeros), ``[B, T, D]`` / ``[B, D]``, and their
    magnitudes ``size_*``: the recurrence of absolute values, in which nothing cancels; ``memory``, the longest 1 / s of a step that counts."""
    z, v = np.asarray(gate, np.float64), np.asarray(value, np.float64)
    B, T, D = z.shape
    h0 = np.zeros((B, D)) if state is None else np.asarray(state, np.float64)
    dh = np.zeros((B, T, D)) if dh is None else np.asarray(dh, np.float64)
    dlast = np.zeros((B, D)) if dlast is None else np.asarray(dlast, np.float64)
    reset = np.zeros((B, T), bool) if reset is None else np.asarray(reset)
    n = np.full(B, T) if lengths is None else np.clip(np.asarray(lengths), 0, T)
    out = {k: np.zeros((B, T, D)) for k in ("h", "dgate", "dvalue", "size_h", "size_dgate", "size_dvalue")}
    out.update({k: np.zeros((B, D)) for k in ("last", "dstate", "size_last", "size_dstate")})
    out["memory"] = 1.0
    for b in range(B):
        s, a = _sigmoid(z[b, :n[b]]), _sigmoid(-z[b, :n[b]])
        f, df = v[b, :n[b]], np.ones((n[b], D))
        if activation == "positive":
            low = _sigmoid(f)
            f, df = np.where(f < 0, low, f + 0.5), np.where(f < 0, low * (1 - low), 1.0)
        before, size_before = np.zeros((n[b], D)), np.zeros((n[b], D))
        h, size = h0[b], np.abs(h0[b])
        for t in range(n[b]):
            if reset[b, t]:
                h, size = np.zeros(D), np.zeros(D)
            before[t], size_before[t] = h, size
            h, size = a[t] * h + s[t] * f[t], a[t] * size + s[t] * np.abs(f[t])
            out["h"][b, t], out["size_h"][b, t] = h, size
        out["last"][b], out["size_last"][b] = h, size
        q, size = dlast[b], np.abs(dlast[b])
        for t in range(n[b] - 1, -1, -1):
            g, size = q + dh[b, t], size + np.abs(dh[b, t])
            out["dvalue"][b, t], out["size_dvalue"][b, t] = g * s[t] * df[t], size * s[t] * df[t]
            out["dgate"][b, t] = g * (f[t] - before[t]) * s[t] * a[t]
            out["size_dgate"][b, t] = size * (np.abs(f[t]) + size_before[t]) * s[t] * a[t]
            q, size = (np.zeros(D), np.zeros(D)) if reset[b, t] else (a[t] * g, a[t] * size)
        out["dstate"][b], out["size_dstate"][b] = q, size
        if n[b]:
            out["memory"] = max(out["memory"], float(1 / s.min()))
    return out


_erf = np.vectorize(math.erf, otypes=[np.float64])


def activation(g, kind):
    """f(g), f'(g)."""
    if kind == "silu":
        p = _sigmoid(g)
        return g * p, p * (1 + g * (1 - p))
    if kind == "gelu":
        p = 0.5 * (1 + _erf(g / math.sqrt(2)))
        return g * p, p + g * np.exp(-0.5 * g * g) / math.sqrt(2 * math.pi)
    return np.maximum(g, 0), (g > 0).astype(np.float64)
