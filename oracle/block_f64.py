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


def gated_ffn(x, w_gate, w_up, w_down, kind="silu", dy=None, step=0.0):
    """dict of ``y`` and, for an upstream ``dy``, ``dx``, ``dw_gate``, ``dw_up``, ``dw_down``; ``noise_*``: the standard deviation that these have when h, dg
    and du are rounded independently, each by a standard deviation of ``step`` of its value (so with 1 it is to be scaled), and ``size_*``: the sums of their summands' magnitudes."""
    x, wg, wu, wd = (np.asarray(t, np.float64) for t in (x, w_gate, w_up, w_down))
    g, u = x @ wg.T, x @ wu.T
    a, da = activation(g, kind)
    h = a * u
    out = {"y": h @ wd.T, "noise_y": step * np.sqrt((h * h) @ (wd * wd).T), "g": g, "u": u, "h": h}
    # what an error of g or u in proportion to their own summands does to h, dg and du
    size_g, size_u = np.abs(x) @ np.abs(wg).T, np.abs(x) @ np.abs(wu).T
    size_h = np.abs(h) + 1.2 * size_g * np.abs(u) + np.abs(a) * size_u
    out["size_y"] = size_h @ np.abs(wd).T
    if dy is None:
        return out
    dy = np.asarray(dy, np.float64)
    dh = dy @ wd
    du, dg = dh * a, dh * u * da
    size_dh = np.abs(dy) @ np.abs(wd)
    size_du = size_dh * (np.abs(a) + 1.2 * size_g)
    size_dg = size_dh * (np.abs(u * da) + 1.2 * size_u + 1.2 * np.abs(u) * size_g)      # |f'| < 1.2, |f''| < 1.2
    out.update(dx=dg @ wg + du @ wu, dw_gate=dg.T @ x, dw_up=du.T @ x, dw_down=dy.T @ h, dg=dg, du=du)
    out["size_dx"] = size_dg @ np.abs(wg) + size_du @ np.abs(wu)
    out["size_dw_gate"], out["size_dw_up"], out["size_dw_down"] = size_dg.T @ np.abs(x), size_du.T @ np.abs(x), np.abs(dy).T @ size_h
    sq = np.square
    out["noise_dx"] = step * np.sqrt(sq(dg) @ sq(wg) + sq(du) @ sq(wu))
    out["noise_dw_gate"], out["noise_dw_up"] = step * np.sqrt(sq(dg).T @ sq(x)), step * np.sqrt(sq(du).T @ sq(x))
    out["noise_dw_down"] = step * np.sqrt(sq(dy).T @ sq(h))
    return out
