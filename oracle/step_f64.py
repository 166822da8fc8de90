"""Float64 restatement of the ends of a training step: linear cross entropy, token embedding, norm and clip.

Plain numpy on the definitions; with each result the sums of magnitudes its error bound is made of.
"""
from __future__ import annotations

import numpy as np


def linear_cross_entropy(x, w, targets, ignore_index=-1, reduction="mean", grad=None):
    """``x [n, d]``, ``w [V, d]``, ``targets [n]`` -> dict of the loss, its gradients for an upstream ``grad`` (default 1),
    and: ``logit_sum`` the largest sum of |x w| of a logit, ``dx_sum`` / ``dw_sum`` the sums of |dl w| / |dl x|, ``dx_p`` / ``dw_p``
    those of (|g| p) |w| / (|g| p) |x|."""
    x, w = np.asarray(x, np.float64), np.asarray(w, np.float64)
    keep = np.flatnonzero(np.asarray(targets) != ignore_index)
    n, V = x.shape[0], w.shape[0]
    xs, ts = x[keep], np.asarray(targets)[keep]
    logits = xs @ w.T
    top = logits.max(axis=1, keepdims=True) if len(keep) else np.zeros((0, 1))
    e = np.exp(logits - top)
    total = e.sum(axis=1, keepdims=True)
    each = np.zeros(n)
    each[keep] = (top + np.log(total))[:, 0] - logits[np.arange(len(keep)), ts]
    if reduction == "none":
        loss, g = each, np.ones(n) if grad is None else np.asarray(grad, np.float64)
    else:
        scale = 1.0 if grad is None else float(grad)
        with np.errstate(invalid="ignore", divide="ignore"):
            loss = each.sum() / len(keep) if reduction == "mean" else each.sum()
        g = np.full(n, scale / max(len(keep), 1) if reduction == "mean" else scale)
    p = e / total * g[keep][:, None] if len(keep) else e
    dl = p.copy()
    dl[np.arange(len(keep)), ts] -= g[keep]
    out = {"loss": loss, "each": each, "dx": np.zeros(x.shape), "dw": dl.T @ xs, "dx_sum": np.zeros(x.shape),
           "dw_sum": np.abs(dl).T @ np.abs(xs), "dx_p": np.zeros(x.shape), "dw_p": np.abs(p).T @ np.abs(xs),
           "logit_sum": float((np.abs(xs) @ np.abs(w).T).max()) if len(keep) else 0.0}
    out["dx"][keep], out["dx_sum"][keep], out["dx_p"][keep] = dl @ w, np.abs(dl) @ np.abs(w), np.abs(p) @ np.abs(w)
    return out


def embedding_backward(g, ids, rows, scale=1.0, padding=None):
    """``dw [rows, d]`` of ``scale * w[ids]``, and the sums of magnitudes of its elements' summands."""
    g, ids = np.asarray(g, np.float64), np.asarray(ids)
    dw, size = np.zeros((rows, g.shape[1])), np.zeros((rows, g.shape[1]))
    for i, v in enumerate(ids):
        if 0 <= v < rows and v != padding:
            dw[v] += scale * g[i]
            size[v] += abs(scale) * np.abs(g[i])
    return dw, size


def clip(grads, max_norm, norm=2.0):
    """(norm, clipped gradients) of a list of arrays."""
    flat = np.concatenate([np.asarray(g, np.float64).ravel() for g in grads])
    total = np.sqrt((flat * flat).sum()) if norm == 2.0 else np.abs(flat).max()
    factor = max_norm / (total + 1e-6)
    if factor >= 1.0:
        factor = 1.0
    return total, [np.asarray(g, np.float64) * factor for g in grads]
