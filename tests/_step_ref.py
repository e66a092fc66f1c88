"""Plain 64-bit forms of sampling and truncation, in numpy (not a test module)."""

from __future__ import annotations

import math

import numpy as np


def kept(z: np.ndarray, ok, temp: float, top_k: int, top_p: float, min_p: float):
    """(tokens kept, in the order of falling z and rising index; their weights)
    of one row of float64 logits; nothing where there is no softmax."""
    if not ok.any() or np.isnan(z[ok]).any() or np.isposinf(z[ok]).any():
        return np.zeros(0, np.int64), np.zeros(0)
    tokens = np.nonzero(ok & ~np.isneginf(z))[0]
    if len(tokens) == 0:
        return tokens, np.zeros(0)
    tokens = tokens[np.argsort(-z[tokens], kind="stable")]
    if not (temp > 0 and math.isfinite(temp)):
        return tokens[:1], np.ones(1)
    if top_k > 0:
        tokens = tokens[:top_k]
    x = z[tokens]
    w = np.exp((x - x[0]) / temp)
    n = len(w)
    if top_p < 1:
        n = max(1, 1 + int((np.cumsum(w)[:-1] < max(top_p, 0.0) * w.sum()).sum()))
    if min_p > 0:
        n = min(n, int((x - x[0] >= temp * math.log(min(min_p, 1.0))).sum()))
    return tokens[:n], w[:n]


def draw(tokens, w, u: float):
    """(token, log-probability)."""
    if len(tokens) == 0:
        return -1, -math.inf
    run = np.cumsum(w)
    at = min(int((run <= u * run[-1]).sum()), int(np.nonzero(w)[0][-1]))
    return int(tokens[at]), math.log(w[at]) - math.log(run[-1])


def per_row(x, B: int):
    return [float(v) for v in (x if np.ndim(x) else [x] * B)]


def rows(logits, B, V, asked, allow=None):
    """Kept tokens and weights of every row; ``allow`` [B, V] of bools."""
    t, k, p, m = (per_row(x, B) for x in asked)
    return [kept(logits[b, :V], np.ones(V, bool) if allow is None else allow[b], t[b], int(k[b]), p[b], m[b])
            for b in range(B)]
