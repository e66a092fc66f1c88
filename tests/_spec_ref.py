"""Plain 64-bit forms of the speculative step's operators, in numpy (not a
test module): verification of drafts, the 4-bit cache, attention over it."""

from __future__ import annotations

import math

import numpy as np
import torch

LEVELS = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])
SCALE_BYTES = {torch.bfloat16: (2, 252), torch.float16: (104, 140)}


# ------------------------------------------------------------------ verify --
def verify(logits, tokens, uniforms, *, probs=None, lens=None, temps=None, vocab=None, tok_next=None, states=None):
    """(accepted, next_token, next_state or None) as lists; every argument a
    numpy array, logits and probs in float64."""
    B, T = tokens.shape
    V = vocab or logits.shape[2]
    acc, nxt, after = [], [], []
    for b in range(B):
        n_max = T if lens is None else min(max(int(lens[b]), 0), T)
        t = 1.0 if temps is None else float(temps[b])
        s = None if states is None else int(states[b])
        n = 0
        while True:
            ok = np.ones(V, bool)
            if tok_next is not None:
                ok = tok_next[s] >= 0 if 0 <= s < tok_next.shape[0] else np.zeros(V, bool)
            z = np.where(ok, logits[b, n, :V], -np.inf)
            p = None
            if not (np.isnan(z).any() or np.isposinf(z).any() or np.isneginf(z).all()):
                if t > 0 and math.isfinite(t):
                    p = np.exp((z - z.max()) / t)
                    p /= p.sum()
                else:
                    p = (np.arange(V) == int(np.argmax(z))).astype(np.float64)
            x = int(tokens[b, n]) if n < n_max else -1
            inside = 0 <= x < V
            q = np.zeros(V)
            if n < n_max:
                if probs is not None:
                    q = probs[b, n, :V].astype(np.float64)
                elif inside:
                    q[x] = 1.0
            if n == n_max or p is None or not inside or not float(uniforms[b, n]) * q[x] < p[x]:
                break
            if s is not None:
                s = int(tok_next[s, x])
            n += 1
        token = -1
        if p is not None:
            rest = np.maximum(p - q, 0.0) if n < n_max else p
            if not rest.sum() > 0:
                rest = p
            run = np.cumsum(rest)
            token = int(np.searchsorted(run, float(uniforms[b, T]) * run[-1], side="right"))
            token = min(token, int(np.nonzero(rest)[0][-1]))
        acc.append(n)
        nxt.append(token)
        after.append(-1 if s is None or token < 0 or s < 0 else int(tok_next[s, token]))
    return acc, nxt, (None if states is None else after)


# ------------------------------------------------------------------- cache --
def rotated(x: np.ndarray, cos, sin, interleaved: bool) -> np.ndarray:
    """[..., D] float32 by cos/sin float32 [..., R / 2], every product and sum
    rounded to float32."""
    y = x.astype(np.float32).copy()
    h = cos.shape[-1]
    a, b = (slice(0, 2 * h, 2), slice(1, 2 * h, 2)) if interleaved else (slice(0, h), slice(h, 2 * h))
    u, w = y[..., a].copy(), y[..., b].copy()
    y[..., a] = u * cos - w * sin
    y[..., b] = w * cos + u * sin
    return y


def kept(x: np.ndarray, dtype) -> np.ndarray:
    """The values that the cache keeps of float32 [..., D], in float64: each
    group of 32 at the smallest power of two s with max|x| <= 7 s that the type
    holds, rounded to the nearest level, ties to the even code."""
    lo, hi = SCALE_BYTES[dtype]
    g = x.astype(np.float64).reshape(-1, 32)
    out = np.empty_like(g)
    for i, row in enumerate(g):
        most = np.abs(row).max()
        if not np.isfinite(most):
            out[i] = np.nan
            continue
        e = lo - 127
        while e < hi - 127 and most > 7.0 * 2.0 ** e:
            e += 1
        y = np.abs(row) / 2.0 ** e
        d = np.abs(y[:, None] - LEVELS[None])
        best = d.min(1)
        code = np.where(d == best[:, None], np.arange(8)[None] % 2 * 8 + np.arange(8)[None], 99).argmin(1)
        out[i] = np.copysign(LEVELS[code], row) * 2.0 ** e
    return out.reshape(x.shape)


def block_tables(B: int, blocks: int, pages: int, seed: int) -> torch.Tensor:
    """Distinct pages for every block, in random order."""
    g = torch.Generator().manual_seed(seed)
    return torch.randperm(pages, generator=g)[:B * blocks].view(B, blocks).to(torch.int32)


# --------------------------------------------------------------- attention --
def attend(q: np.ndarray, k, v, lengths, dtype, query_lens=None, scale=None):
    """(out, tolerance) in float64 for q [B, T, H, D] and per-request k, v
    [tokens, KV, D] (NaN-free rows of left-out tokens marked by ``None``
    handled by the caller).  The tolerance counts, per element: the weights
    rounded to the type once and the output once (half a step h each, a
    weight below the type's normal range by its smallest step), and float32
    scores: (D + 4) 2^-24 of the sum of |q k|, which moves a weight by that
    share of itself, twice (the weight and the sum)."""
    B, T, H, D = q.shape
    scale = 1.0 / math.sqrt(D) if scale is None else scale
    h = torch.finfo(dtype).eps / 2
    out, tol = np.zeros(q.shape), np.zeros(q.shape)
    for b in range(B):
        KV = k[b].shape[1]
        n = T if query_lens is None else min(int(query_lens[b]), T)
        for i in range(n):
            m = int(lengths[b]) - n + 1 + i
            if m <= 0:
                continue
            for hh in range(H):
                kk, vv = k[b][:m, hh // (H // KV)], v[b][:m, hh // (H // KV)]
                there = ~np.isnan(kk[:, 0]) if np.isnan(kk).any() else slice(None)
                kk, vv = kk[there], vv[there]
                if len(kk) == 0:
                    continue
                s = kk @ q[b, i, hh] * scale
                w = np.exp(s - s.max())
                total = w.sum()
                w = w / total
                out[b, i, hh] = w @ vv
                size = w @ np.abs(vv)
                es = (D + 4) * 2.0 ** -24 * float((np.abs(kk) @ np.abs(q[b, i, hh])).max()) * abs(scale)
                tol[b, i, hh] = h * (size + np.abs(out[b, i, hh])) * 1.01 + 2 * es * size + 1e-6 * size
                tol[b, i, hh] += torch.finfo(dtype).tiny
    return out, tol
