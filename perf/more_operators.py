"""Operators of a serving step next to the speculative one, as cases that can
be timed, with their plain forms.

A loop that writes many documents at once under one long instruction rotates
and appends each block (images in the prompt give a token a position on
several axes), attends to the instruction's keys and to each request's own,
and draws the next token: from the softmax at a temperature, among the tokens
that the grammar allows, cut to the k largest, to the smallest set that holds
a share of the probability, and to those not much less likely than the first.
A loop that verifies drafts under the same cuts needs the cut logits.

The order that cuts and draws go by is that of falling logits, and of rising
index among equal ones.

The cache.  ``pages`` is uint8 [num_pages, kv_heads, bytes]; the block of one
page and head holds page_size tokens as four sections: key codes
[page_size, D / 2], value codes [page_size, D / 2], key scales
[page_size, D / 32], value scales [page_size, D / 32].  An element is an
e2m1 code (element 2j of a token in the low half of byte j), a scale one byte
e that stands for 2^(e - 127), shared by 32 neighbouring elements; e = 255
marks a group that held an infinity or a NaN.  Token p of request b lies in
page block_table[b, p // page_size].
"""

from __future__ import annotations

import math

import numpy as np
import torch

own = False

DEVICE = torch.device("cuda:0" if torch.cuda.is_available() else "cpu")
DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
BYTES = {"fp32": 4, "bf16": 2, "fp16": 2}
LEVELS = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
# smallest and largest scale byte of the cache's type
SCALE_BYTES = {torch.bfloat16: (2, 252), torch.float16: (104, 140)}
# what requests ask for, dealt out to the rows of a batch in turn:
# (temperature, top_k, top_p, min_p); 0, 1.0 and 0.0 leave a cut out
ASKED = {
    "one": [(0.8, 40, 0.95, 0.0)],
    "nucleus": [(1.0, 0, 0.9, 0.0)],
    "plain": [(1.0, 0, 1.0, 0.0)],
    "mixed": [(0.7, 0, 0.9, 0.0), (1.0, 50, 1.0, 0.0), (0.0, 0, 1.0, 0.0), (1.2, 0, 1.0, 0.05), (0.6, 20, 0.8, 0.02),
              (1.0, 0, 1.0, 0.0), (0.9, 1000, 0.98, 0.0)],
}


# ------------------------------------------------------------------ cases --
def listed() -> list[dict]:
    return [
        # one interactive request
        {"name": "sample 1", "kind": "sample", "rows": 1, "vocab": 32_000, "cols": 32_000, "dtype": "bf16", "asked": "one",
         "grammar": False},
        # a serving batch under a grammar, requests that ask for different things, a padded lm_head
        {"name": "sample grammar 48", "kind": "sample", "rows": 48, "vocab": 151_936, "cols": 152_064, "dtype": "bf16",
         "asked": "mixed", "grammar": True},
        # logits that the caller holds in 32 bits, an odd vocabulary
        {"name": "sample fp32 97", "kind": "sample", "rows": 97, "vocab": 100_003, "cols": 100_003, "dtype": "fp32",
         "asked": "mixed", "grammar": False},
        # the largest batch, all by top-p
        {"name": "sample 256", "kind": "sample", "rows": 256, "vocab": 151_936, "cols": 151_936, "dtype": "bf16",
         "asked": "nucleus", "grammar": False},
        # the positions of one drafted block
        {"name": "truncate 5", "kind": "truncate", "rows": 5, "vocab": 50_257, "cols": 50_257, "dtype": "fp16", "asked": "one",
         "grammar": False},
        # the positions of a batch's drafted blocks under a grammar
        {"name": "truncate 160", "kind": "truncate", "rows": 160, "vocab": 151_936, "cols": 151_936, "dtype": "bf16",
         "asked": "mixed", "grammar": True},
        # a few requests that share a short instruction
        {"name": "shared 6", "kind": "shared", "rows": 6, "tokens": 1, "shared": 1_000, "length": 150, "heads": 32, "kv_heads": 8,
         "dim": 128, "page": 16, "dtype": "bf16"},
        # drafted blocks of a batch, a key head for every query head
        {"name": "shared drafts 48", "kind": "shared", "rows": 48, "tokens": 4, "shared": 4_100, "length": 700, "heads": 16,
         "kv_heads": 16, "dim": 64, "page": 32, "dtype": "fp16"},
        # the largest: a long instruction with its documents, many requests
        {"name": "shared 128", "kind": "shared", "rows": 128, "tokens": 1, "shared": 32_768, "length": 1_000, "heads": 32,
         "kv_heads": 8, "dim": 128, "page": 64, "dtype": "bf16"},
        # one token of each request of a batch that had images in its prompts
        {"name": "axes 24", "kind": "axes", "rows": 24, "tokens": 1, "start": 2_000, "heads": 28, "kv_heads": 4, "dim": 128,
         "rotary": 128, "sections": "blocks", "interleaved": False, "page": 16, "dtype": "bf16"},
        # prompts with images
        {"name": "axes prompts 12", "kind": "axes", "rows": 12, "tokens": 2_900, "start": 0, "heads": 28, "kv_heads": 4, "dim": 128,
         "rotary": 128, "sections": "blocks", "interleaved": False, "page": 64, "dtype": "bf16"},
        # a video's frames, the axes dealt to neighbouring pairs in turn
        {"name": "axes video 3", "kind": "axes", "rows": 3, "tokens": 1_533, "start": 611, "heads": 16, "kv_heads": 8, "dim": 96,
         "rotary": 96, "sections": "turns", "interleaved": True, "page": 32, "dtype": "fp16"},
    ]


def _log(rng, lo: float, hi: float) -> int:
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng) -> dict:
    kind = rng.choice(("sample", "truncate", "shared", "axes"))
    if kind in ("sample", "truncate"):
        vocab = _log(rng, 5_000, 160_000)
        dtype = rng.choice(("fp32", "bf16", "bf16", "fp16"))
        rows = _log(rng, 1, max(1, min(256, 38_000_000 * 2 // (vocab * BYTES[dtype]))))
        return {"kind": kind, "rows": rows, "vocab": vocab, "cols": vocab + rng.choice((0, 0, 1, 77, 128)), "dtype": dtype,
                "asked": rng.choice(tuple(ASKED)), "grammar": rng.random() < 0.5}
    kv_heads = rng.choice((1, 2, 4, 5, 8, 16))
    heads = kv_heads * rng.choice((1, 1, 2, 3, 4, 5, 7, 8))
    dim = rng.choice((64, 96, 128, 128, 128, 192, 256))
    page = rng.choice((16, 32, 64, 128))
    dtype = rng.choice(("bf16", "bf16", "fp16"))
    if kind == "shared":
        tokens = rng.choice((1, 1, 1, 2, 3, 5, 8))
        shared, length = _log(rng, 128, 33_000), _log(rng, tokens, 1_500)
        products = 17_000_000_000 // (heads * dim * tokens * (shared + length))
        held = min(400_000_000 // (length * kv_heads * dim), 1_600_000_000 // (heads * tokens * (shared + length)))
        return {"kind": kind, "rows": _log(rng, 1, max(1, min(160, products, held))), "tokens": tokens, "shared": shared,
                "length": length, "heads": heads, "kv_heads": kv_heads, "dim": dim, "page": page, "dtype": dtype}
    tokens = _log(rng, 1, 3_500)
    rows = _log(rng, 1, max(1, min(96, 120_000_000 // (tokens * (heads + kv_heads) * dim))))
    return {"kind": kind, "rows": rows, "tokens": tokens, "start": _log(rng, 1, 9_000) - 1, "heads": heads,
            "kv_heads": kv_heads, "dim": dim, "rotary": dim // rng.choice((1, 1, 2)),
            "sections": rng.choice(("blocks", "turns")), "interleaved": rng.random() < 0.4, "page": page, "dtype": dtype}


def _lengths(c) -> list[int]:
    """Tokens of the requests, shared ones and the block's own among them: the own ones from the most down to a half."""
    return [c["shared"] + max(c["tokens"], c["length"] - i * c["length"] // (2 * c["rows"])) for i in range(c["rows"])]


def work(c) -> dict:
    if c["kind"] in ("sample", "truncate"):
        n = c["rows"] * c["vocab"]
        # every logit read once; written once where cut logits are asked for
        return {"bytes": n * BYTES[c["dtype"]] + (c["rows"] * c["cols"] * BYTES[c["dtype"]] if c["kind"] == "truncate" else 0)
                + (n // 8 if c["grammar"] else 0), "flops": 4 * n}
    D, KV, H, T = c["dim"], c["kv_heads"], c["heads"], c["tokens"]
    held = 2 * (D // 2 + D // 32)  # bytes of one token of one head, keys and values
    if c["kind"] == "axes":
        n = c["rows"] * T
        # q, k and v read, q rotated, the cache written and read back as k and v
        return {"bytes": n * (2 * 2 * H * D + 2 * 2 * KV * D + 2 * KV * held + 2 * 2 * KV * D + 12),
                "flops": n * (6 * H * D + 12 * KV * D)}
    mine = sum(_lengths(c)) - c["rows"] * c["shared"]
    # the shared tokens read once, each request's own
    return {"bytes": (c["shared"] + mine) * KV * held + 2 * 2 * c["rows"] * T * H * D, "flops": 4 * sum(_lengths(c)) * T * H * D}


# ---------------------------------------------------------------- prepare --
def prepare(c, seed):
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    return {"sample": _prepare_logits, "truncate": _prepare_logits, "shared": _prepare_shared, "axes": _prepare_axes}[c["kind"]](c, g)


def _rand(g, *shape):
    return torch.rand(*shape, generator=g, device=DEVICE)


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device=DEVICE)


def _permuted(g, values) -> torch.Tensor:
    return torch.tensor(values, dtype=torch.int32, device=DEVICE)[torch.randperm(len(values), generator=g, device=DEVICE)]


def _prepare_logits(c, g):
    """Logits with a few likely tokens above a wide rest, what each request
    asks for, uniform numbers; the tables of a grammar of 40 states whose
    tokens are few in some states and most of the vocabulary in others."""
    B, V = c["rows"], c["vocab"]
    logits = 2.0 * _randn(g, B, c["cols"])
    logits += torch.where(_rand(g, B, c["cols"]) < 1e-3, 3.0 * _randn(g, B, c["cols"]).abs(), 0.0)
    asked = [ASKED[c["asked"]][i % len(ASKED[c["asked"]])] for i in range(B)]
    order = torch.randperm(B, generator=g, device=DEVICE)
    t, k, p, m = ([row[j] for row in asked] for j in range(4))
    st = {"kind": c["kind"], "logits": logits.to(DTYPES[c["dtype"]]), "vocab": V, "uniforms": _rand(g, B),
          "temperature": torch.tensor(t, device=DEVICE)[order], "top_k": torch.tensor(k, dtype=torch.int32, device=DEVICE)[order],
          "top_p": torch.tensor(p, device=DEVICE)[order], "min_p": torch.tensor(m, device=DEVICE)[order],
          "tok_next": None, "allow_bits": None, "states": None}
    if c["grammar"]:
        S = 40
        share = torch.exp(math.log(2e-4) + (math.log(0.95) - math.log(2e-4)) * _rand(g, S))
        nxt = torch.randint(0, S, (S, V), generator=g, device=DEVICE, dtype=torch.int32)
        tok_next = torch.where(_rand(g, S, V) < share[:, None], nxt, torch.full_like(nxt, -1))
        allowed = torch.nn.functional.pad(tok_next >= 0, (0, -V % 32)).view(S, -1, 32)
        words = (allowed.to(torch.int64) << torch.arange(32, device=DEVICE)).sum(-1)
        st["tok_next"] = tok_next
        st["allow_bits"] = torch.where(words >= 2 ** 31, words - 2 ** 32, words).to(torch.int32)
        st["states"] = torch.randint(0, S, (B,), generator=g, device=DEVICE, dtype=torch.int32)
    return st


def _pool(g, N, P, KV, D):
    """Pages that hold what the requests wrote: any codes, scales near one."""
    pages = torch.randint(0, 256, (N, KV, P * (D + D // 16)), generator=g, device=DEVICE, dtype=torch.uint8)
    pages[:, :, P * D:] = torch.randint(124, 128, (N, KV, P * (D // 16)), generator=g, device=DEVICE, dtype=torch.uint8)
    return pages


def _prepare_shared(c, g):
    """Block tables as a serving loop keeps them: the pages of the instruction
    first, the same for all requests (its last tokens that fill no page belong
    to each request), then each request's own, in random order."""
    B, T, D, KV, H, P = c["rows"], c["tokens"], c["dim"], c["kv_heads"], c["heads"], c["page"]
    shared = c["shared"] // P * P
    first, per = shared // P, -(-(c["shared"] + max(c["length"], T)) // P) - shared // P
    N = first + B * per + 3
    order = torch.randperm(N, generator=g, device=DEVICE).to(torch.int32)
    table = torch.cat((order[:first].expand(B, first), order[first:first + B * per].view(B, per)), 1).contiguous()
    return {"kind": "shared", "q": (1.5 * _randn(g, B, T, H, D)).to(DTYPES[c["dtype"]]), "pages": _pool(g, N, P, KV, D),
            "prefix": order[:first].clone(), "shared": shared, "block_table": table, "lengths": _permuted(g, _lengths(c)), "page": P,
            "kv_heads": KV}


def _image_positions(c) -> np.ndarray:
    """int32 [3, rows, tokens]: text counts on every axis alike; an image or a
    frame of h x w patches keeps its time and counts rows and columns; what
    follows goes on from the largest position so far."""
    B, T = c["rows"], c["tokens"]
    out = np.zeros((3, B, T), np.int32)
    for b in range(B):
        at, i, n = c["start"] - b * c["start"] // (3 * B), 0, 0
        while i < T:
            text = min(T - i, 37 + 11 * (b % 5))
            out[:, b, i:i + text] = at + np.arange(text)
            at, i = at + text, i + text
            h, w = 12 + (b + n) % 9, 16 + (b + 2 * n) % 13
            grid = np.stack((np.zeros(h * w, np.int64), np.arange(h * w) // w, np.arange(h * w) % w))[:, :T - i]
            if grid.shape[1]:
                out[:, b, i:i + grid.shape[1]] = at + grid
                at, i, n = at + int(grid.max()) + 1, i + grid.shape[1], n + 1
    return out


def _axes(c) -> list[int]:
    """The axis of each channel pair: a quarter of them time and the rest rows
    and columns, in blocks or dealt out in turn."""
    n = c["rotary"] // 2
    if c["sections"] == "turns":
        return [j % 3 for j in range(n)]
    t = n // 4
    h = t + (n - t) // 2
    return [0 if j < t else 1 if j < h else 2 for j in range(n)]


def _prepare_axes(c, g):
    B, T, D, KV, H, R, P = c["rows"], c["tokens"], c["dim"], c["kv_heads"], c["heads"], c["rotary"], c["page"]
    dt = DTYPES[c["dtype"]]
    starts = [c["start"] - i * c["start"] // (3 * B) for i in range(B)]
    per = -(-(c["start"] + T) // P)
    N = B * per + 3
    table = torch.randperm(N, generator=g, device=DEVICE)[:B * per].view(B, per).to(torch.int32)
    large = torch.where(_rand(g, KV, D) < 0.05, 8.0, 1.0)
    positions = torch.from_numpy(_image_positions(c))
    angle = torch.arange(int(positions.max()) + 1, dtype=torch.float64)[:, None] * \
        (1e6 ** (-torch.arange(0, R, 2, dtype=torch.float64) / R))[None]
    return {"kind": "axes", "q": _randn(g, B, T, H, D).to(dt), "k": (_randn(g, B, T, KV, D) * large).to(dt),
            "v": _randn(g, B, T, KV, D).to(dt), "pages": _pool(g, N, P, KV, D), "block_table": table,
            "starts": torch.tensor(starts, dtype=torch.int32, device=DEVICE), "positions": positions.to(DEVICE),
            "axes": torch.tensor(_axes(c), dtype=torch.int32, device=DEVICE), "cos": torch.cos(angle).float().to(DEVICE),
            "sin": torch.sin(angle).float().to(DEVICE), "interleaved": c["interleaved"], "page": P}


# -------------------------------------------------------------------- run --
def run(st):
    if st["kind"] == "sample":
        return _own_sample(st) if own else _plain_sample(st)
    if st["kind"] == "truncate":
        return _own_truncate(st) if own else _plain_truncate(st)
    if st["kind"] == "shared":
        return _own_shared(st) if own else _plain_shared(st)
    return _own_axes(st) if own else _plain_axes(st)


def _own_sample(st):
    from bpdecode_amd import ops

    return ops.dense_sample(st["logits"], st["uniforms"], temperature=st["temperature"], top_k=st["top_k"], top_p=st["top_p"],
                            min_p=st["min_p"], vocab=st["vocab"], tok_next=st["tok_next"], allow_bits=st["allow_bits"],
                            states=st["states"])


def _own_truncate(st):
    from bpdecode_amd import ops

    return ops.dense_truncate(st["logits"], temperature=st["temperature"], top_k=st["top_k"], top_p=st["top_p"],
                              min_p=st["min_p"], vocab=st["vocab"], allow_bits=st["allow_bits"], bit_rows=st["states"])


def _own_shared(st):
    from bpdecode_amd.kv import PagedKV4

    cache = PagedKV4(st["pages"], st["page"], st["q"].shape[3], st["q"].dtype)
    return cache.attend_shared(st["q"], st["prefix"], st["shared"], st["block_table"], st["lengths"])


def _own_axes(st):
    from bpdecode_amd.kv import PagedKV4

    cache = PagedKV4(st["pages"], st["page"], st["k"].shape[3], st["k"].dtype)
    q = cache.append(st["k"], st["v"], st["block_table"], st["starts"], cos=st["cos"], sin=st["sin"], positions=st["positions"],
                     axes=st["axes"], interleaved=st["interleaved"], q=st["q"])
    k, v = cache.read(st["block_table"], st["starts"], st["k"].shape[1])
    return q, k, v


def _order(st):
    """What both forms cut by: (logits in 64 bits in the order of the draw, the
    tokens there, weights, how many are kept).  In 64 bits: a token next to a
    border of a running sum must not depend on the order of the sum."""
    z = st["logits"][:, :st["vocab"]].double()
    if st["allow_bits"] is not None:
        bits = st["allow_bits"][st["states"].long()]
        on = (bits[:, :, None] >> torch.arange(32, dtype=torch.int32, device=z.device)) & 1
        z = z.masked_fill(on.flatten(1)[:, :st["vocab"]] == 0, -math.inf)
    z, token = torch.sort(z, dim=1, descending=True, stable=True)
    top = z[:, :1]
    some = top > -math.inf
    t = st["temperature"].double()[:, None]
    away = (z - torch.where(some, top, 0.0)) / torch.where(t > 0, t, 1.0)
    w = torch.exp(away)
    at = torch.arange(z.shape[1], device=z.device)
    k = st["top_k"].long()[:, None]
    kept = (at < torch.where(k > 0, k, z.shape[1])) & (z > -math.inf)
    w = torch.where(kept, w, 0.0)
    before = w.cumsum(1) - w
    p = st["top_p"].double()[:, None]
    kept &= (p >= 1.0) | (before < p * w.sum(1, keepdim=True))
    m = st["min_p"].double()[:, None]
    kept &= (m <= 0.0) | (away >= torch.log(torch.where(m > 0, m, 1.0)))
    kept = torch.where(t > 0, kept, at < 1) & some
    kept[:, :1] |= some
    return z, token, torch.where(kept, torch.where(t > 0, w, 1.0), 0.0), kept


def _plain_sample(st):
    """(token, log-probability, state after it); -1, -inf, -1 for a row that
    allows nothing."""
    z, token, w, kept = _order(st)
    run_sum = w.cumsum(1)
    whole = run_sum[:, -1:]
    n = (run_sum <= st["uniforms"].double()[:, None] * whole).sum(1, keepdim=True)
    n = torch.minimum(n, kept.sum(1, keepdim=True) - 1).clamp(min=0)
    some = kept[:, 0]
    out = torch.where(some, token.gather(1, n)[:, 0], -1)
    logprob = torch.where(some, torch.log(w.gather(1, n) / torch.where(whole > 0, whole, 1.0))[:, 0], -math.inf).float()
    if st["tok_next"] is None:
        return out.int(), logprob
    state = torch.where(out < 0, -1, st["tok_next"][st["states"].long(), out.clamp(min=0)].long())
    return out.int(), logprob, state.int()


def _plain_truncate(st):
    """The logits of the kept tokens, -inf elsewhere."""
    z, token, w, kept = _order(st)
    cut = torch.full_like(st["logits"], -math.inf)
    keep = torch.zeros_like(kept).scatter_(1, token, kept)
    cut[:, :st["vocab"]] = torch.where(keep, st["logits"][:, :st["vocab"]], -math.inf)
    return cut


def _sections(pages, P: int, D: int):
    """The four sections of [..., bytes], views [..., P, width]."""
    half, g = D // 2, D // 32
    ends = (0, P * half, P * D, P * (D + g), P * (D + 2 * g))
    return [pages[..., a:b].unflatten(-1, (P, -1)) for a, b in zip(ends, ends[1:])]


def _values(codes, scales):
    """float32 values of packed codes [..., D / 2] and scale bytes [..., D / 32]."""
    level = torch.tensor(LEVELS + tuple(-v for v in LEVELS), device=codes.device)
    pair = torch.stack((level.repeat(16), level.repeat_interleave(16)), 1)
    s = torch.where(scales == 255, math.nan, torch.exp2(scales.float() - 127.0))
    return (pair[codes.long()].flatten(-2).unflatten(-1, (-1, 32)) * s[..., None]).flatten(-2)


def _keys_values(st, table):
    """float32 [..., KV, tokens, D] of the pages that ``table`` [..., blocks] names."""
    parts = [x.movedim(-3, -4).flatten(-3, -2) for x in _sections(st["pages"][table.long()], st["page"], st["q"].shape[3])]
    return _values(parts[0], parts[2]), _values(parts[1], parts[3])


def _plain_shared(st):
    """softmax(q k^T / sqrt(D)) v over the shared tokens and each request's
    own: token i of a block of T sees the first length - T + 1 + i tokens."""
    q, KV, S = st["q"], st["kv_heads"], st["shared"]
    B, T, H, D = q.shape
    x = q.float().view(B, T, KV, H // KV, D).permute(2, 0, 3, 1, 4)  # [KV, B, share, T, D]
    x = x * (1.0 / math.sqrt(D))
    k, v = _keys_values(st, st["prefix"])  # [KV, S, D]
    s = torch.matmul(x.reshape(KV, -1, D), k.transpose(1, 2)).view(KV, B, -1, S)
    ok, ov = _keys_values(st, st["block_table"][:, S // st["page"]:])  # [B, KV, own, D]
    mine = torch.matmul(x.transpose(0, 1).reshape(B, KV, -1, D), ok.transpose(2, 3))
    sees = st["lengths"].long()[:, None] - S - T + 1 + torch.arange(T, device=q.device)
    seen = torch.arange(ok.shape[2], device=q.device) < sees[:, :, None]
    mine = mine.view(B, KV, H // KV, T, -1).masked_fill(~seen[:, None, None], -math.inf).view(B, KV, (H // KV) * T, -1)
    mine = mine.transpose(0, 1)
    top = torch.maximum(s.amax(-1, keepdim=True), mine.amax(-1, keepdim=True))
    s, mine = torch.exp(s - top), torch.exp(mine - top)
    whole = s.sum(-1, keepdim=True) + mine.sum(-1, keepdim=True)
    y = torch.matmul(s.view(KV, -1, S), v).view(KV, B, -1, D) + torch.matmul(mine, ov.transpose(0, 1))
    y = (y / whole).view(KV, B, H // KV, T, D)
    return y.permute(1, 3, 0, 2, 4).reshape(B, T, H, D).to(q.dtype)


def _rotated(x, cos, sin, interleaved: bool):
    """Pairs of the first 2 * cos.shape[-1] channels turned by their angle:
    (a, b) -> (a cos - b sin, b cos + a sin); neighbours with ``interleaved``,
    else channel i and i + R / 2."""
    h = cos.shape[-1]
    cos, sin = cos[:, :, None], sin[:, :, None]
    if interleaved:
        a, b = x[..., 0:2 * h:2], x[..., 1:2 * h:2]
        turned = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    else:
        a, b = x[..., :h], x[..., h:2 * h]
        turned = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    return torch.cat((turned, x[..., 2 * h:]), -1)


def _quantised(x, dt):
    """(codes, scale bytes) of [..., D]: a group's scale is the smallest power
    of two s with max|x| <= 7 s, its codes the nearest levels, ties to the even
    code."""
    lo, hi = SCALE_BYTES[dt]
    x = x.unflatten(-1, (-1, 32))
    most = x.abs().amax(-1)
    bits = most.view(torch.int32)
    e = ((bits >> 23) - 2 + ((bits & 0x7FFFFF) > 0x600000).int()).clamp(lo, hi)
    y = x.abs() * ((254 - e) << 23).view(torch.float32)[..., None]
    code = ((y > 0.25).int() + (y >= 0.75).int() + (y > 1.25).int() + (y >= 1.75).int() + (y > 2.5).int()
            + (y >= 3.5).int() + (y > 5.0).int() + 8 * (x < 0).int())
    bad = ~torch.isfinite(most)
    code = torch.where(bad[..., None], 0, code).flatten(-2)
    return (code[..., 0::2] + 16 * code[..., 1::2]).to(torch.uint8), torch.where(bad, 255, e).to(torch.uint8)


def _plain_axes(st):
    """Pair j turned by the angle of the token's position on axis axes[j], then
    appended, and read back."""
    k, v, pages, P = st["k"], st["v"], st["pages"], st["page"]
    B, T, KV, D = k.shape
    dt = k.dtype
    pair = torch.arange(st["axes"].numel(), device=k.device)
    row = st["positions"].long()[st["axes"].long()].permute(1, 2, 0)  # [B, T, R / 2]
    cos, sin = st["cos"][row, pair], st["sin"][row, pair]
    q = _rotated(st["q"].float(), cos, sin, st["interleaved"]).to(dt)
    kc, ks = _quantised(_rotated(k.float(), cos, sin, st["interleaved"]), dt)
    vc, vs = _quantised(v.float(), dt)
    pos = st["starts"].long()[:, None] + torch.arange(T, device=k.device)
    page, slot = st["block_table"].long().gather(1, pos // P), pos % P
    where = (page[:, :, None], torch.arange(KV, device=k.device), slot[:, :, None])
    sections = _sections(pages, P, D)
    for part, new in zip(sections, (kc, vc, ks, vs)):
        part[where] = new
    got = [part[where] for part in sections]
    return q, _values(got[0], got[2]).to(dt), _values(got[1], got[3]).to(dt)


# ------------------------------------------------------------------ exact --
def exact(c, seed):
    """In 64 bits, with numpy: None for tokens and states, which are whole."""
    st = prepare(c, seed)
    if c["kind"] in ("sample", "truncate"):
        return _exact_cut(c, st)
    return _exact_axes(c, st) if c["kind"] == "axes" else _exact_shared(c, st)


def _exact_cut(c, st):
    B, V = c["rows"], c["vocab"]
    logits = st["logits"].double().cpu().numpy()
    asked = [st[n].double().cpu().numpy() for n in ("temperature", "top_k", "top_p", "min_p")]
    u = st["uniforms"].double().cpu().numpy()
    bits = None if st["allow_bits"] is None else st["allow_bits"].cpu().numpy()
    states = None if bits is None else st["states"].cpu().numpy()
    logprobs, cut = np.full(B, -np.inf), np.full(logits.shape, -np.inf) if c["kind"] == "truncate" else None
    for b in range(B):
        t, k, p, m = (x[b] for x in asked)
        there = np.arange(V)
        if bits is not None:
            there = np.nonzero(np.unpackbits(bits[states[b]].view(np.uint8), bitorder="little")[:V])[0]
        z = logits[b, there]
        if not len(z):
            continue
        order = np.argsort(-z, kind="stable")
        if t <= 0:
            order = order[:1]
            t = 1.0
        if k > 0:
            order = order[:int(k)]
        z = z[order]
        w = np.exp((z - z[0]) / t)
        upto = np.cumsum(w)
        n = len(w)
        if p < 1:
            n = min(n, int(np.searchsorted(upto, p * upto[-1], side="left")) + 1)
        if m > 0:
            n = min(n, int(((z - z[0]) >= t * math.log(m)).sum()))
        at = min(int(np.searchsorted(upto[:n], u[b] * upto[n - 1], side="right")), n - 1)
        logprobs[b] = (z[at] - z[0]) / t - math.log(upto[n - 1])
        if cut is not None:
            keep = there[order[:n]]
            cut[b, keep] = logits[b, keep]
    if cut is not None:
        return torch.from_numpy(cut)
    return (None, torch.from_numpy(logprobs)) + ((None,) if bits is not None else ())


def _exact_group(x: np.ndarray, dt) -> np.ndarray:
    """What 4 bits keep of [n, 32] float64."""
    lo, hi = SCALE_BYTES[dt]
    most = np.abs(x).max(1)
    e = np.ceil(np.log2(np.maximum(most, 1e-300) / 7.0))
    e = np.where(most > 7.0 * 2.0 ** e, e + 1, np.where(most <= 7.0 * 2.0 ** (e - 1), e - 1, e))
    s = 2.0 ** np.clip(e, lo - 127, hi - 127)[:, None]
    y = np.minimum(np.abs(x) / s, 6.0)
    step = np.where(y < 2.0, 0.5, np.where(y < 4.0, 1.0, 2.0))
    return np.sign(x) * np.rint(y / step) * step * s


def _exact_axes(c, st):
    T, R = c["tokens"], c["rotary"]
    dt = DTYPES[c["dtype"]]
    if c["rows"] * T * (c["heads"] + 2 * c["kv_heads"]) * c["dim"] > 200_000_000:
        return None
    turn = st["cos"].double().cpu().numpy() + 1j * st["sin"].double().cpu().numpy()
    positions, axes = st["positions"].cpu().numpy(), st["axes"].cpu().numpy()
    a, b = (slice(0, R, 2), slice(1, R, 2)) if c["interleaved"] else (slice(0, R // 2), slice(R // 2, R))

    def kept(y):
        return _exact_group(y.reshape(-1, 32), dt).reshape(y.shape)

    out = []
    for r in range(c["rows"]):
        by = np.stack([turn[positions[x, r], j] for j, x in enumerate(axes)], -1)[:, None]
        q, k = (st[n][r].double().cpu().numpy().copy() for n in ("q", "k"))
        for y in (q, k):
            z = (y[..., a] + 1j * y[..., b]) * by
            y[..., a], y[..., b] = z.real, z.imag
        out.append((q, kept(k), kept(st["v"][r].double().cpu().numpy())))
    return tuple(torch.from_numpy(np.stack(y)) for y in zip(*out))


def _exact_shared(c, st):
    B, T, H, D, KV, P = c["rows"], c["tokens"], c["heads"], c["dim"], c["kv_heads"], c["page"]
    lens, S = st["lengths"].tolist(), st["shared"]
    if sum(lens) * T * H * D > 20_000_000_000:
        return None
    table = np.array([math.copysign(LEVELS[i & 7], 1.0 if i < 8 else -1.0) for i in range(16)])
    half, g = D // 2, D // 32

    def numbers(blocks, h, codes_at, scales_at):
        codes = blocks[:, h, codes_at:codes_at + P * half].reshape(-1, half)
        scales = blocks[:, h, scales_at:scales_at + P * g].reshape(-1, g)
        both = np.empty((len(codes), D))
        both[:, 0::2], both[:, 1::2] = table[codes & 15], table[codes >> 4]
        return both * np.repeat(2.0 ** (scales.astype(np.float64) - 127), 32, axis=1)

    def keys_values(rows, h):
        blocks = st["pages"][rows.long()].cpu().numpy()
        return numbers(blocks, h, 0, P * D), numbers(blocks, h, P * half, P * (D + g))

    out = torch.zeros(B, T, H, D, dtype=torch.float64)
    q = st["q"].double().cpu().numpy().reshape(B, T, KV, H // KV, D) / math.sqrt(D)
    share = H // KV
    for h in range(KV):
        k, v = keys_values(st["prefix"], h)
        at_once = max(1, 16_000_000 // (S * T * share))
        for b0 in range(0, B, at_once):
            mine = q[b0:b0 + at_once, :, h]  # [requests, T, share, D]
            s = (mine.reshape(-1, D) @ k.T).reshape(-1, T, share, S)
            top = s.max(3)
            w = np.exp(s - top[..., None])
            whole, y = w.sum(3), (w.reshape(-1, S) @ v).reshape(mine.shape)
            for b in range(b0, b0 + len(mine)):
                ok, ov = keys_values(st["block_table"][b, S // P:-(-lens[b] // P)], h)
                for i in range(T):
                    n = lens[b] - S - T + 1 + i
                    own_s = mine[b - b0, i] @ ok[:n].T
                    most = np.maximum(own_s.max(1), top[b - b0, i])
                    own_w, less = np.exp(own_s - most[:, None]), np.exp(top[b - b0, i] - most)
                    z = own_w @ ov[:n] + y[b - b0, i] * less[:, None]
                    z /= (own_w.sum(1) + whole[b - b0, i] * less)[:, None]
                    out[b, i, h * share:(h + 1) * share] = torch.from_numpy(z)
    return out
