"""The operators of a speculative step, as cases that can be timed, with their plain forms.

A serving loop that checks a block of drafted tokens in one pass of its model
does three things around the model's own products: the block's keys are
rotated to their positions and appended, with the values, to a paged cache
held in 4 bits; the block's queries attend to that cache; and the block's
logits decide how many of the drafted tokens stand and which token follows
them, under the grammar that the request has to obey.

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
BYTES = {"fp32": 4, "bf16": 2, "fp16": 2, "": 0}
LEVELS = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
# smallest and largest scale byte: half a step of the smallest scale is a
# normal number of the cache's type (a subnormal one in fp16), six steps of
# the largest still finite
SCALE_BYTES = {torch.bfloat16: (2, 252), torch.float16: (104, 140)}


# ------------------------------------------------------------------ cases --
def listed() -> list[dict]:
    return [
        # one interactive request, three drafted tokens of a small draft model
        {"name": "verify 1", "kind": "verify", "rows": 1, "drafts": 3, "vocab": 32_000, "cols": 32_000, "dtype": "bf16",
         "probs": "fp32", "grammar": False, "ragged": False, "greedy": 0},
        # a serving batch under a grammar, drafts of different lengths, a padded lm_head
        {"name": "verify grammar 48", "kind": "verify", "rows": 48, "drafts": 5, "vocab": 151_936, "cols": 152_064,
         "dtype": "bf16", "probs": "fp32", "grammar": True, "ragged": True, "greedy": 0},
        # drafts looked up in the prompt (no probabilities), some requests greedy
        {"name": "verify lookup 97", "kind": "verify", "rows": 97, "drafts": 7, "vocab": 100_003, "cols": 100_003,
         "dtype": "fp16", "probs": "", "grammar": False, "ragged": True, "greedy": 4},
        # the largest batch: five positions of every request, 256 requests
        {"name": "verify 256", "kind": "verify", "rows": 256, "drafts": 4, "vocab": 151_936, "cols": 151_936,
         "dtype": "bf16", "probs": "bf16", "grammar": True, "ragged": False, "greedy": 0},
        # one token of one request: launch latency
        {"name": "append 1", "kind": "append", "rows": 1, "tokens": 1, "start": 700, "heads": 32, "kv_heads": 8, "dim": 128,
         "rotary": 128, "interleaved": False, "page": 16, "dtype": "bf16", "ragged": False},
        # drafted blocks of a batch, half of each head rotated in neighbouring pairs
        {"name": "append drafts 61", "kind": "append", "rows": 61, "tokens": 5, "start": 4_000, "heads": 16, "kv_heads": 16,
         "dim": 64, "rotary": 32, "interleaved": True, "page": 32, "dtype": "fp16", "ragged": True},
        # prompts of different lengths
        {"name": "append prompts 16", "kind": "append", "rows": 16, "tokens": 4_100, "start": 0, "heads": 32, "kv_heads": 8,
         "dim": 128, "rotary": 128, "interleaved": False, "page": 64, "dtype": "bf16", "ragged": True},
        # one token of one request over a short cache
        {"name": "attend 1", "kind": "attend", "rows": 1, "tokens": 1, "length": 1_000, "heads": 32, "kv_heads": 8,
         "dim": 128, "page": 16, "dtype": "bf16"},
        # one request with a very long context
        {"name": "attend long", "kind": "attend", "rows": 1, "tokens": 4, "length": 200_001, "heads": 32, "kv_heads": 4,
         "dim": 128, "page": 64, "dtype": "bf16"},
        # single tokens, a key head for every query head
        {"name": "attend heads 37", "kind": "attend", "rows": 37, "tokens": 1, "length": 2_500, "heads": 16, "kv_heads": 16,
         "dim": 64, "page": 32, "dtype": "fp16"},
        # drafted blocks of a batch
        {"name": "attend drafts 64", "kind": "attend", "rows": 64, "tokens": 5, "length": 4_096, "heads": 32, "kv_heads": 8,
         "dim": 128, "page": 16, "dtype": "bf16"},
        # the largest: long contexts in a batch
        {"name": "attend 32", "kind": "attend", "rows": 32, "tokens": 2, "length": 32_768, "heads": 64, "kv_heads": 8,
         "dim": 128, "page": 64, "dtype": "bf16"},
    ]


def _log(rng, lo: float, hi: float) -> int:
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng) -> dict:
    kind = rng.choice(("verify", "append", "attend"))
    if kind == "verify":
        drafts = rng.randint(1, 9)
        vocab = _log(rng, 5_000, 160_000)
        probs = rng.choice(("fp32", "bf16", "fp16", ""))
        rows = _log(rng, 1, max(1, min(256, 190_000_000 // ((drafts + 1) * vocab))))
        return {"kind": kind, "rows": rows, "drafts": drafts, "vocab": vocab,
                "cols": vocab + rng.choice((0, 0, 1, 77, 128)), "dtype": rng.choice(("fp32", "bf16", "bf16", "fp16")),
                "probs": probs, "grammar": rng.random() < 0.5, "ragged": rng.random() < 0.5,
                "greedy": rng.choice((0, 0, 1, 3))}
    kv_heads = rng.choice((1, 2, 4, 5, 8, 16))
    heads = kv_heads * rng.choice((1, 1, 2, 3, 4, 5, 7, 8))
    dim = rng.choice((64, 96, 128, 128, 128, 192, 256))
    page = rng.choice((16, 32, 64, 128))
    dtype = rng.choice(("bf16", "bf16", "fp16"))
    if kind == "append":
        tokens = _log(rng, 1, 4_100)
        rows = _log(rng, 1, max(1, min(128, 160_000_000 // (tokens * (heads + kv_heads) * dim))))
        return {"kind": kind, "rows": rows, "tokens": tokens, "start": _log(rng, 1, 20_000) - 1, "heads": heads,
                "kv_heads": kv_heads, "dim": dim, "rotary": dim // rng.choice((1, 1, 2)),
                "interleaved": rng.random() < 0.4, "page": page, "dtype": dtype, "ragged": rng.random() < 0.5}
    tokens = rng.choice((1, 1, 2, 3, 4, 5, 8, 9))
    products = 16_000_000_000 // (heads * dim * tokens)
    length = min(_log(rng, 1, 200_000), products)
    most = max(1, min(96, 1_000_000_000 // (length * kv_heads * dim), products // length))
    return {"kind": kind, "rows": _log(rng, 1, most), "tokens": tokens, "length": length, "heads": heads,
            "kv_heads": kv_heads, "dim": dim, "page": page, "dtype": dtype}


def _draft_lens(c) -> list[int]:
    return [c["drafts"] - (i % (c["drafts"] + 1) if c["ragged"] else 0) for i in range(c["rows"])]


def _counts(c) -> list[int]:
    return [c["tokens"] - (i * c["tokens"] // (2 * c["rows"]) if c["ragged"] else 0) for i in range(c["rows"])]


def _lengths(c) -> list[int]:
    """Lengths of the requests, the block's own tokens among them: from the longest down to a half."""
    return [max(1, c["length"] - i * c["length"] // (2 * c["rows"])) for i in range(c["rows"])]


def work(c) -> dict:
    if c["kind"] == "verify":
        rows = sum(n + 1 for n in _draft_lens(c))
        V = c["vocab"]
        # every position's logits, and of the draft's probabilities the one
        # row that the next token is drawn against
        return {"bytes": rows * V * BYTES[c["dtype"]] + c["rows"] * V * BYTES[c["probs"]], "flops": 4 * rows * V}
    D, KV, H = c["dim"], c["kv_heads"], c["heads"]
    held = 2 * (D // 2 + D // 32)  # bytes of one token of one head, keys and values
    if c["kind"] == "append":
        n = sum(_counts(c))
        # q, k and v read, q rotated, the cache written and read back as k and v
        return {"bytes": n * (2 * 2 * H * D + 2 * 2 * KV * D + 2 * KV * held + 2 * 2 * KV * D) + n * 4 * c["rotary"],
                "flops": n * (6 * H * D + 12 * KV * D)}
    n = sum(_lengths(c))
    M = c["rows"] * c["tokens"] * H * D
    return {"bytes": n * KV * held + 2 * 2 * M, "flops": 4 * n * c["tokens"] * H * D}


# ---------------------------------------------------------------- prepare --
def prepare(c, seed):
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    return {"verify": _prepare_verify, "append": _prepare_append, "attend": _prepare_attend}[c["kind"]](c, g)


def _rand(g, *shape):
    return torch.rand(*shape, generator=g, device=DEVICE)


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device=DEVICE)


def _permuted(g, values) -> torch.Tensor:
    return torch.tensor(values, dtype=torch.int32, device=DEVICE)[torch.randperm(len(values), generator=g, device=DEVICE)]


def _prepare_verify(c, g):
    """Logits of a target model, a draft's block sampled from its own
    probabilities (the target's, blurred), uniform numbers, temperatures; the
    tables of a grammar of 40 states whose tokens are few in some states and
    most of the vocabulary in others."""
    B, T, V, C = c["rows"], c["drafts"], c["vocab"], c["cols"]
    logits = (3.0 * _randn(g, B, T + 1, C)).to(DTYPES[c["dtype"]])
    temperature = 0.6 + 0.6 * _rand(g, B)
    if c["greedy"]:
        temperature[::c["greedy"]] = 0.0
    st = {"logits": logits, "temperature": temperature, "draft_lens": _permuted(g, _draft_lens(c)), "vocab": V,
          "tok_next": None, "allow_bits": None, "states": None}
    state = None
    if c["grammar"]:
        S = 40
        share = torch.exp(math.log(2e-4) + (math.log(0.95) - math.log(2e-4)) * _rand(g, S))
        nxt = torch.randint(0, S, (S, V), generator=g, device=DEVICE, dtype=torch.int32)
        tok_next = torch.where(_rand(g, S, V) < share[:, None], nxt, torch.full_like(nxt, -1))
        allowed = torch.nn.functional.pad(tok_next >= 0, (0, -V % 32)).view(S, -1, 32)
        words = (allowed.to(torch.int64) << torch.arange(32, device=DEVICE)).sum(-1)
        st["tok_next"] = tok_next
        st["allow_bits"] = torch.where(words >= 2 ** 31, words - 2 ** 32, words).to(torch.int32)
        state = torch.randint(0, S, (B,), generator=g, device=DEVICE, dtype=torch.int32)
        st["states"] = state.clone()
    probs, tokens = [], []
    for i in range(T):
        z = logits[:, i, :V].float() + 1.2 * _randn(g, B, V)
        if state is not None:
            z = z.masked_fill((tok_next[state.clamp(min=0).long()] < 0) | (state < 0)[:, None], -math.inf)
        q = torch.softmax(z / temperature.clamp(min=0.05)[:, None], -1).nan_to_num(0.0)
        x = (q / -torch.log(_rand(g, B, V).clamp(min=1e-30))).argmax(-1)
        if state is not None:
            state = torch.where(state < 0, state, tok_next[state.clamp(min=0).long(), x])
        tokens.append(x)
        if c["probs"]:
            probs.append(q.to(DTYPES[c["probs"]]))
    st["draft_tokens"] = torch.stack(tokens, 1).to(torch.int32)
    st["draft_probs"] = torch.stack(probs, 1) if c["probs"] else None
    st["uniforms"] = _rand(g, B, T + 1)
    return st


def _tables(c, g, longest: int):
    """(pages, block_table): a pool of pages handed out in random order; the
    pages hold what earlier requests left in them."""
    B, P, D, KV = c["rows"], c["page"], c["dim"], c["kv_heads"]
    per = -(-longest // P)
    N = B * per + 3
    pages = torch.randint(0, 256, (N, KV, P * (D + D // 16)), generator=g, device=DEVICE, dtype=torch.uint8)
    scales = torch.randint(124, 128, (N, KV, P * (D // 16)), generator=g, device=DEVICE, dtype=torch.uint8)
    pages[:, :, P * D:] = scales
    order = torch.randperm(N, generator=g, device=DEVICE)[:B * per]
    return pages, order.view(B, per).to(torch.int32)


def _prepare_append(c, g):
    """A block's queries, keys and values (keys with a few large channels, as
    models have them), where each request stands, and the rotation's tables."""
    B, T, D, KV, H, R = c["rows"], c["tokens"], c["dim"], c["kv_heads"], c["heads"], c["rotary"]
    dt = DTYPES[c["dtype"]]
    starts = [c["start"] - i * c["start"] // (3 * B) for i in range(B)]
    pages, table = _tables(c, g, c["start"] + T)
    large = torch.where(_rand(g, KV, D) < 0.05, 8.0, 1.0)
    angle = torch.arange(c["start"] + T, dtype=torch.float64)[:, None] * \
        (1e4 ** (-torch.arange(0, R, 2, dtype=torch.float64) / R))[None]
    return {"q": _randn(g, B, T, H, D).to(dt), "k": (_randn(g, B, T, KV, D) * large).to(dt),
            "v": _randn(g, B, T, KV, D).to(dt), "pages": pages, "block_table": table,
            "starts": _permuted(g, starts), "counts": _permuted(g, _counts(c)),
            "cos": torch.cos(angle).float().to(DEVICE), "sin": torch.sin(angle).float().to(DEVICE),
            "interleaved": c["interleaved"], "page": c["page"]}


def _prepare_attend(c, g):
    B, T, D, H = c["rows"], c["tokens"], c["dim"], c["heads"]
    pages, table = _tables(c, g, c["length"])
    return {"q": (1.5 * _randn(g, B, T, H, D)).to(DTYPES[c["dtype"]]), "pages": pages, "block_table": table,
            "lengths": _permuted(g, _lengths(c)), "page": c["page"], "kv_heads": c["kv_heads"]}


# -------------------------------------------------------------------- run --
def run(st):
    if "logits" in st:
        return _own_verify(st) if own else _plain_verify(st)
    if "k" in st:
        return _own_append(st) if own else _plain_append(st)
    return _own_attend(st) if own else _plain_attend(st)


def _own_verify(st):
    from bpdecode_amd import ops

    return ops.dense_verify(st["logits"], st["draft_tokens"], st["uniforms"], draft_probs=st["draft_probs"],
                            draft_lens=st["draft_lens"], temperature=st["temperature"], vocab=st["vocab"],
                            tok_next=st["tok_next"], allow_bits=st["allow_bits"], states=st["states"])


def _own_append(st):
    from bpdecode_amd.kv import PagedKV4

    cache = PagedKV4(st["pages"], st["page"], st["k"].shape[3], st["k"].dtype)
    q = cache.append(st["k"], st["v"], st["block_table"], st["starts"], counts=st["counts"], cos=st["cos"], sin=st["sin"],
                     interleaved=st["interleaved"], q=st["q"])
    k, v = cache.read(st["block_table"], st["starts"], st["k"].shape[1], counts=st["counts"])
    return q, k, v


def _own_attend(st):
    from bpdecode_amd.kv import PagedKV4

    cache = PagedKV4(st["pages"], st["page"], st["q"].shape[3], st["q"].dtype)
    return cache.attend(st["q"], st["block_table"], st["lengths"])


def _plain_verify(st):
    """Draft i stands while u_i q_i(x_i) < p_i(x_i); after the last that
    stands, the next token is the first whose running sum of max(p - q, 0)
    (of p, where every draft stands or that sum is nothing) passes the last
    uniform number's share of the whole.  p is the softmax over the tokens
    that the grammar allows, at temperature 0 all on the first largest; q is 1
    on the drafted token where the draft gives no probabilities.  A row that
    allows nothing takes no draft and yields -1.  In 64 bits: a token next to
    a border of the running sum must not depend on the order of the sum."""
    logits, x, u, V = st["logits"], st["draft_tokens"].long(), st["uniforms"].double(), st["vocab"]
    B, T = x.shape
    rows = torch.arange(B, device=x.device)
    z = logits[:, :, :V].double()
    if st["tok_next"] is not None:
        s = [st["states"].long()]
        for i in range(T):
            s.append(torch.where(s[i] < 0, -1, st["tok_next"][s[i].clamp(min=0), x[:, i]].long()))
        s = torch.stack(s, 1)
        z = z.masked_fill((st["tok_next"][s.clamp(min=0)] < 0) | (s < 0)[:, :, None], -math.inf)
    top = z.max(-1, keepdim=True).values
    some = top > -math.inf
    t = st["temperature"].double()[:, None, None]
    w = torch.exp((z - torch.where(some, top, 0.0)) / torch.where(t > 0, t, 1.0))
    first = torch.where((z == top) & some, torch.arange(V, device=x.device), V).min(-1, keepdim=True).values
    w = torch.where(t > 0, w, (torch.arange(V, device=x.device) == first).double())
    p = w / torch.where(some, w.sum(-1, keepdim=True), 1.0)
    px = p[:, :T].gather(2, x[:, :, None])[:, :, 0]
    q = st["draft_probs"]
    qx = torch.ones_like(px) if q is None else q.gather(2, x[:, :, None])[:, :, 0].double()
    stands = (u[:, :T] * qx < px) & (torch.arange(T, device=x.device) < st["draft_lens"][:, None])
    n = stands.long().cumprod(1).sum(1)
    whole = p[rows, n]
    at = n.clamp(max=T - 1)
    if q is None:
        q_n = torch.zeros_like(whole).scatter_(1, x.gather(1, at[:, None]), 1.0)
    else:
        q_n = q[rows, at].double()
    rest = torch.where((n < st["draft_lens"])[:, None], (whole - q_n).clamp(min=0.0), whole)
    rest = torch.where(rest.sum(1, keepdim=True) > 0, rest, whole)
    run_sum = rest.cumsum(1)
    token = (run_sum <= u[:, T:] * run_sum[:, -1:]).sum(1)
    token = torch.where(some[rows, n, 0], token, -1)
    if st["tok_next"] is None:
        return n.int(), token.int()
    last = s[rows, n]
    state = torch.where((last < 0) | (token < 0), -1, st["tok_next"][last.clamp(min=0), token.clamp(min=0)].long())
    return n.int(), token.int(), state.int()


def _rotated(x, cos, sin, interleaved: bool):
    """Pairs of the first 2 * cos.shape[-1] channels turned by their position's
    angle: (a, b) -> (a cos - b sin, b cos + a sin); neighbours with
    ``interleaved``, else channel i and i + R / 2."""
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
    of two s with max|x| <= 7 s (nothing is then off by more than one s, half
    the step between 4 and 6), its codes the nearest levels, ties to the even
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


def _values(codes, scales):
    """float32 values of packed codes [..., D / 2] and scale bytes [..., D / 32]."""
    level = torch.tensor(LEVELS + tuple(-v for v in LEVELS), device=codes.device)
    pair = torch.stack((level.repeat(16), level.repeat_interleave(16)), 1)
    s = torch.exp2(scales.float() - 127.0)
    s = torch.where(scales == 255, math.nan, s)
    return (pair[codes.long()].flatten(-2).unflatten(-1, (-1, 32)) * s[..., None]).flatten(-2)


def _places(table, starts, T: int, page: int):
    """(page, slot) of tokens starts[b] + 0..T-1."""
    pos = starts.long()[:, None] + torch.arange(T, device=table.device)
    block = (pos // page).clamp(max=table.shape[1] - 1)
    return pos, table.long().gather(1, block), pos % page


def _plain_append(st):
    k, v, pages, P = st["k"], st["v"], st["pages"], st["page"]
    B, T, KV, D = k.shape
    dt = k.dtype
    pos, page, slot = _places(st["block_table"], st["starts"], T, P)
    valid = torch.arange(T, device=k.device) < st["counts"][:, None]
    at = pos.clamp(max=st["cos"].shape[0] - 1)
    cos, sin = st["cos"][at], st["sin"][at]
    keep = valid[:, :, None, None]
    q = torch.where(keep, _rotated(st["q"].float(), cos, sin, st["interleaved"]), 0.0).to(dt)
    kc, ks = _quantised(_rotated(k.float(), cos, sin, st["interleaved"]), dt)
    vc, vs = _quantised(v.float(), dt)
    sections = _sections(pages, P, D)
    head = torch.arange(KV, device=k.device)
    where = (page[valid][:, None], head, slot[valid][:, None])
    for part, new in zip(sections, (kc, vc, ks, vs)):
        part[where] = new[valid]
    got = [part[page[:, :, None], head, slot[:, :, None]] for part in sections]
    k = torch.where(keep, _values(got[0], got[2]), 0.0).to(dt)
    v = torch.where(keep, _values(got[1], got[3]), 0.0).to(dt)
    return q, k, v


def _sections(pages, P: int, D: int):
    """The four sections of [..., bytes], views [..., P, width]."""
    half, g = D // 2, D // 32
    ends = (0, P * half, P * D, P * (D + g), P * (D + 2 * g))
    return [pages[..., a:b].unflatten(-1, (P, -1)) for a, b in zip(ends, ends[1:])]


def _plain_attend(st):
    """softmax(q k^T / sqrt(D)) v over the cache: token i of a block of T sees
    the first length - T + 1 + i tokens; one that sees none yields zeros."""
    q, P, KV = st["q"], st["page"], st["kv_heads"]
    B, T, H, D = q.shape
    kc, vc, ks, vs = (x.transpose(1, 2).flatten(2, 3) for x in _sections(st["pages"][st["block_table"].long()], P, D))
    k = _values(kc, ks)
    L = k.shape[2]
    x = q.float().view(B, T, KV, H // KV, D).permute(0, 2, 3, 1, 4).reshape(B, KV, -1, D)
    s = torch.matmul(x, k.transpose(2, 3)) * (1.0 / math.sqrt(D))
    del k
    sees = st["lengths"].long()[:, None] - T + 1 + torch.arange(T, device=q.device)
    seen = torch.arange(L, device=q.device) < sees[:, :, None]
    seen = seen[:, None, None].expand(B, 1, H // KV, T, L).reshape(B, 1, -1, L)
    s = s.masked_fill(~seen, -math.inf)
    top = s.amax(-1, keepdim=True)
    w = torch.exp(s - torch.where(top > -math.inf, top, 0.0))
    whole = w.sum(-1, keepdim=True)
    v = torch.where(seen.any(2)[:, :, :, None], _values(vc, vs), 0.0)
    out = torch.matmul(w, v) / torch.where(whole > 0, whole, 1.0)
    return out.view(B, KV, H // KV, T, D).permute(0, 3, 1, 2, 4).reshape(B, T, H, D).to(q.dtype)


# ------------------------------------------------------------------ exact --
def exact(c, seed):
    """In 64 bits, with numpy for the cache's numbers: None for the verdicts
    and tokens, which are whole."""
    if c["kind"] == "verify":
        return None
    st = prepare(c, seed)
    return _exact_append(c, st) if c["kind"] == "append" else _exact_attend(c, st)


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


def _exact_append(c, st):
    T, R = c["tokens"], c["rotary"]
    dt = DTYPES[c["dtype"]]
    if c["rows"] * T * (c["heads"] + 2 * c["kv_heads"]) * c["dim"] > 60_000_000:
        return None
    pos = st["starts"].cpu().numpy()[:, None] + np.arange(T)
    top = st["cos"].shape[0] - 1
    turn = (st["cos"].double().cpu().numpy() + 1j * st["sin"].double().cpu().numpy())[np.minimum(pos, top)][:, :, None]
    keep = (np.arange(T) < st["counts"].cpu().numpy()[:, None])[:, :, None, None]

    def rotated(x):
        y = x.double().cpu().numpy().copy()
        a, b = (slice(0, R, 2), slice(1, R, 2)) if c["interleaved"] else (slice(0, R // 2), slice(R // 2, R))
        z = (y[..., a] + 1j * y[..., b]) * turn
        y[..., a], y[..., b] = z.real, z.imag
        return y

    def kept(y):
        return _exact_group(y.reshape(-1, 32), dt).reshape(y.shape)

    out = (rotated(st["q"]), kept(rotated(st["k"])), kept(st["v"].double().cpu().numpy()))
    return tuple(torch.from_numpy(np.where(keep, y, 0.0)) for y in out)


def _exact_attend(c, st):
    B, T, H, D, KV, P = c["rows"], c["tokens"], c["heads"], c["dim"], c["kv_heads"], c["page"]
    lens = st["lengths"].tolist()
    if sum(lens) * KV * D > 400_000_000:
        return None
    table = np.array([math.copysign(LEVELS[i & 7], 1.0 if i < 8 else -1.0) for i in range(16)])
    out = torch.zeros(B, T, H, D, dtype=torch.float64)
    half, g = D // 2, D // 32
    for b, L in enumerate(lens):
        blocks = st["pages"][st["block_table"][b, :-(-L // P)].long()].cpu().numpy()
        q = st["q"][b].double().cpu().numpy().reshape(T, KV, H // KV, D)
        for h in range(KV):
            def section(a, width):
                return blocks[:, h, a:a + P * width].reshape(-1, width)[:L]

            def numbers(codes, scales):
                both = np.empty((L, D))
                both[:, 0::2], both[:, 1::2] = table[codes & 15], table[codes >> 4]
                return both * np.repeat(2.0 ** (scales.astype(np.float64) - 127), 32, axis=1)

            k = numbers(section(0, half), section(P * D, g))
            v = numbers(section(P * half, half), section(P * (D + g), g))
            for i in range(T):
                n = L - T + 1 + i
                if n > 0:
                    s = q[i, h] @ k[:n].T / math.sqrt(D)
                    w = np.exp(s - s.max(1, keepdims=True))
                    y = w @ v[:n] / w.sum(1, keepdims=True)
                    out[b, i, h * (H // KV):(h + 1) * (H // KV)] = torch.from_numpy(y)
    return out
