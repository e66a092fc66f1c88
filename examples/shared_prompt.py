"""Many documents under one prompt, over a 4-bit paged cache.

    python examples/shared_prompt.py [--device cuda] [--requests 4] [--drafts 3]

A small model of random weights reads one instruction with an image in it --
its patches stand at rotary positions of time, height and width -- and then
writes a document of a regular expression for each of several requests.  The
instruction lies in the cache once: every step appends one block per request
behind it, attends to the instruction for all requests at once and to each
request's own tokens, and draws the next token under the grammar, cut by
top-k, top-p and min-p.  With drafts (looked up in what a request has written)
the block's logits are truncated by the same cuts and verified.
"""

from __future__ import annotations

import argparse
import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parent.parent))

from bpdecode_amd import ops  # noqa: E402
from bpdecode_amd.batch import ConstraintBatch  # noqa: E402
from bpdecode_amd.kv import PagedKV4  # noqa: E402
from bpdecode_amd.ops import FsaTensors  # noqa: E402
from examples.speculative import PATTERN, Model, look_up, norm, vocabulary  # noqa: E402

CUTS = {"top_k": 40, "top_p": 0.95, "min_p": 0.01}


def prompt_positions(text: int, height: int, width: int, more: int) -> torch.Tensor:
    """int32 [3, tokens]: text counts on every axis alike, the patches of an
    image keep their time and count rows and columns, and what follows goes on
    from the largest position."""
    t = torch.arange(text).expand(3, text)
    patch = torch.arange(height * width)
    image = text + torch.stack((torch.zeros_like(patch), patch // width, patch % width))
    after = text + max(height, width) + torch.arange(more).expand(3, more)
    return torch.cat((t, image, after), 1).to(torch.int32)


class Reader(Model):
    """The model of the speculative example with positions of three axes and a
    prefix that requests share."""

    def __init__(self, vocab: int, device, **kw) -> None:
        super().__init__(vocab, device, **kw)
        pairs = self.dim // 2
        self.axes = (torch.arange(pairs) * 3 // pairs).to(torch.int32).to(device)

    def block(self, tokens, caches, table, starts, counts, positions, prefix=None, shared: int = 0):
        """Logits [requests, tokens, vocab] of a block of tokens at ``starts``
        in the cache and at ``positions`` [3, requests, tokens]."""
        x = self.embed[tokens]
        H, KV, D = self.heads, self.kv_heads, self.dim
        for w, cache in zip(self.layers, caches):
            q, k, v = ((norm(x) @ w["qkv"]).unflatten(-1, (-1, D)).to(cache.dtype)).split((H, KV, KV), 2)
            q = cache.append(k, v, table, starts, counts=counts, cos=self.cos, sin=self.sin, positions=positions,
                             axes=self.axes, q=q)
            if prefix is None:
                y = cache.attend(q, table, starts + counts, query_lens=counts)
            else:
                y = cache.attend_shared(q, prefix, shared, table, starts + counts, query_lens=counts)
            x = x + y.flatten(2).double() @ w["out"]
            a, b = (norm(x) @ w["up"]).chunk(2, -1)
            x = x + (torch.nn.functional.silu(a) * b) @ w["down"]
        return (norm(x) @ self.head).float()


def generate(model: Reader, fsa: FsaTensors, instruction: list[int], positions: torch.Tensor, requests: list[list[int]], *,
             tokens: int, drafts: int = 0, temperature: float = 0.9, device="cpu", page_size=16, seed=0,
             share: bool = True) -> list[list[int]]:
    """Up to about ``tokens`` tokens for each request behind the instruction;
    without ``share`` attention reads the instruction for each by itself."""
    B, S, eos = len(requests), len(instruction), fsa.eos_id
    first = S // page_size  # pages that are whole: the rest of the instruction is each request's own
    longest = S + max(map(len, requests)) + tokens + drafts + 1
    per = -(-longest // page_size) - first
    g = torch.Generator().manual_seed(seed)
    pages = torch.randperm(first + B * per, generator=g).to(torch.int32)
    prefix = pages[:first].clone().to(device)
    table = torch.cat((pages[:first].expand(B, first), pages[first:].view(B, per)), 1).contiguous().to(device)
    caches = [PagedKV4.empty(first + B * per, page_size, model.kv_heads, model.dim, torch.bfloat16, device)
              for _ in model.layers]
    batch = ConstraintBatch(fsa, capacity=B, device=device)
    ids = list(range(B))
    for i in ids:
        batch.add(i)

    def int32(values):
        return torch.tensor(values, dtype=torch.int32, device=device)

    # The instruction once, up to its last whole page, by the first request's table.
    whole = first * page_size
    if whole:
        model.block(torch.tensor([instruction[:whole]], device=device), caches, table[:1], int32([0]), int32([whole]),
                    positions[:, None, :whole].to(device))
    base = int(positions.max()) + 1  # the rotary position behind the instruction

    def block(rows: list[list[int]], starts: list[int]):
        T = max(map(len, rows))
        padded = torch.tensor([r + [0] * (T - len(r)) for r in rows], device=device)
        places = []
        for start, row in zip(starts, rows):
            at = [positions[:, p] if p < S else torch.full((3,), base + p - S, dtype=torch.int32)
                  for p in range(start, start + len(row))] + [torch.zeros(3, dtype=torch.int32)] * (T - len(row))
            places.append(torch.stack(at, 1))
        shared = {"prefix": prefix, "shared": whole} if share else {}
        return model.block(padded, caches, table, int32(starts), int32([len(r) for r in rows]),
                           torch.stack(places, 1).to(device), **shared)

    def uniforms(n):
        return torch.rand(B, n, generator=g).to(device)

    rows = [instruction[whole:] + r for r in requests]
    last = torch.tensor([len(r) - 1 for r in rows], device=device)
    logits = block(rows, [whole] * B)[torch.arange(B, device=device), last]
    token, _ = batch.sample(ids, logits, uniforms(1)[:, 0], temperature=temperature, **CUTS)
    written = [[t] for t in token.tolist()]
    while any(w[-1] not in (eos, -1) and len(w) < tokens for w in written):
        going = [w[-1] not in (eos, -1) and len(w) < tokens for w in written]
        drafted = [look_up(requests[i] + written[i], drafts) if drafts and going[i] else [] for i in ids]
        rows = [[max(written[i][-1], 0)] + drafted[i] for i in ids]
        starts = [S + len(requests[i]) + len(written[i]) - 1 for i in ids]
        logits = block(rows, starts)
        T = logits.shape[1] - 1
        if T == 0:
            token, _ = batch.sample(ids, logits[:, 0], uniforms(1)[:, 0], temperature=temperature, **CUTS)
            n = [0] * B
        else:
            # the states that the drafts lead to, a row of logits for each
            x = torch.tensor([d + [0] * (T - len(d)) for d in drafted], dtype=torch.int32, device=device)
            states = [int32([batch.state_of(i) for i in ids])]
            for i in range(T):
                states.append(ops.advance_state(fsa, states[i], x[:, i].contiguous()))
            ops.truncate_(logits.flatten(0, 1), fsa, torch.stack(states, 1).flatten(), temperature=temperature, **CUTS)
            n, token = batch.verify(ids, logits, x, uniforms(T + 1), draft_lens=int32([len(d) for d in drafted]),
                                    temperature=temperature)
            n = n.tolist()
        for i, t in zip(ids, token.tolist()):
            if going[i]:
                new = drafted[i][:n[i]] + [t]
                written[i] += new[:new.index(eos) + 1] if eos in new else new
    for cache in caches:
        cache.check_errors()
    return written


def main() -> None:
    p = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    p.add_argument("--device", default="cuda" if torch.cuda.is_available() else "cpu")
    p.add_argument("--requests", type=int, default=4)
    p.add_argument("--drafts", type=int, default=3)
    p.add_argument("--tokens", type=int, default=40)
    a = p.parse_args()
    vocab = vocabulary()
    fsa = FsaTensors.build(PATTERN, vocab, dense=True).to(a.device)
    model = Reader(vocab.size, a.device)
    positions = prompt_positions(30, 6, 9, 16)
    instruction = [(7 * i) % 256 for i in range(positions.shape[1])]
    requests = [list(b"ab12,"[:1 + i % 5]) for i in range(a.requests)]
    for drafts in (0, a.drafts):
        out = generate(model, fsa, instruction, positions, requests, tokens=a.tokens, drafts=drafts, device=a.device)
        print(f"{drafts} drafts a step:")
        for w in out:
            print("   ", b"".join(vocab.token_bytes[t] for t in w if t >= 0))


if __name__ == "__main__":
    main()
