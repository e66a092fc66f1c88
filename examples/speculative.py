"""Speculative decoding under a grammar, over a 4-bit paged cache.

    python examples/speculative.py [--device cuda] [--drafts 4] [--temperature 0.8]

A small model of random weights writes documents of a regular expression.  Each
step looks the next tokens up in what a request has written (a certain draft),
runs one block per request through the model -- its keys and values are rotated
and appended to the cache, its queries attend to it -- and lets the constraint
batch decide how many drafted tokens stand and which token follows them.  What
a refused draft left in the cache is overwritten by the next block.
"""

from __future__ import annotations

import argparse
import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parent.parent))

from bpdecode_amd.batch import ConstraintBatch  # noqa: E402
from bpdecode_amd.kv import PagedKV4  # noqa: E402
from bpdecode_amd.ops import FsaTensors  # noqa: E402
from bpdecode_amd.tokenizer import Vocabulary  # noqa: E402

PATTERN = r"(ab|ba|[0-9]{2},)+!"


def vocabulary() -> Vocabulary:
    """All bytes, the digits in pairs, a few pieces of the pattern, EOS."""
    pairs = [f"{i:02d}".encode() for i in range(100)]
    return Vocabulary((*(bytes([i]) for i in range(256)), *pairs, b"ab", b"ba", b"abab", b",ab", b"</s>"), eos_id=360)


class Model:
    """Layers of attention and a gated product over random weights, in 64 bits
    but for what goes through the cache."""

    def __init__(self, vocab: int, device, layers=2, heads=4, kv_heads=2, dim=64, width=96, positions=512, seed=0) -> None:
        g = torch.Generator().manual_seed(seed)

        def weight(*shape):
            return (torch.randn(*shape, generator=g, dtype=torch.float64) * shape[0] ** -0.5).to(device)

        self.heads, self.kv_heads, self.dim = heads, kv_heads, dim
        self.embed = torch.randn(vocab, width, generator=g, dtype=torch.float64).to(device)
        self.layers = [{"qkv": weight(width, (heads + 2 * kv_heads) * dim), "out": weight(heads * dim, width),
                        "up": weight(width, 4 * width), "down": weight(2 * width, width)} for _ in range(layers)]
        self.head = weight(width, vocab) * 2.0
        angle = torch.arange(positions, dtype=torch.float64)[:, None] * 1e4 ** (-torch.arange(0, dim, 2) / dim)
        self.cos, self.sin = torch.cos(angle).float().to(device), torch.sin(angle).float().to(device)

    def __call__(self, tokens, caches, table, starts, counts):
        """Logits [requests, tokens, vocab] of a block of tokens that begins at
        ``starts`` and of which ``counts`` are there."""
        x = self.embed[tokens]
        H, KV, D = self.heads, self.kv_heads, self.dim
        for w, cache in zip(self.layers, caches):
            q, k, v = ((norm(x) @ w["qkv"]).unflatten(-1, (-1, D)).to(cache.dtype)).split((H, KV, KV), 2)
            q = cache.append(k, v, table, starts, counts=counts, cos=self.cos, sin=self.sin, q=q)
            y = cache.attend(q, table, starts + counts, query_lens=counts)
            x = x + y.flatten(2).double() @ w["out"]
            a, b = (norm(x) @ w["up"]).chunk(2, -1)
            x = x + (torch.nn.functional.silu(a) * b) @ w["down"]
        return (norm(x) @ self.head).float()


def norm(x: torch.Tensor) -> torch.Tensor:
    return x / (x.pow(2).mean(-1, keepdim=True) + 1e-6).sqrt()


def look_up(history: list[int], most: int) -> list[int]:
    """The tokens that followed the last earlier place of the newest token."""
    for i in range(len(history) - 2, -1, -1):
        if history[i] == history[-1]:
            return history[i + 1:i + 1 + most]
    return []


def generate(model: Model, fsa: FsaTensors, prompts: list[list[int]], *, tokens: int, drafts: int, temperature=0.0,
             device="cpu", page_size=16, seed=0) -> tuple[list[list[int]], int]:
    """Up to about ``tokens`` tokens for each prompt, and the steps it took."""
    B, eos = len(prompts), fsa.eos_id
    longest = max(map(len, prompts)) + tokens + drafts + 1
    blocks = -(-longest // page_size)
    caches = [PagedKV4.empty(B * blocks, page_size, model.kv_heads, model.dim, torch.bfloat16, device) for _ in model.layers]
    g = torch.Generator().manual_seed(seed)
    table = torch.randperm(B * blocks, generator=g).view(B, blocks).to(torch.int32).to(device)
    batch = ConstraintBatch(fsa, capacity=B, device=device)
    ids = list(range(B))
    for i in ids:
        batch.add(i)

    def int32(values):
        return torch.tensor(values, dtype=torch.int32, device=device)

    def block(rows: list[list[int]], starts: list[int]):
        """Logits of blocks of different lengths, padded."""
        T = max(map(len, rows))
        padded = torch.tensor([r + [0] * (T - len(r)) for r in rows], device=device)
        return model(padded, caches, table, int32(starts), int32([len(r) for r in rows]))

    def decide(logits, drafted: list[list[int]]):
        T = logits.shape[1] - 1
        x = torch.tensor([d + [0] * (T - len(d)) for d in drafted], dtype=torch.int32, device=device).view(B, T)
        u = torch.rand(B, T + 1, generator=g).to(device)
        n, token = batch.verify(ids, logits, x, u, draft_lens=int32([len(d) for d in drafted]), temperature=temperature)
        return n.tolist(), token.tolist()

    # the prompts, and the first token of each
    last = torch.tensor([len(p) - 1 for p in prompts], device=device)
    logits = block(prompts, [0] * B)[torch.arange(B, device=device), last][:, None]
    _, first = decide(logits, [[] for _ in ids])
    written = [[t] for t in first]
    steps = 1
    while any(w[-1] not in (eos, -1) and len(w) < tokens for w in written):
        going = [w[-1] not in (eos, -1) and len(w) < tokens for w in written]
        drafted = [look_up(prompts[i] + written[i], drafts) if going[i] else [] for i in ids]
        rows = [[max(written[i][-1], 0)] + drafted[i] for i in ids]
        starts = [len(prompts[i]) + len(written[i]) - 1 for i in ids]
        n, token = decide(block(rows, starts), drafted)
        steps += 1
        for i in ids:
            if going[i]:
                new = drafted[i][:n[i]] + [token[i]]
                written[i] += new[:new.index(eos) + 1] if eos in new else new
    for cache in caches:
        cache.check_errors()
    return written, steps


def main() -> None:
    p = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    p.add_argument("--device", default="cuda" if torch.cuda.is_available() else "cpu")
    p.add_argument("--drafts", type=int, default=4)
    p.add_argument("--temperature", type=float, default=0.0)
    p.add_argument("--tokens", type=int, default=60)
    a = p.parse_args()
    vocab = vocabulary()
    fsa = FsaTensors.build(PATTERN, vocab, dense=True).to(a.device)
    model = Model(vocab.size, a.device)
    prompts = [list(b"ab12,"), list(b"12,34,56,78,"), [97]]
    for drafts in (0, a.drafts):
        out, steps = generate(model, fsa, prompts, tokens=a.tokens, drafts=drafts, temperature=a.temperature, device=a.device)
        print(f"{drafts} drafts a step: {sum(map(len, out))} tokens in {steps} steps")
        for w in out:
            print("   ", b"".join(vocab.token_bytes[t] for t in w if t >= 0))


if __name__ == "__main__":
    main()
