"""Attention weights over their range: tokens that leading ones outweigh by 10
to 17.5 nats and whose values are all that comes out, as behind the first
tokens of real contexts, whose values are small.

Per element the tolerance counts, with r the weights relative to the largest,
h half a step of the type, l the sum of r: the weights rounded to the type,
max(h r, 2^-32) each (a weight of float16 is a multiple of 2^-24 where the
largest is 2^7 or more; bfloat16 has float's range); the output rounded once, h of
itself or 2^-25; scores in float32, (D + 4) 2^-24 of sum |q k|, twice (the
weight and the sum); and sums of n numbers in float32, n 2^-24."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from bpdecode_amd.kv import PagedKV4
from tests.test_kv4 import BF16, FP16, stored

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


def led_cache(g, B: int, n: int, KV: int, D: int, P: int, dt, device):
    """Every 64th token leads, with keys of 4 and values of 0; the others' keys
    are 2, a few 3 and 1.5, and their values positive."""
    lead = torch.arange(n) % 64 == 5
    k = torch.full((B, n, KV, D), 2.0)
    at = torch.randint(0, D, (B, n, KV, 4), generator=g)
    k.scatter_(3, at, torch.tensor([1.5, 3.0])[torch.randint(0, 2, at.shape, generator=g)])
    k[:, lead] = 4.0
    v = torch.tensor([16.0, 32.0, 48.0, 64.0, 96.0])[torch.randint(0, 5, (B, n, KV, D), generator=g)]
    v[:, lead] = 0.0
    blocks = (n + P - 1) // P
    cache = PagedKV4.empty(B * blocks, P, KV, D, dt, device)
    table = torch.randperm(B * blocks, generator=g).view(B, blocks).to(torch.int32)
    cache.append(k.to(dt).to(device), v.to(dt).to(device), table.to(device),
                 torch.zeros(B, dtype=torch.int32, device=device))
    return cache, table


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("gap", [10.0, 14.0, 16.5, 17.5])
@pytest.mark.parametrize("T, KV, H, D, P, n", [(1, 1, 2, 64, 16, 200), (1, 2, 4, 128, 16, 1_000), (3, 1, 8, 128, 64, 4_500)])
@pytest.mark.parametrize("dt", [FP16, BF16])
def test_tokens_far_below_the_leading_ones(dt, T, KV, H, D, P, n, gap, device):
    print(f"{dt} {n} tokens {gap} nats below on {device}", flush=True)
    g = torch.Generator().manual_seed(n)
    cache, table = led_cache(g, 2, n, KV, D, P, dt, device)
    k, v = stored(cache, table, n)
    q = torch.ones(2, T, H, D, dtype=dt)
    scale = gap / (2.0 * D)
    lengths = torch.tensor([n, n], dtype=torch.int32, device=device)
    out = cache.attend(q.to(device), table.to(device), lengths, scale=scale).cpu().double().numpy()
    h = torch.finfo(dt).eps / 2
    for b in range(2):
        for i in range(T):
            m = n - T + 1 + i
            for kv in range(KV):
                s = k[b, :m, kv].sum(1) * scale
                r = np.exp(s - s.max())
                low = np.maximum(h * r, 2.0 ** -32) if dt == FP16 else h * r
                want, size = r @ v[b, :m, kv] / r.sum(), r @ np.abs(v[b, :m, kv]) / r.sum()
                es = (D + 4) * 2.0 ** -24 * float(np.abs(k[b, :m, kv]).sum(1).max()) * scale
                tol = low @ np.abs(v[b, :m, kv]) / r.sum() + h * np.abs(want) + 2.0 ** -25 + (2 * es + m * 2.0 ** -24) * size
                off = np.abs(out[b, i, kv * (H // KV):(kv + 1) * (H // KV)] - want)
                assert (off <= tol).all(), float((off / want).max())
