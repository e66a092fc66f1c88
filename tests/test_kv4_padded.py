"""Attention over the 4-bit cache with fewer queries than the block has rows:
rows past ``query_lens`` are zeros whatever their request holds, also where
whole tiles of 64 tokens are seen by every real query.  Tolerances as in
tests/_spec_ref.py."""

from __future__ import annotations

import pytest
import torch

from tests import _spec_ref as R
from tests.test_kv4 import BF16, FP16, close, filled_cache, stored

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]

PADDED = [  # tokens, kv heads, heads, dim, page, dtype, lengths
    (4, 1, 1, 64, 16, BF16, [64, 65, 200, 128, 64]),               # short units, one column tile
    (4, 2, 12, 128, 16, FP16, [64, 65, 200, 300, 127]),            # two column tiles
    (4, 2, 16, 96, 32, BF16, [64, 1_000, 200]),
    (20, 1, 7, 128, 32, BF16, [64, 500, 200]),                     # 140 columns: groups of padded columns alone
    (4, 24, 24, 64, 16, BF16, [64, 1_100, 200]),                   # 72 units of up to 18 tiles
    (4, 24, 144, 128, 16, FP16, [65, 1_100, 200]),
    (4, 1, 2, 192, 16, BF16, [5_000, 64, 200, 1_100, 5_000, 65]),  # cut into runs and joined
    (4, 1, 8, 128, 64, FP16, [5_000, 64, 200, 1_100, 5_000]),
    (9, 2, 8, 256, 16, BF16, [200, 4_700]),
]


def query_lens(T: int, rows: int) -> list[int]:
    """One query, two, ... for requests in turn, none for the last of many."""
    return [b % (T - 1) + 1 if b < 4 else 0 for b in range(rows)]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("case", range(len(PADDED)))
def test_rows_past_a_request_s_queries_are_zeros(case, device):
    T, KV, H, D, P, dt, lengths = PADDED[case]
    print(f"padded case {case} on {device}", flush=True)
    B = len(lengths)
    n = query_lens(T, B)
    g = torch.Generator().manual_seed(300 + case)
    cache, table = filled_cache(g, B, P, KV, D, dt, (max(lengths) + P - 1) // P, device, case)
    k, v = stored(cache, table, max(lengths))
    q = (1.2 * torch.randn(B, T, H, D, generator=g)).to(dt)
    call = lambda: cache.attend(q.to(device), table.to(device),  # noqa: E731
                                torch.tensor(lengths, dtype=torch.int32, device=device),
                                query_lens=torch.tensor(n, dtype=torch.int32, device=device)).cpu()
    out = call()
    for b in range(B):
        assert not out[b, n[b]:].any(), (b, float(out[b, n[b]:].abs().max()))
    want, tol = R.attend(q.double().numpy(), k, v, lengths, dt, query_lens=n)
    close(out, want, tol)
    # a bad value group in a token that every real query sees
    G = D // 32
    for b in range(B):
        cache.pages[int(table[b, 0]), 0, P * D + P * G + 3 * G] = 255
    bad = call()
    nan = torch.zeros(bad.shape, dtype=torch.bool)
    for b in range(B):
        nan[b, :n[b], :H // KV, :32] = True
    assert torch.equal(bad.isnan(), nan)
    assert torch.equal(bad[~nan], out[~nan])
    cache.check_errors()
