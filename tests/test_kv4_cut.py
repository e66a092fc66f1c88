"""How attention over the 4-bit cache cuts its work: long and short requests
in one batch, more requests than a wave has lanes, more query columns than a
block holds, tokens that only some queries of a block see, scales of either
sign.  Tolerances as in tests/_spec_ref.py."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from bpdecode_amd.kv import PagedKV4
from tests import _spec_ref as R
from tests.test_kv4 import BF16, FP16, close, filled_cache, stored

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


CUTS = [  # tokens, kv heads, heads, dim, page, dtype, lengths
    (1, 1, 2, 64, 16, BF16, [5_000, 1, 0, 17, 4_999, 64]),      # long and short ones, equal runs
    (2, 2, 4, 128, 64, FP16, [4_500, 300, 2, 4_400]),
    (1, 2, 2, 96, 32, BF16, [4_200, 63, 64, 65]),
    (3, 1, 24, 128, 16, BF16, [4_300, 70]),                      # 72 columns: groups of two tiles
    (9, 1, 8, 64, 32, FP16, [5_100, 9, 8]),
    (20, 1, 7, 128, 32, BF16, [500, 21]),                        # 140 columns
    (5, 1, 8, 256, 16, BF16, [4_200, 33]),                       # 40 columns of 256 channels
    (7, 2, 8, 192, 64, FP16, [4_120, 200]),
    (1, 1, 1, 256, 256, BF16, [4_600, 255, 257]),
    (1, 1, 5, 64, 16, BF16, [(37 * i) % 90 for i in range(70)]),  # more requests than lanes, one block each
    (1, 1, 1, 64, 128, FP16, [4_400] + [(11 * i) % 300 for i in range(130)]),
]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("case", range(len(CUTS)))
def test_cuts_against_plain_form(case, device):
    T, KV, H, D, P, dt, lengths = CUTS[case]
    print(f"cut case {case} on {device}", flush=True)
    B = len(lengths)
    g = torch.Generator().manual_seed(150 + case)
    blocks = (max(lengths) + P - 1) // P
    cache, table = filled_cache(g, B, P, KV, D, dt, blocks, device, case)
    k, v = stored(cache, table, max(lengths))
    for b, n in enumerate(lengths):
        table[b, (n + P - 1) // P:] = -1
    q = (1.2 * torch.randn(B, T, H, D, generator=g)).to(dt)
    out = cache.attend(q.to(device), table.to(device), torch.tensor(lengths, dtype=torch.int32, device=device))
    close(out, *R.attend(q.double().numpy(), k, v, lengths, dt))
    cache.check_errors()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("T", [1, 17])
@pytest.mark.parametrize("D", [64, 96, 128, 192, 256])
def test_units_no_more_than_compute_units(D, T, device):
    """72 units of up to 18 tiles: one wide block each, two column tiles with 17
    tokens; a request without tokens, one that ends inside its first tile, one
    in its last; a bad value group in the third's last token."""
    print(f"units of {D} channels, {T} tokens on {device}", flush=True)
    KV, P, lengths = 24, 16, [0, T + 3, 1_097]
    g = torch.Generator().manual_seed(90 + D + T)
    cache, table = filled_cache(g, 3, P, KV, D, BF16, 69, device, 12)
    k, v = stored(cache, table, max(lengths))
    for b, n in enumerate(lengths):
        table[b, (n + P - 1) // P:] = -1
    q = (1.2 * torch.randn(3, T, KV, D, generator=g)).to(BF16)
    call = lambda: cache.attend(q.to(device), table.to(device),  # noqa: E731
                                torch.tensor(lengths, dtype=torch.int32, device=device))
    good = call()
    close(good, *R.attend(q.double().numpy(), k, v, lengths, BF16))
    cache.check_errors()
    at = P * D + P * (D // 32) + (lengths[2] - 1) % P * (D // 32)  # the value scales of that token
    cache.pages[int(table[2, 68]), 5, at] = 255
    bad = call().cpu()
    nan = torch.zeros(bad.shape, dtype=torch.bool)
    nan[2, T - 1, 5, :32] = True
    assert torch.equal(torch.isnan(bad), nan)
    assert torch.equal(bad[~nan], good.cpu()[~nan])


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("D", [64, 96, 128, 192, 256])
def test_a_bad_value_shows_only_where_its_token_is_seen(D, device):
    """A value group of infinities in a token that the last query alone sees:
    NaN in that query's channels of the group and nowhere else."""
    g = torch.Generator().manual_seed(80)
    P, KV, T, n = 16, 2, 3, 75
    cache, table = filled_cache(g, 2, P, KV, D, BF16, 5, device, 6)
    pages = cache.pages.cpu()
    G = D // 32
    for at, group in ((n - 1, G - 1), (n - 2, 0)):
        pages[table[0, at // P], 1, P * (D + G) + at % P * G + group] = 255
    cache.pages.copy_(pages)
    q = torch.randn(2, T, 4, D, generator=g).to(BF16)
    lengths = torch.tensor([n, n], dtype=torch.int32, device=device)
    out = cache.attend(q.to(device), table.to(device), lengths).cpu().isnan().view(2, T, KV, 2, G, 32)
    want = torch.zeros_like(out)
    want[0, 2, 1, :, G - 1] = True  # the last query sees both tokens
    want[0, 1:, 1, :, 0] = True
    assert torch.equal(out, want)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("scale", [-0.3, 0.0, 1e-6, 4.0])
def test_scales_of_either_sign(scale, device):
    g = torch.Generator().manual_seed(81)
    lengths = [40, 130]
    cache, table = filled_cache(g, 2, 16, 2, 64, FP16, 9, device, 7)
    k, v = stored(cache, table, max(lengths))
    q = torch.randn(2, 2, 6, 64, generator=g).to(FP16)
    out = cache.attend(q.to(device), table.to(device), torch.tensor(lengths, dtype=torch.int32, device=device), scale=scale)
    close(out, *R.attend(q.double().numpy(), k, v, lengths, FP16, scale=scale))


@pytest.mark.parametrize("device", DEVICES)
def test_pages_shared_between_requests_and_no_pages_at_all(device):
    """Two requests over one prefix (the same pages in both tables); a pool of
    no pages attends to nothing and says so."""
    g = torch.Generator().manual_seed(82)
    cache, table = filled_cache(g, 1, 32, 2, 128, BF16, 6, device, 8)
    both = table.expand(2, -1)
    q = torch.randn(1, 2, 8, 128, generator=g).to(BF16)
    lengths = torch.tensor([150, 99], dtype=torch.int32, device=device)
    out = cache.attend(q.expand(2, 2, 8, 128).to(device), both.to(device), lengths)
    for b in range(2):
        assert torch.equal(out[b:b + 1], cache.attend(q.to(device), table.to(device), lengths[b:b + 1]))
    none = PagedKV4.empty(0, 32, 2, 128, BF16, device)
    assert not none.attend(q.to(device), table.to(device), lengths[:1]).any()
    with pytest.raises(IndexError):
        none.check_errors()


@pytest.mark.parametrize("device", DEVICES)
def test_infinite_and_nan_queries_stay_in_their_rows(device):
    g = torch.Generator().manual_seed(83)
    cache, table = filled_cache(g, 2, 16, 2, 64, BF16, 3, device, 9)
    q = torch.randn(2, 3, 4, 64, generator=g).to(BF16)
    q[0, 1, 2, 5], q[1, 0, 0, 63] = float("nan"), float("inf")
    out = cache.attend(q.to(device), table.to(device), torch.tensor([40, 33], dtype=torch.int32, device=device)).cpu()
    bad = out.isnan().all(-1)
    want = torch.zeros_like(bad)
    want[0, 1, 2] = True
    assert bool(bad[0, 1, 2]) and not out[~(want | (torch.arange(4) == 0) & (torch.arange(3)[:, None] == 0)
                                           & torch.tensor([False, True])[:, None, None])].isnan().any()


@pytest.mark.gpu
def test_the_same_answer_every_time(dev):
    """No sum depends on the order in which blocks run."""
    g = torch.Generator().manual_seed(84)
    cache, table = filled_cache(g, 3, 64, 4, 128, BF16, 150, dev, 10)
    q = torch.randn(3, 2, 16, 128, generator=g).to(BF16).to(dev)
    lengths = torch.tensor([9_000, 20, 6_001], dtype=torch.int32, device=dev)
    table = table.to(dev)
    first = cache.attend(q, table, lengths)
    for _ in range(5):
        assert torch.equal(first, cache.attend(q, table, lengths))
    assert np.isfinite(first.float().cpu().numpy()).all()
