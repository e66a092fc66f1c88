"""Attention of a batch that shares a prefix (PagedKV4.attend_shared) against
the plain 64-bit form over the whole requests, and against attend.

The tolerance is that of tests/_spec_ref.py's attention and, for joining the
prefix's pieces (at most 128 of them) with the rest, 2 * 130 roundings of
2^-24 of the weighted values' size: below 2e-5 of the largest value."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from bpdecode_amd.kv import PagedKV4, block_bytes
from tests import _spec_ref as R
from tests.test_kv4 import BF16, DEVICES, FP16, filled_cache, stored

CASES = [  # tokens, kv heads, heads, dim, page, dtype, shared, lengths of the whole requests
    (1, 1, 1, 64, 16, BF16, 64, [64, 65, 66, 100, 3, 0]),
    (1, 2, 8, 128, 16, BF16, 1_000, [1_001, 1_064, 1_130, 1_000, 999]),
    (4, 2, 4, 64, 32, FP16, 352, [360, 356, 355, 354, 353, 352, 500, 2, 0]),
    (5, 1, 8, 128, 64, BF16, 130, [135, 200, 129, 133]),
    (3, 3, 3, 96, 16, FP16, 200, [203, 260, 201]),
    (2, 1, 7, 192, 128, BF16, 300, [302, 420, 257]),
    (3, 2, 4, 256, 16, FP16, 80, [85, 83, 300]),
    (1, 4, 20, 256, 256, BF16, 512, [600, 513]),
    (20, 1, 5, 128, 16, BF16, 96, [130, 117, 116, 115, 97]),
    (1, 1, 16, 128, 32, BF16, 2_080, [2_081 + 13 * b for b in range(21)]),
    (7, 2, 6, 64, 16, FP16, 1_500, [1_507 + b for b in range(12)]),
    (1, 1, 4, 128, 16, BF16, 48, [50, 120]),  # less than a tile shared
    (1, 1, 4, 128, 64, FP16, 63, [70, 120]),  # less than a page
    (2, 1, 4, 64, 16, BF16, 0, [2, 77]),
]


def shared_cache(g, B, P, KV, D, dt, shared, blocks, device, seed):
    """A cache, the shared pages' table, whole tables for the plain form, and
    the same with nothing where the shared pages are."""
    cache, table = filled_cache(g, B, P, KV, D, dt, blocks, device, seed)
    n = shared // P
    table[:, :n] = table[0, :n].clone()
    hidden = table.clone()
    hidden[:, :n] = -1
    return cache, table[0, :-(-shared // P)].clone(), table, hidden


def close(got, want, tol, v):
    got = got.cpu().double().numpy()
    off = np.abs(got - want)
    assert np.isfinite(got).all()
    tol = np.where(tol > 0, tol + 2e-5 * np.abs(v).max(), 0.0)
    assert (off <= tol).all(), float((off - tol).max())


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("case", range(len(CASES)))
def test_attention_behind_a_prefix_against_the_plain_form(case, device):
    T, KV, H, D, P, dt, shared, lengths = CASES[case]
    print(f"shared case {case} on {device}", flush=True)
    B = len(lengths)
    g = torch.Generator().manual_seed(300 + case)
    blocks = max(max(lengths), shared) // P + 2
    cache, prefix, table, hidden = shared_cache(g, B, P, KV, D, dt, shared, blocks, device, case)
    k, v = stored(cache, table, max(lengths))
    for b, n in enumerate(lengths):
        hidden[b, (n + P - 1) // P:] = -1
    q = (1.3 * torch.randn(B, T, H, D, generator=g)).to(dt)
    ql = torch.tensor([(T + b) % (T + 1) if b else T + 3 for b in range(B)], dtype=torch.int32) if case % 3 == 2 else None
    to = lambda t: None if t is None else t.to(device)  # noqa: E731
    scale = 0.2 if case % 4 == 1 else -0.15 if case % 4 == 3 else None
    lens = torch.tensor(lengths, dtype=torch.int32)
    count = torch.tensor([shared], dtype=torch.int32, device=device) if case % 2 else shared
    out = cache.attend_shared(to(q), to(prefix), count, to(hidden), to(lens), query_lens=to(ql), scale=scale)
    want, tol = R.attend(q.double().numpy(), k, v, lengths, dt, query_lens=None if ql is None else ql.tolist(), scale=scale)
    close(out, want, tol, v)
    cache.check_errors()
    for b in range(B):
        for i in range(T):
            if not tol[b, i].any():
                assert not out[b, i].any()


@pytest.mark.parametrize("device", DEVICES)
def test_one_request_is_attend(device):
    """A batch of one, and prefixes of every length up to the request's."""
    KV, H, D, P, n = 2, 6, 64, 16, 200
    g = torch.Generator().manual_seed(31)
    cache, table = filled_cache(g, 1, P, KV, D, BF16, 13, device, 1)
    q = torch.randn(1, 2, H, D, generator=g).to(BF16).to(device)
    table, lens = table.to(device), torch.tensor([n], dtype=torch.int32, device=device)
    want = cache.attend(q, table, lens).double().cpu()
    k, v = stored(cache, table.cpu(), n)
    plain, tol = R.attend(q.double().cpu().numpy(), k, v, [n], BF16)
    for shared in (0, 15, 16, 63, 64, 80, 127, 128, 192, 198, 199, 200, 208):
        out = cache.attend_shared(q, table[0], shared, table, lens)
        close(out, plain, tol, v)
        if shared < 64:
            assert torch.equal(out.double().cpu(), want)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dt", [BF16, FP16])
def test_a_token_that_outweighs_all_others(dt, device):
    """In the prefix, or in a request's own part; the other's weights vanish."""
    B, KV, D, P, shared, n = 3, 1, 128, 16, 320, 400
    g = torch.Generator().manual_seed(32)
    cache, prefix, table, hidden = shared_cache(g, B, P, KV, D, dt, shared, 26, device, 2)
    pages = cache.pages.cpu()
    pages[prefix[7], :, P * D + 5 * 4:P * D + 6 * 4] = 127 + 4
    pages[table[1, 22], :, P * D + 2 * 4:P * D + 3 * 4] = 127 + 6
    cache.pages.copy_(pages)
    q = torch.randn(B, 1, 8, D, generator=g).to(dt)
    k, v = stored(cache, table, n)
    lens = torch.full((B,), n, dtype=torch.int32, device=device)
    out = cache.attend_shared(q.to(device), prefix.to(device), shared, hidden.to(device), lens)
    close(out, *R.attend(q.double().numpy(), k, v, [n] * B, dt), v)


@pytest.mark.parametrize("device", DEVICES)
def test_pages_outside_the_pool_and_nan(device):
    """A prefix page that is not there is left out for all and noted, a shared
    count past the table is cut, a NaN in the prefix shows in its heads for
    those who see it."""
    B, KV, H, D, P, shared = 4, 2, 4, 64, 16, 256
    g = torch.Generator().manual_seed(33)
    cache, prefix, table, hidden = shared_cache(g, B, P, KV, D, BF16, shared, 20, device, 3)
    lengths = [300, 257, 290, 100]
    to = lambda t: t.to(device)  # noqa: E731
    lens = to(torch.tensor(lengths, dtype=torch.int32))
    q = torch.randn(B, 1, H, D, generator=g).to(BF16)
    k, v = stored(cache, table, 300)
    for bad, at in ((-1, 3), (cache.num_pages, 9), (2 ** 31 - 1, 0)):
        broken = prefix.clone()
        broken[at] = bad
        out = cache.attend_shared(to(q), to(broken), shared, to(hidden), lens)
        with pytest.raises(IndexError):
            cache.check_errors()
        kk = k.copy()
        kk[:, at * P:(at + 1) * P] = np.nan
        close(out, *R.attend(q.double().numpy(), kk, v, lengths, BF16), v)
    count = to(torch.tensor([shared + P], dtype=torch.int32))
    out = cache.attend_shared(to(q), to(prefix), count, to(hidden), lens)
    with pytest.raises(IndexError):
        cache.check_errors()
    close(out, *R.attend(q.double().numpy(), k, v, lengths, BF16), v)
    out = cache.attend_shared(to(q), to(prefix), to(torch.tensor([-5], dtype=torch.int32)), to(table), lens)
    close(out, *R.attend(q.double().numpy(), k, v, lengths, BF16), v)
    cache.check_errors()
    cache.pages[int(prefix[10]), 1, P * D + 3 * 2] = 255  # key group of token 163, head 1
    cache.pages[int(prefix[5]), 0, P * (D + 2) + 2 * 2 + 1] = 255  # value group of token 82, head 0, channels 32 and up
    out = cache.attend_shared(to(q), to(prefix), shared, to(hidden), lens)
    nan = out.isnan()
    assert nan[:3, :, 2:].all() and not nan[3, :, 2:].any()
    assert nan[:, :, :2, 32:].all() and not nan[:, :, :2, :32].any()


@pytest.mark.parametrize("device", DEVICES)
def test_strided_blocks_and_tables(device):
    B, T, KV, H, D, P, shared = 3, 2, 2, 4, 128, 16, 128
    g = torch.Generator().manual_seed(34)
    cache, prefix, table, hidden = shared_cache(g, B, P, KV, D, FP16, shared, 12, device, 4)
    lens = torch.tensor([[170, 0], [131, 0], [150, 0]], dtype=torch.int32, device=device)[:, 0]
    wide = torch.randn(T, B, H * D + 3, generator=g).to(FP16).to(device).transpose(0, 1)
    q = wide[..., 1:1 + H * D].unflatten(-1, (H, D))
    two = torch.stack((hidden, hidden), 2).flatten(1).to(device)[:, ::2]
    line = torch.stack((prefix, prefix), 1).flatten().to(device)[::2]
    a = cache.attend_shared(q, line, shared, two, lens)
    b = cache.attend_shared(q.contiguous(), prefix.to(device), shared, hidden.to(device), lens.contiguous())
    assert torch.equal(a, b) and bool(a.abs().sum() > 0)


@pytest.mark.gpu
def test_many_requests_agree_with_attend(dev):
    """More columns than a block takes, more tiles than chunks; each request
    equals attend's to the roundings of both."""
    for T, KV, H, D, P, dt, shared, B in ((1, 2, 8, 128, 64, BF16, 5_000, 90), (3, 4, 4, 64, 16, FP16, 3_333, 61),
                                          (1, 1, 8, 256, 32, BF16, 1_300, 40), (2, 1, 2, 96, 16, FP16, 900, 33)):
        print(f"shared {T} {KV} {H} {D} {shared} {B}", flush=True)
        g = torch.Generator().manual_seed(B)
        lengths = [shared + T + (37 * b) % 300 for b in range(B)]
        blocks = max(lengths) // P + 1
        cache, prefix, table, hidden = shared_cache(g, B, P, KV, D, dt, shared, blocks, dev, B)
        q = torch.randn(B, T, H, D, generator=g).to(dt).to(dev)
        lens = torch.tensor(lengths, dtype=torch.int32, device=dev)
        out = cache.attend_shared(q, prefix.to(dev), shared, hidden.to(dev), lens)
        want = cache.attend(q, table.to(dev), lens)
        rows = [0, 1, B // 2, B - 1]
        k, v = stored(cache, table[rows], max(lengths))
        plain, tol = R.attend(q[rows].double().cpu().numpy(), k, v, [lengths[r] for r in rows], dt)
        close(out[rows], plain, tol, v)
        most = float(np.abs(v).max())
        eps = torch.finfo(dt).eps / 2
        assert float((out.double() - want.double()).abs().max()) <= 4 * eps * most
        again = cache.attend_shared(q, prefix.to(dev), shared, hidden.to(dev), lens)
        assert torch.equal(out, again)
        cache.check_errors()


@pytest.mark.gpu
def test_replays_of_a_captured_call(dev):
    B, T, KV, H, D, P = 6, 1, 2, 8, 128, 16
    g = torch.Generator().manual_seed(35)
    cache, prefix, table, hidden = shared_cache(g, B, P, KV, D, BF16, 512, 60, dev, 5)
    prefix = table[0, :40].clone().to(dev)
    q = torch.zeros(B, T, H, D, dtype=BF16, device=dev)
    shared, lens = torch.zeros(1, dtype=torch.int32, device=dev), torch.ones(B, dtype=torch.int32, device=dev)
    whole = table.to(dev)
    cache.attend_shared(q, prefix, shared, whole, lens)
    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
    outs = []
    for graph in graphs:
        with torch.cuda.graph(graph):
            outs.append(cache.attend_shared(q, prefix, shared, whole, lens))
    for step, n in enumerate((0, 512, 130, 64, 500)):
        q.copy_(torch.randn(q.shape, generator=g))
        shared.fill_(n)
        lens.copy_(torch.randint(n, 900, (B,), generator=g))
        want = cache.attend_shared(q, prefix, shared, whole, lens)
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for out in outs:
            assert torch.equal(out, want)
    cache.check_errors()


@pytest.mark.parametrize("device", DEVICES)
def test_refusals_and_empty_calls(device):
    cache = PagedKV4.empty(4, 16, 2, 64, BF16, device)
    q = torch.zeros(2, 1, 4, 64, dtype=BF16, device=device)
    table, lens = torch.zeros(2, 3, dtype=torch.int32, device=device), torch.full((2,), 20, dtype=torch.int32, device=device)
    prefix = torch.zeros(2, dtype=torch.int32, device=device)
    good = (q, prefix, 16, table, lens)
    cases = [
        ((q[..., :32], *good[1:]), {}, "q must be"), ((q.half(), *good[1:]), {}, "q must be"), ((q[:, :, :3], *good[1:]), {}, "multiple"),
        ((q, prefix[None], 16, table, lens), {}, "prefix_table"), ((q, prefix.long(), 16, table, lens), {}, "prefix_table"),
        ((q, prefix.to("meta"), 16, table, lens), {}, "prefix_table"), ((q, prefix, 33, table, lens), {}, "33 shared tokens"),
        ((q, prefix, -1, table, lens), {}, "-1 shared tokens"), ((q, prefix, lens, table, lens), {}, "shared must be"),
        ((q, prefix, torch.ones(1, device=device), table, lens), {}, "shared must be"), ((q, prefix, 16, table[:1], lens), {}, "block_table"),
        ((q, prefix, 16, table.long(), lens), {}, "block_table"), ((q, prefix, 16, table, lens.long()), {}, "lengths"),
        (good, dict(query_lens=lens[:1]), "query_lens"), (good, dict(scale=float("inf")), "scale"),
    ]
    for args, kw, match in cases:
        with pytest.raises(RuntimeError, match=match):
            cache.attend_shared(*args, **kw)
    assert cache.attend_shared(q[:0], prefix, 16, table[:0], lens[:0]).shape == (0, 1, 4, 64)
    assert cache.attend_shared(q[:, :0], prefix, 16, table, lens).shape == (2, 0, 4, 64)
    none = PagedKV4(torch.zeros(0, 2, block_bytes(16, 64), dtype=torch.uint8, device=device), 16, 64, BF16,
                    torch.zeros(1, dtype=torch.int32, device=device))
    assert not none.attend_shared(*good).any()
    with pytest.raises(IndexError):
        none.check_errors()


@pytest.mark.gpu
@pytest.mark.parametrize("T,KV,H,D,P,dt,shared", [
    (77, 4, 4, 64, 16, FP16, 8_400), (25, 8, 16, 96, 32, BF16, 8_260), (18, 8, 32, 128, 64, BF16, 4_224), (18, 8, 32, 128, 16, FP16, 4_100),
    (20, 8, 16, 256, 32, BF16, 8_200), (25, 8, 8, 192, 64, FP16, 16_420)])
def test_wide_blocks_of_long_prefixes(T, KV, H, D, P, dt, shared, dev):
    """Enough work for blocks of 128 and 256 columns: odd numbers of tiles, of
    columns and of tiles in a chunk, and then a page that is not there."""
    print(f"shared {T} {KV} {H} {D} {shared}", flush=True)
    B = 4
    g = torch.Generator().manual_seed(D + T)
    lengths = [shared + T + 31 * b for b in range(B - 1)] + [shared + T - 1]
    blocks = max(lengths) // P + 1
    cache, prefix, table, hidden = shared_cache(g, B, P, KV, D, dt, shared, blocks, dev, T)
    q = torch.randn(B, T, H, D, generator=g).to(dt).to(dev)
    lens = torch.tensor(lengths, dtype=torch.int32, device=dev)
    out = cache.attend_shared(q, prefix.to(dev), shared, hidden.to(dev), lens)
    k, v = stored(cache, table, max(lengths))
    plain, tol = R.attend(q.double().cpu().numpy(), k, v, lengths, dt)
    close(out, plain, tol, v)
    cache.check_errors()
    most, eps = float(np.abs(v).max()), torch.finfo(dt).eps / 2
    gone = 70 * 64 // P if shared > 5_000 else 3
    prefix[gone] = -1
    table[:, gone] = -1
    out = cache.attend_shared(q, prefix.to(dev), shared, hidden.to(dev), lens)
    with pytest.raises(IndexError):
        cache.check_errors()
    want = cache.attend(q, table.to(dev), lens)
    with pytest.raises(IndexError):
        cache.check_errors()
    assert float((out.double() - want.double()).abs().max()) <= 4 * eps * most
