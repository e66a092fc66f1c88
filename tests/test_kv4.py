"""The 4-bit paged cache (bpdecode_amd.kv.PagedKV4): appending with the
rotation, reading back, attention, against plain 64-bit forms.

What is appended and read back has to be equal: the rotation rounds every
product and sum to float32 by itself, a scale is a power of two, and every
level is representable.  Attention is held to a tolerance that counts
roundings (tests/_spec_ref.py)."""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from bpdecode_amd import _lib
from bpdecode_amd.kv import HEAD_DIMS, PagedKV4, block_bytes
from tests import _spec_ref as R

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
BF16, FP16 = torch.bfloat16, torch.float16


def np_(t: torch.Tensor) -> np.ndarray:
    return t.float().numpy()


def rotation(positions: int, rotary: int) -> tuple[torch.Tensor, torch.Tensor]:
    a = torch.arange(positions, dtype=torch.float64)[:, None] * 1e4 ** (-torch.arange(0, rotary, 2) / max(rotary, 1))
    return torch.cos(a).float(), torch.sin(a).float()


def values(g, *shape, dtype, large=0.05):
    x = torch.randn(*shape, generator=g)
    x = torch.where(torch.rand(shape[-1], generator=g) < large, 8 * x, x)
    return x.to(dtype)


APPEND = [  # rows, tokens, kv heads, heads, dim, rotary, interleaved, page, dtype, starts
    (1, 1, 1, 0, 64, 0, False, 16, BF16, [0]),
    (1, 1, 8, 32, 128, 128, False, 16, BF16, [31]),
    (3, 5, 2, 4, 64, 32, True, 32, FP16, [0, 13, 60]),
    (2, 40, 3, 3, 96, 96, False, 16, BF16, [7, 100]),
    (4, 3, 1, 7, 256, 256, True, 64, FP16, [0, 62, 63, 64]),
    (2, 17, 5, 5, 192, 50, False, 128, BF16, [120, 3]),
    (2, 9, 2, 2, 128, 6, True, 16, FP16, [8, 15]),
]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("case", range(len(APPEND)))
def test_append_and_read_equal_the_plain_form(case, device):
    B, T, KV, H, D, rot, inter, P, dt, starts = APPEND[case]
    print(f"append case {case} on {device}", flush=True)
    g = torch.Generator().manual_seed(case)
    blocks = (max(starts) + T + P - 1) // P
    cache = PagedKV4.empty(B * blocks + 2, P, KV, D, dt, device)
    noise = torch.randint(0, 256, cache.pages.shape, generator=g, dtype=torch.uint8)
    cache.pages.copy_(noise)
    table = R.block_tables(B, blocks, B * blocks + 2, case)
    k, v = values(g, B, T, KV, D, dtype=dt), values(g, B, T, KV, D, dtype=dt, large=0.0)
    q = values(g, B, T, H, D, dtype=dt) if H else None
    counts = torch.tensor([max(0, T - 2 * b) for b in range(B)], dtype=torch.int32) if case % 2 == 0 else None
    n = [T] * B if counts is None else counts.tolist()
    cos, sin = rotation(max(starts) + T, rot) if rot else (None, None)
    to = lambda t: None if t is None else t.to(device)  # noqa: E731
    st = torch.tensor(starts, dtype=torch.int32)
    out = cache.append(to(k), to(v), to(table), to(st), counts=to(counts), cos=to(cos), sin=to(sin), interleaved=inter,
                       q=to(q))
    cache.check_errors()
    kr, vr = cache.read(to(table), to(st), T)
    cache.check_errors()
    before = PagedKV4(noise.clone(), P, D, dt)
    k0, v0 = before.read(table, st, T)
    for b in range(B):
        turn = lambda x: x  # noqa: E731
        if rot:
            c, s = (t[starts[b]:starts[b] + n[b], None].numpy() for t in (cos, sin))
            turn = lambda x: R.rotated(x, c, s, inter)  # noqa: E731
        want_k, want_v = R.kept(turn(np_(k[b, :n[b]])), dt), R.kept(np_(v[b, :n[b]]), dt)
        assert np.array_equal(kr[b, :n[b]].cpu().double().numpy(), want_k)
        assert np.array_equal(vr[b, :n[b]].cpu().double().numpy(), want_v)
        # tokens past the count keep what was there
        for got, old in ((kr, k0), (vr, v0)):
            assert torch.equal(got[b, n[b]:].cpu().nan_to_num(7.0), old[b, n[b]:].nan_to_num(7.0))
        if H:
            want_q = torch.from_numpy(turn(np_(q[b, :n[b]]))).to(dt)
            assert torch.equal(out[b, :n[b]].cpu(), want_q) and not out[b, n[b]:].any()
    assert (out is None) == (H == 0)
    # nothing but the appended tokens changed
    wrote = torch.zeros(cache.num_pages, P, dtype=torch.bool)
    for b in range(B):
        for i in range(n[b]):
            p = starts[b] + i
            wrote[table[b, p // P], p % P] = True
    same = torch.zeros(cache.num_pages, KV, block_bytes(P, D), dtype=torch.bool)
    same |= cache.pages.cpu() == noise
    keep = ~wrote[:, None]
    ends = [0, P * D // 2, P * D, P * (D + D // 32), P * (D + D // 16)]
    for a, z in zip(ends, ends[1:]):
        part = same[:, :, a:z].view(cache.num_pages, KV, P, -1).all(-1)
        assert bool(part[keep.expand_as(part)].all())


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dt", [BF16, FP16])
def test_every_border_of_the_levels_and_the_scales(dt, device):
    """Midpoints between levels (ties to the even code), the 7 s border, the
    smallest and largest numbers of the type, zeros, infinities and NaN."""
    rows = []
    for e in (-3, 0, 5):
        for top in (6.0, 7.0, 7.03125, 4.0, 3.5):
            x = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0]) * 2.0 ** e
            row = torch.cat((x, -x, torch.zeros(4)))
            rows.append(torch.cat((torch.tensor([top * 2.0 ** e]), row[:31])))
    fi = torch.finfo(dt)
    for top in (fi.max, fi.max / 2, fi.tiny, fi.tiny / 4, fi.smallest_subnormal if hasattr(fi, "smallest_subnormal") else 0.0,
                0.0, float("inf"), float("nan"), -float("inf")):
        rows.append(torch.cat((torch.tensor([top]), torch.linspace(-1, 1, 31) * (top if math.isfinite(top) else 1.0))))
    x = torch.stack(rows).to(dt)
    x = torch.cat((x, x.flip(0)), 1)  # [n, 64]: two groups of different scales
    n = x.shape[0]
    cache = PagedKV4.empty(2, 64, 1, 64, dt, device)
    x4 = x.view(1, n, 1, 64).to(device)
    table = torch.tensor([[1]], dtype=torch.int32, device=device)
    zero = torch.zeros(1, dtype=torch.int32, device=device)
    cache.append(x4, x4.flip(1), table, zero)
    k, v = cache.read(table, zero, n)
    want = R.kept(np_(x), dt)
    assert np.array_equal(k[0, :, 0].cpu().double().numpy(), want, equal_nan=True)
    assert np.array_equal(v[0, :, 0].cpu().double().numpy(), want[::-1], equal_nan=True)


@pytest.mark.parametrize("device", DEVICES)
def test_strided_and_broadcast_blocks(device):
    """q, k and v as slices of one projection, values of one head for all,
    tables that are columns of wider ones."""
    B, T, KV, H, D, P = 2, 6, 2, 4, 64, 16
    g = torch.Generator().manual_seed(1)
    qkv = values(g, T, B, (H + 2 * KV) * D + 5, dtype=BF16).to(device).transpose(0, 1)
    q = qkv[..., 1:1 + H * D].unflatten(-1, (H, D))
    k = qkv[..., 1 + H * D:1 + (H + KV) * D].unflatten(-1, (KV, D))
    v = qkv[..., -D:][:, :, None].expand(B, T, KV, D)
    wide = torch.zeros(B, 6, dtype=torch.int32, device=device)
    wide[:, ::2] = R.block_tables(B, 3, 7, 1).to(device)
    starts = torch.tensor([[4, 0], [20, 0]], dtype=torch.int32, device=device)[:, 0]
    cos, sin = (t.to(device) for t in rotation(64, D))
    one = PagedKV4.empty(7, P, KV, D, BF16, device)
    two = PagedKV4.empty(7, P, KV, D, BF16, device)
    a = one.append(k, v, wide[:, ::2], starts, cos=cos, sin=sin, q=q)
    b = two.append(k.contiguous(), v.contiguous(), wide[:, ::2].contiguous(), starts.contiguous(), cos=cos, sin=sin,
                   q=q.contiguous())
    assert torch.equal(one.pages, two.pages) and torch.equal(a, b)
    lengths = starts + T
    x = one.attend(qkv[..., 1:1 + H * D].unflatten(-1, (H, D)), wide[:, ::2], lengths)
    y = two.attend(q.contiguous(), wide[:, ::2].contiguous(), lengths)
    assert torch.equal(x, y) and bool(x.abs().sum() > 0)
    last = two.pages.clone()
    one.append(k[..., :].flip(-1), v, wide[:, ::2], starts, counts=torch.zeros_like(starts))
    assert torch.equal(one.pages, last)


ATTEND = [  # tokens, kv heads, heads, dim, page, dtype, lengths
    (1, 1, 1, 64, 16, BF16, [0, 1, 2, 15, 16, 17, 31, 32, 33]),
    (1, 2, 16, 128, 16, BF16, [63, 64, 65, 127, 128, 129, 257]),
    (4, 2, 8, 128, 32, FP16, [1, 2, 3, 4, 5, 33, 100]),
    (5, 1, 8, 64, 64, BF16, [4, 5, 200, 77]),
    (9, 3, 3, 96, 16, FP16, [9, 31, 50]),
    (2, 1, 7, 192, 128, BF16, [130, 1]),
    (3, 2, 4, 256, 16, FP16, [40, 3, 0]),
    (1, 4, 20, 256, 256, BF16, [300, 511]),
    (20, 1, 5, 128, 16, BF16, [60, 21]),
    (1, 1, 64, 64, 32, FP16, [90, 32]),
    (2, 2, 4, 128, 64, BF16, [3_001, 1_500]),
]


def filled_cache(g, B, P, KV, D, dt, blocks, device, seed, low=122, high=129):
    """A cache of random codes and scales near one, and its block table."""
    N = B * blocks + 1
    pages = torch.randint(0, 256, (N, KV, block_bytes(P, D)), generator=g, dtype=torch.uint8)
    pages[:, :, P * D:] = torch.randint(low, high, (N, KV, P * (D // 16)), generator=g, dtype=torch.uint8)
    return PagedKV4(pages.to(device), P, D, dt, torch.zeros(1, dtype=torch.int32, device=device)), \
        R.block_tables(B, blocks, N, seed)


def stored(cache: PagedKV4, table: torch.Tensor, tokens: int):
    """Keys and values as float64 numpy [requests, tokens, heads, dim]."""
    host = PagedKV4(cache.pages.cpu(), cache.page_size, cache.head_dim, cache.dtype)
    k, v = host.read(table, torch.zeros(table.shape[0], dtype=torch.int32), tokens)
    return k.double().numpy(), v.double().numpy()


def close(got, want, tol):
    got = got.cpu().double().numpy()
    off = np.abs(got - want)
    assert np.isfinite(got).all()
    assert (off <= tol).all(), float((off - tol).max())


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("case", range(len(ATTEND)))
def test_attention_against_plain_form(case, device):
    T, KV, H, D, P, dt, lengths = ATTEND[case]
    print(f"attend case {case} on {device}", flush=True)
    B = len(lengths)
    g = torch.Generator().manual_seed(50 + case)
    blocks = (max(lengths) + P - 1) // P + 1
    cache, table = filled_cache(g, B, P, KV, D, dt, blocks, device, case)
    k, v = stored(cache, table, max(lengths))
    # pages past a request's end are not looked at
    for b, n in enumerate(lengths):
        table[b, (n + P - 1) // P:] = -1
    q = (1.3 * torch.randn(B, T, H, D, generator=g)).to(dt)
    ql = torch.tensor([(T + b) % (T + 1) if b else T + 3 for b in range(B)], dtype=torch.int32) if case % 3 == 2 else None
    to = lambda t: None if t is None else t.to(device)  # noqa: E731
    out = cache.attend(to(q), to(table), to(torch.tensor(lengths, dtype=torch.int32)), query_lens=to(ql),
                       scale=0.2 if case % 4 == 1 else None)
    want, tol = R.attend(q.double().numpy(), k, v, lengths, dt, query_lens=None if ql is None else ql.tolist(),
                         scale=0.2 if case % 4 == 1 else None)
    close(out, want, tol)
    cache.check_errors()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dt", [BF16, FP16])
def test_scores_far_apart_and_garbage_past_the_end(dt, device):
    """One token that outweighs all others, wherever it lies, equal scores,
    and NaN and infinite scales in the slots past the length of the last page."""
    B, D, P, n = 4, 128, 16, 150
    g = torch.Generator().manual_seed(70)
    cache, table = filled_cache(g, B, P, 2, D, dt, 10, device, 1)
    q = torch.randn(B, 1, 8, D, generator=g).to(dt)
    pages = cache.pages.cpu()
    for b, at in enumerate((0, 77, 149)):
        pages[table[b, at // P], :, P * D + at % P * 4:P * D + at % P * 4 + 4] = 127 + 5
    pages[table[3].long(), :, P * D:P * (D + 4)] = 117  # scores of about 0
    for b in range(B):
        last = table[b, (n - 1) // P]
        used = n - (n - 1) // P * P
        for off in (P * D, P * (D + 4)):
            pages[last, :, off + used * 4:off + P * 4] = 255
            pages[last, :, off + used * 4:off + used * 4 + 2] = 254
    cache.pages.copy_(pages)
    k, v = stored(cache, table, n)
    lengths = torch.full((B,), n, dtype=torch.int32, device=device)
    out = cache.attend(q.to(device), table.to(device), lengths)
    close(out, *R.attend(q.double().numpy(), k, v, [n] * B, dt))


@pytest.mark.parametrize("device", DEVICES)
def test_nan_in_a_visible_token_shows_in_its_heads_only(device):
    g = torch.Generator().manual_seed(71)
    cache, table = filled_cache(g, 2, 16, 2, 64, BF16, 3, device, 2)
    cache.pages[int(table[0, 1]), 1, 16 * 64 + 3 * 2] = 255  # a key group of head 1
    q = torch.randn(2, 2, 4, 64, generator=g).to(BF16).to(device)
    out = cache.attend(q, table.to(device), torch.tensor([40, 40], dtype=torch.int32, device=device))
    assert out[0, :, 2:].isnan().all()
    assert not out[0, :, :2].isnan().any() and not out[1].isnan().any()


@pytest.mark.parametrize("device", DEVICES)
def test_pages_and_positions_outside_their_tables(device):
    """Left out and flagged; everything else as without them."""
    g = torch.Generator().manual_seed(72)
    P, D, KV = 16, 64, 2
    cache, table = filled_cache(g, 3, P, KV, D, BF16, 4, device, 3)
    k, v = stored(cache, table, 64)
    table[0, 1], table[1, 0], table[2, 3] = -1, cache.num_pages, 2 ** 31 - 1
    k[0, 16:32], k[1, :16], k[2, 48:] = np.nan, np.nan, np.nan
    q = torch.randn(3, 2, 4, D, generator=g).to(BF16)
    lengths = [50, 40, 64]
    out = cache.attend(q.to(device), table.to(device), torch.tensor(lengths, dtype=torch.int32, device=device))
    close(out, *R.attend(q.double().numpy(), k, v, lengths, BF16))
    with pytest.raises(IndexError):
        cache.check_errors()
    cache.check_errors()
    # a length past the table: its tokens are not there
    table2 = R.block_tables(3, 4, cache.num_pages, 3)
    k, v = stored(cache, table2, 64)
    far = torch.tensor([65, 1_000_000, 2 ** 31 - 1], dtype=torch.int32, device=device)
    out = cache.attend(q[:, :1].to(device), table2.to(device), far)
    close(out, *R.attend(q[:, :1].double().numpy(), k, v, [64] * 3, BF16))
    with pytest.raises(IndexError):
        cache.check_errors()
    # nothing visible at all
    none = cache.attend(q.to(device), torch.full_like(table2, -5).to(device), far)
    assert not none.any()
    cache.err.zero_()
    # appends: before the start, past the table, past the rotation's table, on bad pages
    pages = cache.pages.clone()
    x = torch.randn(3, 4, KV, D, generator=g).to(BF16).to(device)
    for starts in ([-4, 64, 2 ** 31 - 1], [-2 ** 31, 70, 10_000]):
        cache.append(x, x, table2.to(device), torch.tensor(starts, dtype=torch.int32, device=device))
        assert torch.equal(cache.pages, pages)
        with pytest.raises(IndexError):
            cache.check_errors()
    cos, sin = (t.to(device) for t in rotation(10, D))
    turned = cache.append(x, x, table2.to(device), torch.tensor([10, 20, 63], dtype=torch.int32, device=device), cos=cos,
                          sin=sin, q=x)
    assert torch.equal(cache.pages, pages) and not turned.any()
    cache.append(x, x, torch.full_like(table2, cache.num_pages).to(device), torch.zeros(3, dtype=torch.int32, device=device))
    assert torch.equal(cache.pages, pages)
    with pytest.raises(IndexError):
        cache.check_errors()
    kr, vr = cache.read(table2.to(device), torch.tensor([62, -3, 2 ** 31 - 1], dtype=torch.int32, device=device), 4)
    assert not kr[0, 2:].any() and not kr[1, :3].any() and not vr[2].any() and kr[0, :2].any() and kr[1, 3].any()
    with pytest.raises(IndexError):
        cache.check_errors()


@pytest.mark.parametrize("device", DEVICES)
def test_a_refused_block_is_overwritten(device):
    """Append five, keep two, append four more: as six appended at once."""
    g = torch.Generator().manual_seed(73)
    KV, D, P = 2, 128, 16
    x = values(g, 1, 9, KV, D, dtype=FP16).to(device)
    y = values(g, 1, 5, KV, D, dtype=FP16).to(device)
    table = torch.tensor([[2, 0]], dtype=torch.int32, device=device)
    at = lambda i: torch.tensor([i], dtype=torch.int32, device=device)  # noqa: E731
    one, two = (PagedKV4.empty(3, P, KV, D, FP16, device) for _ in range(2))
    one.append(x[:, :2], x[:, :2], table, at(13))
    one.append(y, y, table, at(15))
    one.append(x[:, 2:], x[:, 2:], table, at(15))
    two.append(x, x, table, at(13))
    for a, b in zip(one.read(table, at(13), 9), two.read(table, at(13), 9)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("device", DEVICES)
def test_block_attention_equals_its_tokens_one_by_one(device):
    """A block of five queries sees what five single tokens see in turn."""
    g = torch.Generator().manual_seed(74)
    cache, table = filled_cache(g, 2, 32, 2, 128, BF16, 3, device, 4)
    q = torch.randn(2, 5, 6, 128, generator=g).to(BF16)
    k, v = stored(cache, table, 96)
    lengths = torch.tensor([96, 37], dtype=torch.int32, device=device)
    block = cache.attend(q.to(device), table.to(device), lengths)
    _, tol = R.attend(q.double().numpy(), k, v, lengths.tolist(), BF16)
    for i in range(5):
        one = cache.attend(q[:, i:i + 1].to(device), table.to(device), lengths - 4 + i)
        close(block[:, i:i + 1], one.cpu().double().numpy(), 2 * tol[:, i:i + 1])


def test_refusals():
    c = PagedKV4.empty(3, 16, 2, 64, BF16, "cpu")
    x = torch.zeros(2, 3, 2, 64, dtype=BF16)
    q = torch.zeros(2, 3, 4, 64, dtype=BF16)
    table = torch.zeros(2, 1, dtype=torch.int32)
    s = torch.zeros(2, dtype=torch.int32)
    cos = torch.zeros(4, 32)
    pages = torch.zeros(3, 2, block_bytes(16, 64), dtype=torch.uint8)
    for bad in (lambda: PagedKV4(pages, 16, 64, torch.float32), lambda: PagedKV4(pages, 16, 80, BF16),
                lambda: PagedKV4(pages, 24, 64, BF16), lambda: PagedKV4(pages, 8, 64, BF16),
                lambda: PagedKV4(pages, 512, 64, BF16), lambda: PagedKV4(pages[:, :, :-1], 16, 64, BF16),
                lambda: PagedKV4(pages.to(torch.int8), 16, 64, BF16), lambda: PagedKV4(pages[:, :0], 16, 64, BF16),
                lambda: PagedKV4(pages, 16, 64, BF16, torch.zeros(1)),
                lambda: c.append(x, x[:, :2], table, s), lambda: c.append(x[:, :, :1], x[:, :, :1], table, s),
                lambda: c.append(x.half(), x.half(), table, s), lambda: c.append(x[..., :32], x[..., :32], table, s),
                lambda: c.append(x, x, table[:1], s), lambda: c.append(x, x, table.long(), s),
                lambda: c.append(x, x, table, s[:1]), lambda: c.append(x, x, table, s.long()),
                lambda: c.append(x, x, table, s, counts=s[:1]), lambda: c.append(x, x, table, s, cos=cos),
                lambda: c.append(x, x, table, s, cos=cos, sin=cos.double()),
                lambda: c.append(x, x, table, s, cos=torch.zeros(4, 33), sin=torch.zeros(4, 33)),
                lambda: c.append(x, x, table, s, q=q[:, :2]), lambda: c.append(x, x, table, s, q=q.float()),
                lambda: c.read(table, s[:1], 3), lambda: c.read(table.long(), s, 3),
                lambda: c.attend(q[:, :, :3], table, s), lambda: c.attend(q.float(), table, s),
                lambda: c.attend(q, table, s.long()), lambda: c.attend(q, table, s, query_lens=s[:1]),
                lambda: c.attend(q, table, s, scale=float("nan")), lambda: c.attend(q[0], table, s)):
        with pytest.raises(RuntimeError):
            bad()
    assert c.attend(q[:0], table[:0], s[:0]).shape == (0, 3, 4, 64)
    assert c.attend(q[:, :0], table, s).shape == (2, 0, 4, 64)
    assert not c.attend(q, table[:, :0], s).any()
    assert c.append(x[:, :0], x[:, :0], table, s, q=q[:, :0]).shape == (2, 0, 4, 64)
    assert c.read(table, s, 0)[0].shape == (2, 0, 2, 64)
    assert sorted(HEAD_DIMS) == list(HEAD_DIMS) and _lib.FLAG_PAGE_RANGE == 4


@pytest.mark.gpu
def test_a_long_request_and_offsets_past_32_bits(dev):
    """40,000 tokens of one request in pages at the far end of a pool of over
    2^32 bytes."""
    P, KV, D = 64, 8, 128
    N = 2 ** 32 // (KV * block_bytes(P, D)) + 700
    pages = torch.zeros((N, KV, block_bytes(P, D)), dtype=torch.uint8, device=dev)
    g = torch.Generator().manual_seed(75)
    n = 40_000
    blocks = -(-n // P)
    part = torch.randint(0, 256, (blocks, KV, block_bytes(P, D)), generator=g, dtype=torch.uint8)
    part[:, :, P * D:] = torch.randint(124, 128, (blocks, KV, P * (D // 16)), generator=g, dtype=torch.uint8)
    order = N - blocks + torch.randperm(blocks, generator=g)
    pages[order.to(dev)] = part.to(dev)
    cache = PagedKV4(pages, P, D, BF16)
    table = order.to(torch.int32)[None].to(dev)
    q = torch.randn(1, 2, 8, D, generator=g).to(BF16)
    out = cache.attend(q.to(dev), table, torch.tensor([n], dtype=torch.int32, device=dev))
    host = PagedKV4(part, P, D, BF16)
    k, v = stored(host, torch.arange(blocks, dtype=torch.int32)[None], n)
    close(out, *R.attend(q.double().numpy(), k, v, [n], BF16))
    x = values(g, 1, 3, KV, D, dtype=BF16)
    at = torch.tensor([n - 2], dtype=torch.int32, device=dev)
    cache.append(x.to(dev), x.to(dev), table, at)
    got = cache.read(table, at, 3)[0]
    # the table ends at n: the third token has no place
    assert np.array_equal(got[:, :2].cpu().double().numpy(), R.kept(np_(x[:, :2]), BF16)) and not got[:, 2].any()


@pytest.mark.gpu
def test_graph_replays_and_another_stream(dev):
    """Append and attention captured, replayed over new inputs, against eager
    calls on a second cache; and on a side stream."""
    g = torch.Generator().manual_seed(76)
    B, T, KV, H, D, P = 3, 2, 2, 8, 128, 16
    one, table = filled_cache(g, B, P, KV, D, BF16, 12, dev, 5)
    two = PagedKV4(one.pages.clone(), P, D, BF16)
    table = table.to(dev)
    cos, sin = (t.to(dev) for t in rotation(200, D))
    x = [torch.randn(B, T, n, D, generator=g).to(BF16).to(dev) for n in (KV, KV, H)]
    starts = torch.tensor([0, 60, 150], dtype=torch.int32, device=dev)

    def step(cache, k, v, q, at):
        return cache.attend(cache.append(k, v, table, at, cos=cos, sin=sin, q=q), table, at + T)

    step(two, *x, starts)
    torch.cuda.synchronize()
    two.pages.copy_(one.pages)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(one, *x, starts)
    for i in range(4):
        for t in x:
            t.copy_(torch.randn(t.shape, generator=g))
        starts += T
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, step(two, *x, starts))
        assert torch.equal(one.pages, two.pages)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = step(two, *x, starts)
    side.synchronize()
    assert torch.equal(out, again)


@pytest.mark.gpu
def test_the_device_refuses_other_devices(dev):
    c = PagedKV4.empty(3, 16, 2, 64, BF16, dev)
    x = torch.zeros(2, 3, 2, 64, dtype=BF16, device=dev)
    s = torch.zeros(2, dtype=torch.int32, device=dev)
    table = torch.zeros(2, 1, dtype=torch.int32, device=dev)
    for bad in (lambda: c.append(x.cpu(), x, table, s), lambda: c.append(x, x, table.cpu(), s),
                lambda: c.attend(x, table, s.cpu()), lambda: c.read(table, s.cpu(), 1)):
        with pytest.raises(RuntimeError):
            bad()
