"""Appending with rotary positions of several axes (PagedKV4.append with
``positions`` and ``axes``).  What is appended, read back and returned has to be
equal to the plain form: the rotation rounds every product and sum to float32
by itself, whatever row of its tables a pair takes."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from bpdecode_amd import _lib
from bpdecode_amd.kv import PagedKV4
from tests import _spec_ref as R
from tests.test_kv4 import BF16, DEVICES, FP16, np_, rotation, values

CASES = [  # rows, tokens, kv heads, heads, dim, rotary, interleaved, page, dtype, starts, num axes, how the axes lie
    (1, 1, 1, 0, 64, 64, False, 16, BF16, [0], 1, "none"),
    (2, 7, 2, 6, 128, 128, False, 16, BF16, [31, 4], 3, "blocks"),
    (3, 5, 4, 4, 64, 32, True, 32, FP16, [0, 13, 60], 3, "turns"),
    (2, 40, 3, 3, 96, 96, False, 16, BF16, [7, 100], 2, "turns"),
    (4, 3, 1, 7, 256, 256, True, 64, FP16, [0, 62, 63, 64], 4, "blocks"),
    (2, 17, 5, 5, 192, 50, False, 128, BF16, [120, 3], 3, "turns"),
    (2, 9, 2, 2, 128, 6, True, 16, FP16, [8, 15], 2, "blocks"),
    (5, 130, 2, 8, 128, 128, False, 32, BF16, [0, 1, 2, 3, 4], 3, "blocks"),
    (4, 150, 1, 4, 128, 128, True, 16, FP16, [0, 9, 2, 30], 3, "any"),
]


def axes_of(how, pairs, n, g):
    j = torch.arange(pairs)
    if how == "none":
        return None
    if how == "any":
        return torch.randint(0, n, (pairs,), generator=g, dtype=torch.int32)
    return (j % n if how == "turns" else j * n // pairs).to(torch.int32)


def inputs(case):
    B, T, KV, H, D, rot, inter, P, dt, starts, n, how = CASES[case]
    g = torch.Generator().manual_seed(500 + case)
    k, v = values(g, B, T, KV, D, dtype=dt), values(g, B, T, KV, D, dtype=dt, large=0.0)
    q = values(g, B, T, H, D, dtype=dt) if H else None
    positions = torch.randint(0, 300, (n, B, T), generator=g, dtype=torch.int32)
    return g, k, v, q, positions, axes_of(how, rot // 2, n, g), *rotation(300, rot)


def turned(x, cos, sin, positions, axes, inter):
    """float32 [T, heads, D] of one request by positions [axes, T]."""
    row = positions[(axes if axes is not None else torch.zeros(cos.shape[1])).long()].T.long()  # [T, pairs]
    pair = torch.arange(cos.shape[1])
    return R.rotated(np_(x), cos[row, pair][:, None].numpy(), sin[row, pair][:, None].numpy(), inter)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("case", range(len(CASES)))
def test_append_by_axes_equals_the_plain_form(case, device):
    print(f"axes case {case} on {device}", flush=True)
    B, T, KV, H, D, rot, inter, P, dt, starts, n, how = CASES[case]
    g, k, v, q, positions, axes, cos, sin = inputs(case)
    blocks = (max(starts) + T + P - 1) // P
    cache = PagedKV4.empty(B * blocks + 2, P, KV, D, dt, device)
    table = R.block_tables(B, blocks, B * blocks + 2, case)
    counts = torch.tensor([max(0, T - 2 * b) for b in range(B)], dtype=torch.int32) if case % 2 else None
    m = [T] * B if counts is None else counts.tolist()
    to = lambda t: None if t is None else t.to(device)  # noqa: E731
    st = torch.tensor(starts, dtype=torch.int32)
    out = cache.append(to(k), to(v), to(table), to(st), counts=to(counts), cos=to(cos), sin=to(sin), interleaved=inter,
                       q=to(q), positions=to(positions), axes=to(axes))
    cache.check_errors()
    kr, vr = cache.read(to(table), to(st), T, counts=to(counts))
    for b in range(B):
        p = positions[:, b, :m[b]]
        assert np.array_equal(kr[b, :m[b]].cpu().double().numpy(), R.kept(turned(k[b, :m[b]], cos, sin, p, axes, inter), dt))
        assert np.array_equal(vr[b, :m[b]].cpu().double().numpy(), R.kept(np_(v[b, :m[b]]), dt))
        if H:
            assert torch.equal(out[b, :m[b]].cpu(), torch.from_numpy(turned(q[b, :m[b]], cos, sin, p, axes, inter)).to(dt))
            assert not out[b, m[b]:].any()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("case", range(len(CASES)))
def test_positions_that_are_the_places_change_nothing(case, device):
    B, T, KV, H, D, rot, inter, P, dt, starts, n, how = CASES[case]
    g, k, v, q, _, axes, cos, sin = inputs(case)
    to = lambda t: None if t is None else t.to(device)  # noqa: E731
    blocks = (max(starts) + T + P - 1) // P
    table = to(R.block_tables(B, blocks, B * blocks, case))
    st = torch.tensor(starts, dtype=torch.int32)
    same = (st[:, None] + torch.arange(T, dtype=torch.int32)).to(device)
    one, two, three = (PagedKV4.empty(B * blocks, P, KV, D, dt, device) for _ in range(3))
    kw = {"cos": to(cos), "sin": to(sin), "interleaved": inter, "q": to(q)}
    a = one.append(to(k), to(v), table, to(st), **kw)
    b = two.append(to(k), to(v), table, to(st), positions=same, **kw)
    c = three.append(to(k), to(v), table, to(st), positions=same.expand(n, B, T), axes=to(axes), **kw)
    assert torch.equal(one.pages, two.pages) and torch.equal(one.pages, three.pages)
    assert H == 0 or torch.equal(a, b) and torch.equal(a, c)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("inter", [False, True])
def test_positions_at_any_stride(inter, device):
    B, T, KV, H, D, P = 3, 6, 2, 4, 64, 16
    g = torch.Generator().manual_seed(21)
    k, v, q = (values(g, B, T, h, D, dtype=BF16).to(device) for h in (KV, KV, H))
    cos, sin = (t.to(device) for t in rotation(90, D))
    wide = torch.randint(0, 90, (T, 7, B), generator=g, dtype=torch.int32).to(device)
    axes = torch.randint(0, 3, (D,), generator=g, dtype=torch.int32).to(device)[::2]
    table = R.block_tables(B, 1, B, 1).to(device)
    st = torch.tensor([0, 3, 10], dtype=torch.int32, device=device)
    one, two = (PagedKV4.empty(B, P, KV, D, BF16, device) for _ in range(2))
    view = wide[:, 1::2].permute(1, 2, 0)
    a = one.append(k, v, table, st, cos=cos, sin=sin, interleaved=inter, q=q, positions=view, axes=axes)
    b = two.append(k, v, table, st, cos=cos, sin=sin, interleaved=inter, q=q, positions=view.contiguous(), axes=axes.contiguous())
    assert torch.equal(one.pages, two.pages) and torch.equal(a, b)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("rot,inter", [(64, False), (64, True), (20, False)])
def test_positions_outside_the_tables_leave_tokens_out(rot, inter, device):
    """On any axis, also one that no pair takes; the place in the cache is not
    bound by the rotation's tables.  An axis that is not there counts as the
    nearest, and is noted."""
    B, T, KV, D, P = 2, 4, 1, 64, 16
    g = torch.Generator().manual_seed(22)
    k, v, q = (values(g, B, T, 1, D, dtype=BF16) for _ in range(3))
    cos, sin = rotation(8, rot)
    positions = torch.randint(0, 8, (3, B, T), generator=g, dtype=torch.int32)
    positions[1, 0, 2], positions[2, 1, 0], positions[0, 1, 3] = 8, -1, 2 ** 31 - 1
    axes = torch.arange(rot // 2, dtype=torch.int32) % 2
    table = torch.tensor([[0, 1], [2, 3]], dtype=torch.int32)
    st = torch.tensor([20, 9], dtype=torch.int32)
    to = lambda t: t.to(device)  # noqa: E731
    cache = PagedKV4.empty(4, P, KV, D, BF16, device)
    out = cache.append(to(k), to(v), to(table), to(st), cos=to(cos), sin=to(sin), interleaved=inter, q=to(q),
                       positions=to(positions), axes=to(axes))
    with pytest.raises(IndexError):
        cache.check_errors()
    kr, vr = cache.read(to(table), to(st), T)
    for b in range(B):
        for i in range(T):
            if (b, i) in ((0, 2), (1, 0), (1, 3)):
                assert not out[b, i].any() and not kr[b, i].any() and not vr[b, i].any()
                continue
            want = turned(k[b, i:i + 1], cos, sin, positions[:, b, i:i + 1], axes, inter)
            assert np.array_equal(kr[b, i:i + 1].cpu().double().numpy(), R.kept(want, BF16))
    inside = positions.clamp(0, 7)
    odd = torch.where(axes == 0, -3, 9).to(torch.int32)
    a, b = (PagedKV4.empty(4, P, KV, D, BF16, device) for _ in range(2))
    kw = {"cos": to(cos), "sin": to(sin), "interleaved": inter, "positions": to(inside)}
    a.append(to(k), to(v), to(table), to(st), axes=to(odd), **kw)
    with pytest.raises(IndexError):
        a.check_errors()
    b.append(to(k), to(v), to(table), to(st), axes=to(odd.clamp(0, 2)), **kw)
    b.check_errors()
    assert torch.equal(a.pages, b.pages)


@pytest.mark.gpu
def test_replays_of_a_captured_append_by_axes(dev):
    B, T, KV, H, D, P = 3, 2, 2, 4, 128, 16
    g = torch.Generator().manual_seed(23)
    cos, sin = (t.to(dev) for t in rotation(64, D))
    axes = (torch.arange(D // 2, dtype=torch.int32) % 3).to(dev)
    table = R.block_tables(B, 2, 2 * B, 1).to(dev)
    cache, other = (PagedKV4.empty(2 * B, P, KV, D, BF16, dev) for _ in range(2))
    k, v, q = (torch.zeros(B, T, h, D, dtype=BF16, device=dev) for h in (KV, KV, H))
    positions, starts = torch.zeros(3, B, T, dtype=torch.int32, device=dev), torch.zeros(B, dtype=torch.int32, device=dev)
    kw = {"cos": cos, "sin": sin, "positions": positions, "axes": axes, "q": q}
    cache.append(k, v, table, starts, **kw)
    other.append(k, v, table, starts, **kw)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = cache.append(k, v, table, starts, **kw)
    for step in range(4):
        for t in (k, v, q):
            t.copy_(torch.randn(t.shape, generator=g))
        positions.copy_(torch.randint(0, 64, positions.shape, generator=g))
        starts.fill_(7 * step)
        graph.replay()
        torch.cuda.synchronize()
        want = other.append(k, v, table, starts, **kw)
        assert torch.equal(out, want) and torch.equal(cache.pages, other.pages)
    cache.check_errors()


@pytest.mark.parametrize("device", DEVICES)
def test_refusals(device):
    B, T, D = 2, 3, 64
    cache = PagedKV4.empty(2, 16, 1, D, BF16, device)
    k = torch.zeros(B, T, 1, D, dtype=BF16, device=device)
    table, st = torch.zeros(B, 1, dtype=torch.int32, device=device), torch.zeros(B, dtype=torch.int32, device=device)
    cos, sin = (t.to(device) for t in rotation(16, D))
    p, axes = torch.zeros(3, B, T, dtype=torch.int32, device=device), torch.zeros(D // 2, dtype=torch.int32, device=device)
    turn = {"cos": cos, "sin": sin}
    for kw, match in [
        (dict(positions=p, axes=axes), "cos and sin"), (dict(axes=axes, **turn), "axes need positions"),
        (dict(positions=p, **turn), "axis of each channel pair"), (dict(positions=p.long(), axes=axes, **turn), "positions must be"),
        (dict(positions=p[:, :1], axes=axes, **turn), "positions must be"), (dict(positions=p[..., :2], axes=axes, **turn), "positions must be"),
        (dict(positions=p[:0], axes=axes, **turn), "positions must be"),
        (dict(positions=p[:1].expand(_lib.MAX_AXES + 1, B, T), axes=axes, **turn), "positions must be"),
        (dict(positions=p.to("meta"), axes=axes, **turn), "positions must be"), (dict(positions=p, axes=axes[:-1], **turn), "axes must be"),
        (dict(positions=p, axes=axes.long(), **turn), "axes must be"), (dict(positions=p, axes=axes.to("meta"), **turn), "axes must be"),
        (dict(positions=p[0, 0], axes=axes, **turn), "positions must be"),
    ]:
        with pytest.raises(RuntimeError, match=match):
            cache.append(k, k, table, st, **kw)
    assert not cache.pages.any()
