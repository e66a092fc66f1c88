"""Attention behind a prefix where the requests' own tokens are long: cut into
runs over the device and joined, or a block of eight waves for a unit.

The tolerance is that of tests/test_kv4_shared.py, with at most 7 chunks of a
prefix and 24 runs of a unit to join."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from bpdecode_amd._lib import lib
from tests import _spec_ref as R
from tests.test_kv4 import BF16, FP16, stored
from tests.test_kv4_shared import close, shared_cache

MOST = 16 * 64  # own tokens up to which a unit is one block's, in any case

CASES = [  # tokens, kv heads, heads, dim, page, dtype, shared, lengths of the whole requests; are units cut into runs?
    # few requests: one whose queries do not see the prefix, one that ends at it, one a token past it
    (1, 2, 8, 128, 16, BF16, 448, [448 + 5_000, 300, 448 + 1_500, 448, 449], True),
    (5, 1, 8, 128, 32, FP16, 460, [448 + 2_777, 449, 452, 453, 448 + 1_111, 0], True),  # 40 columns, in two groups
    (3, 2, 2, 64, 16, FP16, 192, [192 + 3_001, 100, 194, 195], True),
    (7, 1, 5, 64, 64, BF16, 64, [64 + 1_999, 70, 64 + 4_200], True),
    (2, 2, 6, 96, 16, BF16, 330, [330 + 2_000, 321, 329], True),
    (1, 1, 20, 192, 32, BF16, 448, [448 + 1_300, 448 + 4_100], True),
    (4, 1, 3, 256, 128, FP16, 640, [640 + 1_200, 643, 640 + 2_500, 20], True),
    # more units than a join takes many waves for
    (1, 8, 8, 64, 16, FP16, 320, [320 + 1_700 - 90 * b for b in range(8)] + [200], True),
    # units that have a CU to themselves
    (1, 8, 32, 128, 64, BF16, 448, [448 + 2_000 - 60 * b for b in range(14)] + [448, 100], False),
    (5, 8, 32, 64, 16, FP16, 448, [448 + 1_500 - 30 * b for b in range(14)] + [450, 452], False),
    # units of a middling length that fill the device
    (1, 4, 4, 256, 16, BF16, 128, [128 + 1_300 - 3 * b for b in range(98)] + [128, 9], False),
    (9, 4, 16, 128, 32, FP16, 200, [200 + 1_200 - 11 * b for b in range(46)] + [207, 192], False),
]


@pytest.mark.gpu
@pytest.mark.parametrize("case", range(len(CASES)))
def test_long_requests_behind_a_prefix(case, dev):
    T, KV, H, D, P, dt, shared, lengths, runs = CASES[case]
    B = len(lengths)
    print(f"shared runs case {case}", flush=True)
    g = torch.Generator().manual_seed(400 + case)
    blocks = -(-max(lengths) // P)
    cache, prefix, table, hidden = shared_cache(g, B, P, KV, D, dt, shared, blocks, dev, case)
    whole = shared // P * P
    # the workspace holds what runs leave, behind this prefix, only where there are some
    need = [lib().bpd_kv_attend_shared_workspace_bytes(B, T, H, KV, D, n, prefix.shape[0] * P)
            for n in (prefix.shape[0] * P + MOST, blocks * P)]
    assert (need[1] > need[0]) == runs and blocks * P - prefix.shape[0] * P > MOST
    q = (1.3 * torch.randn(B, T, H, D, generator=g)).to(dt)
    ql = torch.tensor([T - b % 3 if b else T + 1 for b in range(B)], dtype=torch.int32).clamp(min=0) if case % 2 else None
    for b, n in enumerate(lengths):
        hidden[b, -(-n // P):] = -1
    to = lambda t: None if t is None else t.to(dev)  # noqa: E731
    lens = torch.tensor(lengths, dtype=torch.int32)
    args = (to(q), to(prefix), whole if case % 3 else torch.tensor([shared], dtype=torch.int32, device=dev), to(hidden), to(lens))
    out = cache.attend_shared(*args, query_lens=to(ql))
    want = cache.attend(to(q), to(table), to(lens), query_lens=to(ql))
    cache.check_errors()
    rows = list(range(B)) if B < 10 else [0, 1, 7, B - 2, B - 1]
    k, v = stored(cache, table[rows], max(lengths))
    plain, tol = R.attend(q[rows].double().numpy(), k, v, [lengths[r] for r in rows], dt,
                          query_lens=None if ql is None else ql[rows].tolist())
    close(out[rows], plain, tol, v)
    # the others: both are within half a step for the weights and one for the output of the plain form
    most = float(np.abs(v).max())
    assert float((out.double() - want.double()).abs().max()) <= 4 * torch.finfo(dt).eps / 2 * most
    assert torch.equal(out, cache.attend_shared(*args, query_lens=to(ql)))


@pytest.mark.gpu
def test_replays_over_new_lengths(dev):
    """The cut of a captured call's work follows the lengths of each replay."""
    B, T, KV, H, D, P = 3, 2, 2, 8, 128, 16
    g = torch.Generator().manual_seed(41)
    cache, _, table, _ = shared_cache(g, B, P, KV, D, BF16, 448, 300, dev, 6)
    prefix, whole = table[0, :28].clone().to(dev), table.to(dev)
    q = torch.zeros(B, T, H, D, dtype=BF16, device=dev)
    shared, lens = torch.zeros(1, dtype=torch.int32, device=dev), torch.ones(B, dtype=torch.int32, device=dev)
    cache.attend_shared(q, prefix, shared, whole, lens)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = cache.attend_shared(q, prefix, shared, whole, lens)
    for n, lengths in ((448, [4_800, 460, 3_000]), (0, [10, 0, 4_800]), (448, [449, 448, 450]), (300, [301, 4_000, 299]),
                       (448, [4_800, 4_799, 4_798])):
        q.copy_(torch.randn(q.shape, generator=g))
        shared.fill_(n)
        lens.copy_(torch.tensor(lengths))
        want = cache.attend_shared(q, prefix, shared, whole, lens)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        k, v = stored(cache, table, max(lengths))
        close(out, *R.attend(q.double().cpu().numpy(), k, v, lengths, BF16), v)
    cache.check_errors()
