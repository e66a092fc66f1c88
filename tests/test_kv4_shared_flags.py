"""Which missing pages of a shared prefix are noted: those that some query
sees, on the device as on the host and in PagedKV4.attend."""

from __future__ import annotations

import pytest
import torch

from tests import _spec_ref as R
from tests.test_kv4 import BF16, DEVICES, FP16, stored
from tests.test_kv4_shared import close, shared_cache

P, SHARED = 16, 192  # three tiles, and a missing page in the second (tokens 64 to 79)
GONE = 4
SEEN = [  # tokens of a block, lengths, queries of each request, whether the page is noted
    (1, [20], None, False),
    (1, [64], None, False),
    (1, [65], None, True),
    (1, [0, 20, 63], None, False),
    (1, [20, 300], None, True),
    (1, [20, 300], [1, 0], False),  # no query sees it
    (1, [300, 200, 193], [0, 0, 0], False),
    (3, [194, 30], [3, 3], True),  # sees the prefix, all but its last tokens: not taken from the shared sums
    (3, [66, 30], [3, 3], True),  # with its last two queries
    (3, [66, 30], [3, 0], True),
    (4, [300, 64], [0, 4], False),
    (4, [300, 64], [1, 4], True),
    (1, [50] * 40, None, False),  # three tiles of columns
    (1, [50] * 39 + [192], None, True),
    (2, [300] * 45, [0] * 45, False),
    (2, [300] * 45, [0] * 40 + [1] + [0] * 4, True),
    (2, [300] * 45, [1] + [0] * 44, True),
]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("case", range(len(SEEN)))
@pytest.mark.parametrize("dt,D,share", [(BF16, 128, 2), (FP16, 64, 1)])
def test_only_pages_that_a_query_sees_are_noted(case, dt, D, share, device):
    T, lengths, queries, noted = SEEN[case]
    B, KV = len(lengths), 2
    print(f"flags case {case} {dt} on {device}", flush=True)
    g = torch.Generator().manual_seed(case)
    cache, prefix, table, hidden = shared_cache(g, B, P, KV, D, dt, SHARED, 20, device, case)
    for x in (prefix[None], table):
        x[:, GONE] = -1
    q = torch.randn(B, T, KV * share, D, generator=g).to(dt)
    lens = torch.tensor(lengths, dtype=torch.int32)
    ql = None if queries is None else torch.tensor(queries, dtype=torch.int32)
    to = lambda t: None if t is None else t.to(device)  # noqa: E731
    out = cache.attend_shared(to(q), to(prefix), SHARED, to(hidden), to(lens), query_lens=to(ql))
    assert bool(cache.err.item()) == noted
    cache.err.zero_()
    cache.attend(to(q), to(table), to(lens), query_lens=to(ql))
    assert bool(cache.err.item()) == noted
    cache.err.zero_()
    whole = table.clone()
    whole[:, GONE] = 0
    k, v = stored(cache, whole, 320)
    k[:, GONE * P:(GONE + 1) * P] = float("nan")
    want, tol = R.attend(q.double().numpy(), k, v, lengths, dt, query_lens=queries)
    close(out, want, tol, v)
