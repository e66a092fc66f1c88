"""One number per row for a draw's cuts, in any type that holds it."""

from __future__ import annotations

import pytest
import torch

from bpdecode_amd import ops
from tests.test_kv4 import DEVICES


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.uint8, torch.int8, torch.int16, torch.int32, torch.int64, torch.bool])
def test_top_k_of_every_whole_type(dtype, device):
    g = torch.Generator().manual_seed(17)
    z, u = torch.randn(5, 300, generator=g).to(device), torch.rand(5, generator=g).to(device)
    k = torch.tensor([1, 0, 1, 9, 120]).to(dtype)
    same = [int(x) for x in k]
    k = k.to(device)
    token, logprob = ops.sample(z, u, top_k=k, temperature=0.8)
    cut = ops.truncate(z, top_k=k, temperature=0.8)
    for b, n in enumerate(same):
        one = ops.sample(z[b:b + 1], u[b:b + 1], top_k=n, temperature=0.8)
        assert int(token[b]) == int(one[0]) and float(logprob[b]) == float(one[1])
        assert int(cut[b].isfinite().sum()) == (n or 300)


def test_negative_numbers_of_narrow_types_keep_all():
    z = torch.randn(2, 50)
    for dtype in (torch.int8, torch.int16, torch.int64):
        assert ops.truncate(z, top_k=torch.tensor([-1, -100], dtype=dtype)).isfinite().all()
