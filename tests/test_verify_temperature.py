"""Verification at temperatures and logits next to the end of float32's normal
range: differences of logits are subnormal, their quotients by the temperature
are of order one.  Whole numbers, so host and device have to be equal to the
64-bit form."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from bpdecode_amd import ops

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("V", [61, 2_100])
@pytest.mark.parametrize("temperature", [1.2e-38, 2e-38, 1e-30])
def test_smallest_temperatures(temperature, V, device):
    B = 400
    g = torch.Generator().manual_seed(V)
    t = torch.tensor(temperature, dtype=torch.float32)
    z = (-2.0 * torch.rand(B, 2, V, generator=g).double() * t.double()).float()
    x = torch.randint(0, V, (B, 1), generator=g)
    q = torch.rand(B, 1, V, generator=g)
    w = np.exp(z.double().numpy() / float(t))
    p = w / w.sum(-1, keepdims=True)
    at = np.arange(B)
    px = p[at, 0, x[:, 0]]
    q[at, 0, x[:, 0]] = torch.from_numpy(2.0 * px).float()
    # one of eight steps of a thousandth beside the border
    u = torch.rand(B, 2, generator=g)
    u[:, 0] = torch.from_numpy(px / q[at, 0, x[:, 0]].double().numpy() * (1.0 + (at % 8 - 3.5) * 1e-3)).float()
    stands = u[:, 0].double().numpy() * q[at, 0, x[:, 0]].double().numpy() < px
    rest = np.where(stands[:, None], p[:, 1], np.maximum(p[:, 0] - q[:, 0].double().numpy(), 0.0))
    rest = np.where(rest.sum(1, keepdims=True) > 0, rest, p[:, 0])
    run = rest.cumsum(1)
    token = (run <= u[:, 1:].double().numpy() * run[:, -1:]).sum(1)
    assert 0 < stands.sum() < B
    n, got = ops.dense_verify(z.to(device), x.to(device), u.to(device), draft_probs=q.to(device),
                              temperature=torch.full((B,), float(t), device=device))
    assert np.array_equal(n.cpu().numpy(), stands.astype(np.int32))
    assert np.array_equal(got.cpu().numpy(), token)
