"""Verification of drafted tokens where its sums are near a border: uniform
numbers beside a draft's probability, a draft that is the target itself,
vocabularies about the width of a thread's run and of a chunk, a read that is
cut into steps.  Whole numbers, so they have to be equal: both sides decide in
64 bits, and no uniform number lies within 1e-11 of a border."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from bpdecode_amd import ops
from tests import _spec_ref as R
from tests.test_verify import call, check, inputs, reference

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


def softmax64(z: torch.Tensor, t: float = 1.0) -> torch.Tensor:
    return torch.softmax(z.double() / t, -1)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("V", [33, 5_001, 40_000])
def test_uniform_numbers_beside_the_draft_s_probability(V, device):
    """u one float32 above and below p / q: 6e-8 of it, which a sum in 32 bits
    does not resolve."""
    B = 24
    st = inputs(B, 2, V, V, torch.bfloat16, torch.float32, 30)
    p = softmax64(st["logits"])
    at = torch.arange(B)
    px = p[at, 0, st["tokens"][:, 0]]
    qx = torch.clamp(2.0 * px, max=0.9)  # an acceptance of about a half
    st["probs"][at, 0, st["tokens"][:, 0]] = qx.float()
    u = (px / qx.float().double()).float()
    assert bool((u < 1).all())
    even = (at % 2 == 0).numpy()
    st["uniforms"][:, 0] = torch.from_numpy(np.where(even, np.nextafter(u.numpy(), np.float32(0)),
                                                     np.nextafter(u.numpy(), np.float32(2))))
    want = reference(st, V)
    assert [n > 0 for n in want[0]] == even.tolist()
    check(call(st, V, device), want)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("probs", [torch.float32, torch.bfloat16, torch.float16])
def test_a_draft_whose_probabilities_are_the_target_s(probs, device):
    """max(p - q, 0) is what rounding q left: every token lies at its border."""
    B, V = 16, 9_000
    st = inputs(B, 2, V, V, torch.float16, probs, 31)
    st["probs"] = softmax64(st["logits"][:, :2]).to(probs)
    st["uniforms"][:, 0] = 1.0 + 1.0 / 64  # refused whatever the rounding
    check(call(st, V, device), reference(st, V))
    # q = p / 2 and q = 2 p: everything, and nothing, is left
    for f in (0.5, 2.0):
        st["probs"] = (f * softmax64(st["logits"][:, :2])).to(probs)
        st["uniforms"][:, 0] = 4.0
        check(call(st, V, device), reference(st, V))


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("V", [1, 2, 7, 8, 9, 15, 17, 511, 512, 513, 2_047, 2_048, 2_049, 8_193])
def test_vocabularies_about_the_width_of_a_run_and_a_chunk(V, device):
    for dtype in (torch.bfloat16, torch.float32):
        st = inputs(7, 3, V, V + V % 3, dtype, torch.float16 if V % 2 else None, 32 + V, True)
        check(call(st, V, device), reference(st, V))


@pytest.mark.parametrize("device", DEVICES)
def test_long_chunks_with_odd_rows_and_a_grammar(device):
    """Rows that begin at any element, with and without probabilities."""
    V = 70_001
    st = inputs(17, 3, V, V, torch.float16, torch.bfloat16, 33, True)
    st["uniforms"][:, 0] *= 0.3
    check(call(st, V, device), reference(st, V))
    st["probs"] = None
    check(call(st, V, device), reference(st, V))
    st["temps"] = torch.where(torch.arange(17) % 3 == 0, 0.0, 0.7)
    check(call(st, V, device), reference(st, V))


@pytest.mark.parametrize("device", DEVICES)
def test_temperatures_at_the_ends_of_their_range(device):
    """Tiny (all on the largest logits, ties shared), huge (all alike)."""
    V = 700
    st = inputs(6, 2, V, V, torch.float32, None, 34)
    st["logits"][:, :, 5] = st["logits"][:, :, 600] = 40.0
    st["temps"] = torch.tensor([1e-42, 1e-6, 1e-3, 1e6, 1e30, 3e38])
    st["tokens"][:, 0] = 600
    check(call(st, V, device), reference(st, V))
    st["logits"][3:, :, ::7] = 3.0e38  # further apart than the type's largest number
    st["logits"][3:, :, 1::7] = -3.0e38
    st["tokens"][:, 0] = 8
    check(call(st, V, device), reference(st, V))
    st["logits"] = torch.where(torch.arange(V) % 3 == 0, torch.finfo(torch.float32).min, -3.0e38).expand(6, 3, V).contiguous()
    check(call(st, V, device), reference(st, V))


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("B, V", [(5, 5_001), (21, 100_003)])  # the verdicts in the sums' launch, in their own
def test_grammars_that_leave_few_tokens(B, V, device):
    """Two of eight tokens, of which the first weighs nothing; then wider masks
    here and there, and stretches without any token."""
    st = inputs(B, 3, V, V, torch.bfloat16, torch.bfloat16, 36, True)
    st["uniforms"][:, 0] *= 0.3
    t = torch.arange(V)
    every = st["tok_next"].clamp(min=0)
    two = (t % 8 == 1) | (t % 8 == 4)
    st["logits"][:, :, 1::8] = -float("inf")
    st["tok_next"] = torch.where(two, every, -1)
    check(call(st, V, device), reference(st, V))
    mixed = torch.where(t % 3_000 < 40, True, two) & (t // 2_500 % 2 == 1)
    st["tok_next"] = torch.where(mixed, every, -1)
    check(call(st, V, device), reference(st, V))
    st["probs"] = None
    check(call(st, V, device), reference(st, V))


@pytest.mark.gpu
def test_a_read_in_steps_equals_the_host(dev):
    """Positions of more than 48 MiB: read in steps for the requests whose
    drafts stand; blocks of different lengths, some rows greedy."""
    B, T, V = 37, 4, 700_003
    g = torch.Generator().manual_seed(35)
    z = torch.randn(B, T + 1, V, generator=g).mul_(3.0).to(torch.bfloat16)
    x = z[:, :T].argmax(-1)
    x[::5, 2] = 17
    u = torch.rand(B, T + 1, generator=g) * torch.tensor([1e-4, 1e-4, 1e-4, 1.0, 1.0])
    lens = torch.randint(0, T + 1, (B,), generator=g, dtype=torch.int32)
    temp = torch.where(torch.arange(B) % 4 == 1, 0.0, 0.8)
    want = ops.dense_verify(z, x, u, draft_lens=lens, temperature=temp)
    got = ops.dense_verify(z.to(dev), x.to(dev), u.to(dev), draft_lens=lens.to(dev), temperature=temp.to(dev))
    assert [t.tolist() for t in got] == [t.tolist() for t in want]
    assert len(set(want[0].tolist())) > 3


def test_the_plain_form_refuses_what_the_operator_refuses():
    z = np.zeros((1, 1, 4))
    z[0, 0, 2] = np.inf
    assert R.verify(z, np.zeros((1, 0), int), np.zeros((1, 1)))[1] == [-1]
