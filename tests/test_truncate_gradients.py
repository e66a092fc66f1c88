"""Truncation has no gradient: it refuses logits that want one, and what it
writes in place counts as written."""

from __future__ import annotations

import pytest
import torch

from bpdecode_amd import ops
from bpdecode_amd.batch import ConstraintBatch
from bpdecode_amd.ops import FsaTensors
from tests._util import TOY_VOCAB
from tests.test_kv4 import DEVICES


@pytest.mark.parametrize("device", DEVICES)
def test_logits_that_want_a_gradient_are_refused(device):
    leaf = torch.randn(3, 40, device=device, requires_grad=True)
    before = leaf.detach().clone()
    plain = before.clone()
    for call in (lambda: ops.truncate(leaf, top_k=3), lambda: ops.truncate_(leaf, top_k=3), lambda: ops.truncate(leaf * 2, top_p=0.5),
                 lambda: ops.truncate_(leaf * 2, top_p=0.5), lambda: ops.dense_truncate(leaf, min_p=0.1),
                 lambda: ops.truncate(plain, top_k=3, out=leaf), lambda: ops.truncate(leaf, top_k=3, out=plain)):
        with pytest.raises(RuntimeError, match="no gradient"):
            call()
    assert torch.equal(leaf.detach(), before) and torch.equal(plain, before)
    want = ops.truncate(before, top_k=3)
    with torch.no_grad():
        assert torch.equal(ops.truncate(leaf, top_k=3), want)
    assert torch.equal(ops.truncate(leaf.detach(), top_k=3), want)
    with torch.inference_mode():
        assert torch.equal(ops.truncate(leaf, top_k=3), want)
        assert torch.equal(ops.truncate_(before.clone(), top_k=3), want)


@pytest.mark.parametrize("device", DEVICES)
def test_a_batch_refuses_them_too(device):
    fsa = FsaTensors.build("(ab)*", TOY_VOCAB, dense=True).to(device)
    batch = ConstraintBatch(fsa, capacity=2, device=device)
    batch.add("a")
    z = torch.randn(1, fsa.vocab_size, device=device, requires_grad=True) * 1
    with pytest.raises(RuntimeError, match="no gradient"):
        batch.truncate(["a"], z)
    with torch.no_grad():
        batch.truncate(["a"], z)


@pytest.mark.parametrize("device", DEVICES)
def test_backward_notices_what_was_written(device):
    """Logits that a backward pass still needs, truncated without gradients."""
    for columns in (slice(None), slice(None, None, 2)):  # the second has no neighbouring columns
        x = torch.randn(2, 30, device=device, requires_grad=True)
        z = x * 1.5
        loss = (z * z).sum()
        version = z._version
        with torch.no_grad():
            ops.truncate_(z[:, columns], top_k=2)
        assert z._version > version
        with pytest.raises(RuntimeError, match="inplace"):
            loss.backward()
    z, out = torch.randn(2, 30, device=device), torch.empty(2, 30, device=device)
    version = z._version, out._version
    ops.truncate(z, top_k=2, out=out)
    assert z._version == version[0] and out._version > version[1]
