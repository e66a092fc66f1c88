"""The error word that a call hands to its kernels: anything but int32 with an
element on the call's device is refused before a kernel could write to it."""

from __future__ import annotations

import pytest
import torch

from bpdecode_amd import _lib, ops, synth
from bpdecode_amd.batch import ConstraintBatch
from bpdecode_amd.grammar.device import build_pda_tensors, pda_step
from bpdecode_amd.grammar.gbnf import parse_gbnf
from bpdecode_amd.grammar.pda import CompiledGrammar
from bpdecode_amd.kv import PagedKV4, block_bytes
from bpdecode_amd.ops import FsaTensors
from tests._util import PDA_VOCAB

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


def wrong_words(device) -> list[torch.Tensor]:
    other = torch.zeros(1, dtype=torch.int32, device="cpu" if device == "cuda" else "meta")
    return [other, torch.zeros(1, device=device), torch.zeros(1, dtype=torch.int64, device=device),
            torch.zeros(0, dtype=torch.int32, device=device)]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("which", range(4))
def test_verification_refuses_a_wrong_error_word(which, device):
    z, x = torch.zeros(2, 3, 8, device=device), torch.zeros(2, 2, dtype=torch.int32, device=device)
    u = torch.zeros(2, 3, device=device)
    with pytest.raises(RuntimeError, match="err must be int32"):
        ops.dense_verify(z, x, u, err=wrong_words(device)[which])
    good = torch.zeros(1, dtype=torch.int32, device=device)
    ops.dense_verify(z, x, u, err=good)
    assert not int(good)
    ops.dense_verify(z.fill_(float("nan")), x, u, err=good)
    assert int(good)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("which", range(4))
def test_the_cache_refuses_a_wrong_error_word(which, device):
    pages = torch.zeros(2, 1, block_bytes(16, 64), dtype=torch.uint8, device=device)
    with pytest.raises(RuntimeError, match="err must be int32"):
        PagedKV4(pages, 16, 64, torch.bfloat16, wrong_words(device)[which])


@pytest.mark.gpu
@pytest.mark.parametrize("which", range(4))
def test_masks_and_commits_refuse_a_wrong_error_word(which, dev):
    vocab = synth.serving_vocab(512, seed=1)
    dense = FsaTensors.build("[a-z]+", vocab, dense=True).to(dev)
    walked = FsaTensors.build("[a-z]+", vocab, dense=False).to(dev)
    V = dense.vocab_size
    s, x = torch.zeros(2, dtype=torch.int32, device=dev), torch.full((2,), 5, dtype=torch.int32, device=dev)
    z, pool = torch.zeros(2, V, device=dev), torch.zeros(2, _lib.PDA_CONFIG_WORDS, dtype=torch.int32, device=dev)
    g = build_pda_tensors(CompiledGrammar.build(parse_gbnf(synth.JSON_GBNF)), PDA_VOCAB).to(dev)
    bits = dense.ensure_allow_bits()
    calls = (lambda e: ops.dense_mask_(z, dense.tok_next, s, err=e), lambda e: ops.dense_mask_bits_(z, bits, s, err=e),
             lambda e: ops.dense_advance(dense.tok_next, s, x, err=e),
             lambda e: ops.dense_compute_mask(dense.tok_next, s, err=e),
             lambda e: ops.fsa_mask_(z, walked, s, err=e), lambda e: ops.fsa_compute_mask(walked, s, err=e),
             lambda e: ops.fsa_advance(walked, s, x, err=e), lambda e: ops.apply_soft_prior_(z, dense, s, 2, err=e),
             lambda e: pda_step(pool, g, x, err=e))
    for call in calls:
        with pytest.raises(RuntimeError, match="err must be int32"):
            call(wrong_words("cuda")[which])


@pytest.mark.gpu
def test_a_batch_names_what_its_kernels_met(dev):
    """Logits without a softmax are not reported as an index out of range."""
    vocab = synth.serving_vocab(512, seed=1)
    batch = ConstraintBatch(FsaTensors.build("[a-z]+", vocab, dense=True), capacity=2, device=dev)
    batch.add(0)
    z = torch.zeros(1, 2, vocab.size, device=dev)
    x, u = torch.full((1, 1), -7, dtype=torch.int32, device=dev), torch.full((1, 2), 0.5, device=dev)
    batch.verify([0], z, x, u)
    with pytest.raises(IndexError, match="out-of-range index"):
        batch.check_errors()
    batch.reset(0)
    n, token = batch.verify([0], z.fill_(float("nan")), x.fill_(0), u)
    assert (int(n), int(token)) == (0, -1)
    with pytest.raises(IndexError, match="logit was"):
        batch.check_errors()
    batch.check_errors()
