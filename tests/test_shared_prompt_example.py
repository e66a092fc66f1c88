"""The example that runs positions of several axes, attention behind a shared
prefix, sampling and verification of truncated logits together."""

from __future__ import annotations

import re
import sys
from pathlib import Path

import pytest
import torch

sys.path.insert(0, str(Path(__file__).resolve().parent.parent / "examples"))
import shared_prompt as E  # noqa: E402

from bpdecode_amd.ops import FsaTensors  # noqa: E402

REQUESTS = [list(b"ab12,"), list(b"12,34,"), [97], list(b"77,ab")]


def run(device, text=30, **kw):
    vocab = E.vocabulary()
    fsa = FsaTensors.build(E.PATTERN, vocab, dense=True).to(device)
    positions = E.prompt_positions(text, 5, 7, 9)
    instruction = [(7 * i) % 256 for i in range(positions.shape[1])]
    out = E.generate(E.Reader(vocab.size, device), fsa, instruction, positions, REQUESTS, tokens=16, device=device, **kw)
    return out, [b"".join(vocab.token_bytes[t] for t in w if t != vocab.eos_id).decode() for w in out]


def begins_a_document(text: str) -> bool:
    done = re.match(r"(ab|ba|[0-9]{2},)*", text).end()
    return text[done:] in ("", "!") or any(re.fullmatch(p, text[done:]) for p in ("a", "b", "[0-9]{1,2}"))


@pytest.mark.parametrize("text", [30, 36, 3])
@pytest.mark.parametrize("drafts", [0, 3])
def test_sharing_the_prompt_changes_nothing_on_the_host(text, drafts):
    """The host's attention sums the same tokens in the same order either way."""
    one, text_one = run("cpu", text, drafts=drafts)
    two, _ = run("cpu", text, drafts=drafts, share=False)
    assert one == two and all(map(begins_a_document, text_one))
    assert len({tuple(w) for w in one}) > 1


def test_without_cuts_for_chance_drafts_change_nothing():
    """At temperature 0 truncated verification writes what single draws write."""
    one, _ = run("cpu", drafts=0, temperature=0.0)
    two, _ = run("cpu", drafts=3, temperature=0.0)
    assert all(a[:16] == b[:16] for a, b in zip(one, two))


@pytest.mark.gpu
@pytest.mark.parametrize("drafts", [0, 3])
def test_the_example_runs_on_the_device(drafts, dev):
    for share in (True, False):
        out, text = run("cuda", drafts=drafts, share=share)
        assert all(map(begins_a_document, text)) and all(len(w) >= 1 for w in out)
    assert torch.cuda.is_available()
