"""The example that runs the cache, its attention and the verification of
drafts together: drafts change how many steps it takes, not what is written."""

from __future__ import annotations

import re
import sys
from pathlib import Path

import pytest
import torch

sys.path.insert(0, str(Path(__file__).resolve().parent.parent / "examples"))
import speculative as S  # noqa: E402

from bpdecode_amd.ops import FsaTensors  # noqa: E402

PROMPTS = [list(b"ab12,"), list(b"12,34,56,78,"), [97]]


def run(device, **kw):
    vocab = S.vocabulary()
    fsa = FsaTensors.build(S.PATTERN, vocab, dense=True).to(device)
    out, steps = S.generate(S.Model(vocab.size, device), fsa, PROMPTS, tokens=30, device=device, **kw)
    return out, steps, [b"".join(vocab.token_bytes[t] for t in w if t != vocab.eos_id).decode() for w in out]


def begins_a_document(text: str) -> bool:
    """Whether a document of the pattern can begin so: cut at its last whole
    piece, with what is left a piece's beginning."""
    done = re.match(r"(ab|ba|[0-9]{2},)*", text).end()
    return text[done:] in ("", "!") or any(re.fullmatch(p, text[done:]) for p in ("a", "b", "[0-9]{1,2}"))


@pytest.mark.parametrize("drafts", [1, 3, 7])
def test_greedy_drafts_write_what_single_tokens_write(drafts):
    plain, plain_steps, text = run("cpu", drafts=0)
    assert all(map(begins_a_document, text)) and plain_steps == 30
    fast, steps, _ = run("cpu", drafts=drafts)
    assert all(a[:30] == b[:30] for a, b in zip(fast, plain))
    assert steps < plain_steps


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
@pytest.mark.parametrize("temperature", [0.0, 0.9])
def test_what_is_written_obeys_the_grammar(device, temperature):
    out, steps, text = run(device, drafts=4, temperature=temperature)
    assert all(map(begins_a_document, text)), text
    assert all(-1 not in w for w in out) and steps <= 30
    assert all(len(w) >= 30 or w[-1] == S.vocabulary().eos_id for w in out)
    assert torch.tensor([len(w) for w in out]).min() > 0
