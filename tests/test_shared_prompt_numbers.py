"""Every operator that examples/shared_prompt.py calls on the device, on the
inputs that it meets there, against the host's form of the same call.

Appended pages and rotated queries, tokens and truncated logits have to be
equal, log-probabilities are rounded to float32 on both sides from sums that are
right to 1e-9 (one step of 2^-23).  Of attention the host rounds the output alone
(half a step h), the device the weights and the output, scores as floats: with v
the largest value 3 h v, 2e-5 v for joining the pieces (tests/test_kv4_shared.py),
and twice (D + 4) 2^-24 of the largest sum of |q k| for the scores, of which each
is D times the largest query and key at most."""

from __future__ import annotations

from collections import Counter

import pytest
import torch

from bpdecode_amd import ops
from bpdecode_amd.kv import PagedKV4
from tests.test_shared_prompt_example import run


def on_host(x):
    if isinstance(x, torch.Tensor):
        return x.detach().cpu().clone()
    return {k: on_host(v) for k, v in x.items()} if isinstance(x, dict) else x


def checked(monkeypatch) -> Counter:
    """Wraps the operators; how often each was compared."""
    seen = Counter()

    def host_cache(cache):
        return PagedKV4(cache.pages.cpu(), cache.page_size, cache.head_dim, cache.dtype)

    append = PagedKV4.append

    def checked_append(self, *args, **kw):
        if self.pages.device.type == "cpu":
            return append(self, *args, **kw)
        host = host_cache(self)
        want = append(host, *map(on_host, args), **on_host(kw))
        got = append(self, *args, **kw)
        assert torch.equal(got.cpu(), want) and torch.equal(self.pages.cpu(), host.pages)
        seen["append"] += 1
        return got

    def checked_attend(name):
        call = getattr(PagedKV4, name)

        def f(self, q, *args, **kw):
            if self.pages.device.type == "cpu":
                return call(self, q, *args, **kw)
            host = host_cache(self)
            want = call(host, on_host(q), *map(on_host, args), **on_host(kw)).double()
            got = call(self, q, *args, **kw)
            pages = torch.arange(self.num_pages, dtype=torch.int32)[None]
            k, v = host.read(pages, torch.zeros(1, dtype=torch.int32), self.num_pages * self.page_size)
            k, v, D = float(k.float().nan_to_num(0.0).abs().max()), float(v.float().nan_to_num(0.0).abs().max()), self.head_dim
            scores = (D + 4) * 2.0 ** -24 * D * float(q.float().abs().max()) * k * D ** -0.5
            tol = (3 * torch.finfo(self.dtype).eps / 2 + 2e-5 + 2 * scores) * v
            assert tol < 0.05 * v  # (a bound that tells something)
            off = float((got.cpu().double() - want).abs().max())
            assert off <= tol, (name, off, tol)
            seen[name] += 1
            return got

        return f

    def checked_cut(name, compare):
        call = getattr(ops, name)

        def f(logits, *args, **kw):
            if logits.device.type == "cpu":
                return call(logits, *args, **kw)
            other = on_host(kw)
            if kw.get("out") is logits:
                other["out"] = on_host(logits)
            want = call(other["out"] if "out" in other and other["out"] is not None else on_host(logits), *map(on_host, args), **other)
            got = call(logits, *args, **kw)
            compare(got, want)
            seen[name] += 1
            return got

        return f

    def drawn(got, want):
        assert torch.equal(got[0].cpu(), want[0])
        assert torch.allclose(got[1].cpu().double(), want[1].double(), rtol=2.0 ** -23, atol=1e-8)
        assert len(got) == len(want) == 2 or torch.equal(got[2].cpu(), want[2])

    def cut(got, want):
        assert torch.equal(got.cpu(), want) and bool(want.isfinite().any()) and not bool(want.isfinite().all())

    monkeypatch.setattr(PagedKV4, "append", checked_append)
    for name in ("attend", "attend_shared"):
        monkeypatch.setattr(PagedKV4, name, checked_attend(name))
    for name, compare in (("dense_sample", drawn), ("dense_truncate", cut)):
        monkeypatch.setattr(ops, name, checked_cut(name, compare))
    return seen


@pytest.mark.gpu
@pytest.mark.parametrize("drafts", [0, 3])
@pytest.mark.parametrize("text", [30, 90])
def test_what_the_example_computes_on_the_device(text, drafts, monkeypatch, dev):
    seen = checked(monkeypatch)
    for share in (True, False):
        seen.clear()
        run("cuda", text, drafts=drafts, share=share)
        print(dict(seen), flush=True)
        assert seen["append"] and seen["dense_sample"] and bool(seen["dense_truncate"]) == bool(drafts)
        assert seen["attend"] and bool(seen["attend_shared"]) == share
