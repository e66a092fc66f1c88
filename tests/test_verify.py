"""Verification of drafted tokens (ops.verify_draft, ops.dense_verify,
ConstraintBatch.verify) against a plain 64-bit form.  Verdicts and tokens are
whole numbers and have to be equal: both sides decide them in 64 bits, so a
uniform number would have to lie within about 1e-12 of a border to tell them
apart (1e-6 for a draft's verdict)."""

from __future__ import annotations

import pytest
import torch

from bpdecode_amd import _lib, ops
from bpdecode_amd.batch import BROKEN, ConstraintBatch
from bpdecode_amd.ops import FsaTensors
from tests import _spec_ref as R
from tests._util import TOY_VOCAB, oracle_table

DTYPES = [torch.float32, torch.bfloat16, torch.float16]
DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


def pack(tok_next: torch.Tensor) -> torch.Tensor:
    S, V = tok_next.shape
    a = torch.nn.functional.pad(tok_next >= 0, (0, -V % 32)).view(S, -1, 32)
    w = (a.to(torch.int64) << torch.arange(32)).sum(-1)
    return torch.where(w >= 2 ** 31, w - 2 ** 32, w).to(torch.int32)


def inputs(B, T, V, C, dtype, probs, seed, grammar=False, temps=None, lens=None):
    """Logits, drafts sampled from a blurred target, uniforms; CPU tensors."""
    g = torch.Generator().manual_seed(seed)
    rn = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    logits = (2.5 * rn(B, T + 1, C)).to(dtype)
    tok_next = states = None
    if grammar:
        S = 7
        tok_next = torch.randint(0, S, (S, V), generator=g, dtype=torch.int32)
        share = torch.tensor([0.9, 0.5, 0.3, 0.7, 0.1, 0.95, 0.02])
        tok_next[torch.rand(S, V, generator=g) >= share[:, None]] = -1
        states = torch.randint(-1, S, (B,), generator=g, dtype=torch.int32)
    toks, qs, s = [], [], states
    for i in range(T):
        z = logits[:, i, :V].float() + 0.8 * rn(B, V)
        if s is not None:
            z = z.masked_fill((tok_next[s.clamp(min=0).long()] < 0) | (s < 0)[:, None], -float("inf"))
        q = torch.softmax(z, -1).nan_to_num(0.0) + 0.0
        x = torch.multinomial(q + 1e-30, 1, generator=g)[:, 0]
        if s is not None:
            s = torch.where(s < 0, s, tok_next[s.clamp(min=0).long(), x])
        toks.append(x)
        qs.append(q)
    st = {"logits": logits, "tokens": torch.stack(toks, 1) if T else torch.zeros(B, 0, dtype=torch.int64),
          "probs": torch.stack(qs, 1).to(probs) if T and probs is not None else None,
          "uniforms": torch.rand(B, T + 1, generator=g), "tok_next": tok_next, "states": states,
          "temps": temps, "lens": lens}
    return st


def reference(st, V):
    np_ = lambda t: None if t is None else t.double().numpy() if t.is_floating_point() else t.numpy()  # noqa: E731
    return R.verify(np_(st["logits"]), np_(st["tokens"]), np_(st["uniforms"]), probs=np_(st["probs"]),
                    lens=np_(st["lens"]), temps=np_(st["temps"]), vocab=V, tok_next=np_(st["tok_next"]),
                    states=np_(st["states"]))


def call(st, V, device, **kw):
    to = lambda t: None if t is None else t.to(device)  # noqa: E731
    tn = st["tok_next"]
    return ops.dense_verify(to(st["logits"]), to(st["tokens"]), to(st["uniforms"]), draft_probs=to(st["probs"]),
                            draft_lens=to(st["lens"]), temperature=1.0 if st["temps"] is None else to(st["temps"]),
                            vocab=V, tok_next=to(tn), allow_bits=None if tn is None else to(pack(tn)),
                            states=to(st["states"]), **kw)


def check(got, want):
    assert got[0].tolist() == want[0]
    assert got[1].tolist() == want[1]
    if want[2] is not None:
        assert got[2].tolist() == want[2]


CASES = [  # B, T, V, C, probs dtype, grammar
    (1, 1, 1, 1, torch.float32, False),
    (3, 0, 65, 65, None, False),
    (1, 3, 1_031, 1_031, torch.float32, False),
    (5, 2, 32, 40, torch.float16, True),
    (9, 4, 4_097, 4_100, torch.bfloat16, True),
    (4, 7, 20_011, 20_011, None, True),
    (2, 9, 33_333, 33_400, torch.float32, True),
    (70, 1, 300, 300, torch.float32, True),
    (2, 63, 130, 130, None, False),
    (1, 2, 151_936, 152_064, torch.bfloat16, False),
]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("case", range(len(CASES)))
def test_against_plain_form(case, dtype, device):
    B, T, V, C, probs, grammar = CASES[case]
    g = torch.Generator().manual_seed(case)
    temps = 0.4 + torch.rand(B, generator=g)
    if case % 2:
        temps[::3] = 0.0
    lens = torch.randint(-1, T + 2, (B,), generator=g, dtype=torch.int32) if case % 3 == 1 else None
    st = inputs(B, T, V, C, dtype, probs, 100 + case, grammar, temps, lens)
    print(f"verify case {case} {dtype} on {device}", flush=True)
    check(call(st, V, device), reference(st, V))


@pytest.mark.parametrize("device", DEVICES)
def test_columns_past_the_vocabulary_and_nan_in_rejected_places(device):
    st = inputs(6, 3, 70, 90, torch.float32, torch.float32, 5, True)
    st["logits"][:, :, 70:] = float("inf")
    want = reference(st, 70)
    s = st["states"].clone()
    for i in range(4):  # NaN and infinities wherever the grammar rejects
        bad = (st["tok_next"][s.clamp(min=0).long()] < 0) | (s < 0)[:, None]
        st["logits"][:, i, :70][bad] = float("nan") if i % 2 else float("inf")
        if i < 3:
            s = torch.where(s < 0, s, st["tok_next"][s.clamp(min=0).long(), st["tokens"][:, i]])
    check(call(st, 70, device), want)


@pytest.mark.parametrize("device", DEVICES)
def test_rows_that_allow_nothing(device):
    """All -inf, an allowed NaN, an allowed +inf, a state past the table."""
    st = inputs(5, 2, 50, 50, torch.bfloat16, torch.float32, 6)
    st["uniforms"][:, :2] = 0.0  # every draft stands where its row has a softmax
    st["logits"][0, 0] = -float("inf")
    st["logits"][1, 1, 17] = float("nan")
    st["logits"][2, 2, 49] = float("inf")
    st["logits"][3, 2] = torch.finfo(torch.bfloat16).min  # equal, and as low as the type goes
    err = torch.zeros(1, dtype=torch.int32, device=device)
    n, tok = call(st, 50, device, err=err)
    assert n.tolist() == [0, 1, 2, 2, 2]
    assert tok[:3].tolist() == [-1, -1, -1] and int(tok[3]) == int(st["uniforms"][3, 2].double() * 50)
    assert int(err) == _lib.FLAG_LOGITS
    st = inputs(3, 2, 50, 50, torch.float32, None, 7, True)
    st["states"] = torch.tensor([7, -2, 2 ** 30], dtype=torch.int32)
    err.zero_()
    n, tok, state = call(st, 50, device, err=err)
    assert n.tolist() == [0, 0, 0] and tok.tolist() == [-1] * 3 and state.tolist() == [-1] * 3
    assert int(err) == _lib.FLAG_STATE_RANGE


@pytest.mark.parametrize("device", DEVICES)
def test_draft_that_equals_the_target_always_stands(device):
    """q = p: the drafts of a model that is the target itself."""
    g = torch.Generator().manual_seed(8)
    z = torch.randn(40, 4, 257, generator=g)
    p = torch.softmax(z.double(), -1)
    x = torch.multinomial(p[:, :3].reshape(-1, 257), 1, generator=g).view(40, 3)
    q = (p[:, :3] * (1 - 1e-5)).float()
    st = {"logits": z, "tokens": x, "probs": q, "uniforms": torch.rand(40, 4, generator=g), "tok_next": None,
          "states": None, "temps": None, "lens": None}
    n, _ = call(st, 257, device)
    assert n.tolist() == [3] * 40


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("draft", ["sampled", "certain"])
def test_emitted_tokens_are_distributed_as_the_target(draft, device):
    """First emitted token over many rows of one distribution: shares within
    5 standard deviations of p."""
    N, V = 40_000, 11
    g = torch.Generator().manual_seed(9)
    z = torch.randn(1, 2, V, generator=g)
    q = torch.softmax(torch.randn(V, generator=g), -1)
    x = torch.multinomial(q, N, replacement=True, generator=g)[:, None] if draft == "sampled" else torch.full((N, 1), 4)
    n, tok = ops.dense_verify(z.expand(N, 2, V).to(device), x.to(device), torch.rand(N, 2, generator=g).to(device),
                              draft_probs=q.expand(N, 1, V).contiguous().to(device) if draft == "sampled" else None)
    first = torch.where(n.cpu() > 0, x[:, 0], tok.cpu().long())
    p = torch.softmax(z[0, 0].double(), -1)
    got = torch.bincount(first, minlength=V).double() / N
    assert bool(((got - p).abs() <= 5 * (p * (1 - p) / N).sqrt()).all())


@pytest.mark.parametrize("device", DEVICES)
def test_strides_types_and_a_broadcast_batch(device):
    st = inputs(6, 3, 200, 200, torch.float32, torch.float32, 10, True)
    want = reference(st, 200)
    to = lambda t: t.to(device)  # noqa: E731
    tn = to(st["tok_next"])
    wide = torch.zeros(4, 6, 1_000, device=device)
    wide[:, :, 3:203] = to(st["logits"]).transpose(0, 1)
    qs = torch.zeros(6, 3, 200, 2, device=device)
    qs[..., 1] = to(st["probs"])
    toks = torch.full((6, 7), 9, dtype=torch.int32, device=device)
    toks[:, 1:4] = to(st["tokens"])
    us = torch.zeros(4, 6, device=device)
    us.copy_(to(st["uniforms"]).t())
    got = ops.dense_verify(wide.transpose(0, 1)[:, :, 3:203], toks[:, 1:4], us.t(), draft_probs=qs[..., 1], tok_next=tn,
                           allow_bits=to(pack(st["tok_next"])), states=to(st["states"]).long())
    check(got, want)
    one = {k: (v[:1].expand(5, *v.shape[1:]) if k in ("logits", "tokens", "probs", "uniforms", "states") and v is not None
               else v) for k, v in st.items()}
    got = call(one, 200, device)
    assert [x.tolist() for x in got] == [[w[0]] * 5 for w in want]


@pytest.mark.parametrize("device", DEVICES)
def test_drafted_tokens_outside_the_vocabulary(device):
    """They do not stand, and are flagged; the rest of the row is sampled
    from p where no probabilities were given."""
    st = inputs(3, 2, 40, 40, torch.float32, None, 11, True)
    st["states"][:] = 0
    st["tokens"][0, 0], st["tokens"][1, 0], st["tokens"][2, 0] = -1, 40, 2 ** 40
    err = torch.zeros(1, dtype=torch.int32, device=device)
    got = call(st, 40, device, err=err)
    check(got, reference(st, 40))
    assert got[0].tolist() == [0, 0, 0] and int(err) == _lib.FLAG_TOKEN_RANGE
    st["lens"] = torch.zeros(3, dtype=torch.int32)  # padding past the draft is not looked at
    err.zero_()
    check(call(st, 40, device, err=err), reference(st, 40))
    assert int(err) == 0


@pytest.mark.parametrize("device", DEVICES)
def test_batch_verify_equals_the_walk(device):
    """ConstraintBatch.verify against verify_draft on the same states, and the
    pool it leaves; slots out of order, queued writes, a broken row."""
    for dense in (True, False):
        fsa = FsaTensors.build("[a-c]+(01)*", TOY_VOCAB, dense=dense)
        tn = torch.from_numpy(oracle_table(fsa))
        V = fsa.vocab_size
        batch = ConstraintBatch(fsa, capacity=9, device=device)
        for i in range(8):
            batch.add(i)
        batch.evict(3)
        ids = [6, 0, 5, 2]
        a = TOY_VOCAB.token_bytes.index(b"a")
        batch.commit(ids[:2], torch.tensor([a, 9], dtype=torch.int32, device=device))
        states = torch.tensor([batch.state_of(i) for i in ids], dtype=torch.int32)
        assert BROKEN in states.tolist()
        st = inputs(4, 3, V, V, torch.float32, None, 12)
        st["tokens"][:, 0] = a
        st |= {"tok_next": tn, "states": states}
        want = reference(st, V)
        to = lambda t: t.to(device)  # noqa: E731
        free = ops.verify_draft(to(st["logits"]), to(st["tokens"]), to(st["uniforms"]), fsa.to(device), to(states))
        check(free, want)
        got = batch.verify(ids, to(st["logits"]), to(st["tokens"]), to(st["uniforms"]))
        check((*got, None), (want[0], want[1], None))
        assert [batch.state_of(i) for i in ids] == want[2]
        assert [batch.state_of(i) for i in (1, 4, 7)] == [fsa.start] * 3
        batch.check_errors()


def test_refusals():
    z, x, u = torch.zeros(2, 3, 8), torch.zeros(2, 2, dtype=torch.int32), torch.zeros(2, 3)
    tn = torch.zeros(4, 8, dtype=torch.int32)
    bits, st = pack(tn), torch.zeros(2, dtype=torch.int32)
    ok = ops.dense_verify(z, x, u)
    assert [t.dtype for t in ok] == [torch.int32] * 2
    for bad in (lambda: ops.dense_verify(z[:, :2], x, u),
                lambda: ops.dense_verify(z, x, u[:, :2]),
                lambda: ops.dense_verify(z[0], x, u),
                lambda: ops.dense_verify(z, x, u.double()),
                lambda: ops.dense_verify(z.double(), x, u),
                lambda: ops.dense_verify(z, x, u, vocab=9),
                lambda: ops.dense_verify(z, x, u, vocab=0),
                lambda: ops.dense_verify(z, x, u, temperature=-1.0),
                lambda: ops.dense_verify(z, x, u, temperature=float("inf")),
                lambda: ops.dense_verify(z, x, u, temperature=torch.ones(3)),
                lambda: ops.dense_verify(z, x, u, draft_lens=st[:1]),
                lambda: ops.dense_verify(z, x, u, draft_probs=z),
                lambda: ops.dense_verify(z, x, u, draft_probs=z[:, :2, :7]),
                lambda: ops.dense_verify(z, x, u, draft_probs=z[:, :2].double()),
                lambda: ops.dense_verify(z, x, u, tok_next=tn, allow_bits=bits),
                lambda: ops.dense_verify(z, x, u, tok_next=tn, states=st),
                lambda: ops.dense_verify(z, x, u, allow_bits=bits),
                lambda: ops.dense_verify(z, x, u, tok_next=tn[:3], allow_bits=bits, states=st),
                lambda: ops.dense_verify(z, x, u, tok_next=tn[:, :7], allow_bits=bits, states=st, vocab=8),
                lambda: ops.dense_verify(z, x, u, tok_next=tn, allow_bits=bits, states=st[:1]),
                lambda: ops.dense_verify(z, x, u, tok_next=tn, allow_bits=bits, states=st.long(), write_back=True),
                lambda: ops.dense_verify(z, x, u, allow_bits=bits, bit_rows=x),
                lambda: ops.dense_verify(z, x, u, write_back=True),
                lambda: ops.dense_verify(torch.zeros(1, 65, 8), torch.zeros(1, 64, dtype=torch.int32), torch.zeros(1, 65)),
                lambda: ops.verify_draft(z, x, u, None, st),
                lambda: ops.verify_draft(z, x, u, FsaTensors.build("a", TOY_VOCAB))):
        with pytest.raises(RuntimeError):
            bad()
    assert [t.tolist() for t in ops.dense_verify(z[:0], x[:0], u[:0])] == [[], []]


@pytest.mark.gpu
def test_device_refusals_and_another_stream(dev):
    """Mixed devices are refused; a call on a side stream sees its inputs."""
    st = inputs(8, 4, 5_003, 5_003, torch.bfloat16, torch.float32, 13, True)
    want = reference(st, 5_003)
    with pytest.raises(RuntimeError):
        ops.dense_verify(st["logits"].to(dev), st["tokens"], st["uniforms"].to(dev))
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = call(st, 5_003, dev)
    side.synchronize()
    check(got, want)


@pytest.mark.gpu
def test_graph_replays_equal_eager_calls(dev):
    st = inputs(8, 4, 5_003, 5_003, torch.bfloat16, torch.float32, 14, True)
    sets = [inputs(8, 4, 5_003, 5_003, torch.bfloat16, torch.float32, 15 + i, True) for i in range(4)]
    buf = {k: (v.to(dev) if v is not None else None) for k, v in st.items()}
    bits = pack(st["tok_next"]).to(dev)

    def step():
        return ops.dense_verify(buf["logits"], buf["tokens"], buf["uniforms"], draft_probs=buf["probs"],
                                tok_next=buf["tok_next"], allow_bits=bits, states=buf["states"])

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for s in sets:
        for k in ("logits", "tokens", "uniforms", "probs", "states"):
            buf[k].copy_(s[k])
        graph.replay()
        torch.cuda.synchronize()
        s["tok_next"] = st["tok_next"]
        check(out, reference(s, 5_003))
        check(step(), reference(s, 5_003))
