"""verify_draft against its definition, told one sequence after the other in
float64: whole numbers, equal."""

from __future__ import annotations

import math

import pytest
import torch

import myelin_amd as myelin

pytestmark = pytest.mark.gpu
DEV = "cuda"
DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16}


def _case(**kw):
    print("case:", " ".join(f"{k}={v}" for k, v in kw.items()), flush=True)


def _draw(w, u):
    w = torch.where((w > 0) & (w < math.inf), w, 0.0)
    if not bool((w > 0).any()):
        return None
    cdf = w.cumsum(0)
    at = int(torch.searchsorted(cdf, torch.tensor([u * float(cdf[-1])], dtype=torch.float64), right=True))
    return at if at < w.numel() else int((w > 0).nonzero()[-1])


def _reference(target, tokens, uniforms, draft, lengths):
    target, draft = target.double().cpu(), None if draft is None else draft.double().cpu()
    n, B = tokens.shape
    V = target.shape[2]
    out = torch.full((n + 1, B), -1)
    accepted = torch.zeros(B, dtype=torch.int64)
    for b in range(B):
        drafted = n if lengths is None else min(max(int(lengths[b]), 0), n)
        i = 0
        while i < drafted:
            x = int(tokens[i, b])
            if not 0 <= x < V:
                break
            q = 1.0 if draft is None else float(draft[i, b, x])
            if not float(uniforms[i, b]) * q < float(target[i, b, x]):
                break
            out[i, b] = x
            i += 1
        accepted[b] = i
        p = target[i, b]
        u = float(uniforms[n, b])
        got = None
        if i < drafted:
            if draft is not None:
                rest = p - draft[i, b]
            else:
                rest = p.clone()
                if 0 <= int(tokens[i, b]) < V:
                    rest[int(tokens[i, b])] = 0.0
            got = _draw(rest, u)
        if got is None:
            got = _draw(p, u)
        out[i, b] = -1 if got is None else got
    return accepted, out


def _check(target, tokens, uniforms, draft=None, lengths=None):
    r = myelin.verify_draft(target, tokens, uniforms, draft, lengths=lengths)
    accepted, out = _reference(target, tokens, uniforms, draft, lengths)
    assert r.accepted.dtype == torch.int64 and r.tokens.dtype == torch.int64
    assert torch.equal(r.accepted.cpu(), accepted), (r.accepted.cpu(), accepted)
    assert torch.equal(r.tokens.cpu(), out), (r.tokens.cpu() - out).nonzero()
    return r


def _inputs(n, B, V, dtype, seed=0, noise=0.7):
    g = torch.Generator().manual_seed(seed + 31 * n + 7 * B + V)
    x = 3.0 * torch.randn(n + 1, B, V, generator=g)
    target = torch.softmax(x, -1).to(DTYPES[dtype])
    draft = torch.softmax(x[:n] + noise * torch.randn(n, B, V, generator=g), -1).to(DTYPES[dtype])
    tokens = torch.empty(n, B, dtype=torch.int64)
    for i in range(n):
        tokens[i] = torch.multinomial(draft[i].float(), 1, generator=g)[:, 0]
    uniforms = torch.rand(n + 1, B, generator=g)
    return target.to(DEV), tokens.to(DEV), uniforms.to(DEV), draft.to(DEV)


SIZES = [(1, 1, 1), (0, 3, 20), (3, 5, 2), (4, 40, 63), (8, 3, 1000), (5, 16, 4096), (2, 7, 4097), (12, 4, 9000),
         (3, 2, 100003), (1, 130, 5000), (70, 9, 33), (130, 2, 300), (4, 1, 262147)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,B,V", SIZES)
def test_against_the_definition(n, B, V, dtype):
    _case(test="verify", n=n, B=B, V=V, dtype=dtype)
    g = torch.Generator().manual_seed(n + B + V)
    for noise in (0.1, 1.5):
        target, tokens, uniforms, draft = _inputs(n, B, V, dtype, noise=noise)
        lengths = torch.randint(0, n + 1, (B,), generator=g).to(DEV)
        for q in (draft, None):
            _check(target, tokens, uniforms, q)
            _check(target, tokens, uniforms, q, lengths)
            _check(target, tokens.int(), uniforms, q, lengths.int())


def test_tokens_have_the_target_s_distribution():
    """The first token of each sequence, over 40,000 of them: within 5 standard
    deviations of its count, whether the draft was taken or not."""

    B, V = 40000, 12
    g = torch.Generator().manual_seed(0)
    p, q = (torch.softmax(torch.randn(V, generator=g), -1) for _ in range(2))
    tokens = torch.multinomial(q, B, replacement=True, generator=g)[None].to(DEV)
    uniforms = torch.rand(2, B, generator=g).to(DEV)
    r = myelin.verify_draft(p.to(DEV).expand(2, B, V), tokens, uniforms, q.to(DEV).expand(1, B, V))
    count = torch.bincount(r.tokens[0].cpu(), minlength=V).double()
    room = 5 * torch.sqrt(B * p.double() * (1 - p.double()))
    assert bool(((count - B * p.double()).abs() <= room).all())
    agree = float(torch.minimum(p, q).sum())
    assert abs(int(r.accepted.sum()) - B * agree) <= 5 * math.sqrt(B * agree * (1 - agree))


def test_draws_at_the_borders():
    """Weights of 1 / 8: cumulative ones are exact, and a draw at a border takes the
    token above it."""

    V = 8
    p = torch.full((1, 9, V), 0.125, device=DEV)
    u = torch.tensor([[0.0, 0.125, 0.25, 0.875, 1.0 - 2.0**-24, 0.124999, 1.0, 2.0, math.nan]], device=DEV)
    r = myelin.verify_draft(p, torch.empty(0, 9, dtype=torch.int64, device=DEV), u)
    assert r.tokens[0].tolist() == [0, 1, 2, 7, 7, 0, 7, 7, 7]
    # weights of 0 are never drawn, whatever u
    for V in (100, 5000, 70000):
        p = torch.zeros(1, 4, V, device=DEV)
        p[:, :, V // 2], p[:, :, V // 2 + 3] = 0.5, 0.5
        u = torch.tensor([[0.0, 0.49999, 0.5, 0.99999]], device=DEV)
        r = myelin.verify_draft(p, torch.empty(0, 4, dtype=torch.int64, device=DEV), u)
        assert r.tokens[0].tolist() == [V // 2, V // 2, V // 2 + 3, V // 2 + 3]


def test_every_border_of_a_long_row():
    """u at the cumulative weights of whole numbers: exact sums, so the token right
    behind each border, in every part of the row."""

    V = 20011
    g = torch.Generator().manual_seed(4)
    w = torch.randint(0, 3, (V,), generator=g).float()
    w[0] = w[-1] = 1.0
    # a sum of 2^15: borders are exact multiples of 2^-15
    fill = 2**15 - int(w.sum())
    w[V // 2] += fill
    cdf = w.double().cumsum(0)
    at = torch.cat((torch.arange(0, V - 1, 97), torch.tensor([V - 2])))
    u = (cdf[at] / 2**15).float()
    assert torch.equal(u.double() * 2**15, cdf[at])
    B = at.numel()
    r = myelin.verify_draft(w.to(DEV).expand(1, B, V), torch.empty(0, B, dtype=torch.int64, device=DEV), u[None].to(DEV))
    want = torch.searchsorted(cdf, cdf[at], right=True)
    assert torch.equal(r.tokens[0].cpu(), want)


@pytest.mark.parametrize("V", [6, 5000, 50000])
@pytest.mark.parametrize("dtype", DTYPES)
def test_what_leaves_nothing(V, dtype):
    _case(test="verify_nothing", V=V, dtype=dtype)
    target, tokens, uniforms, draft = _inputs(3, 12, V, dtype)
    uniforms[0] = 0.999
    # 0: q equal to p, refused by u = 1   1: q above p everywhere
    draft[0, 0] = target[0, 0]
    uniforms[0, 0] = 1.0
    draft[0, 1] = target[0, 1] * 2
    # 2: p of zeros   3: p of zeros behind taken tokens   4: p of NaN   5: some NaN
    target[0, 2] = 0.0
    draft[:, 3], target[3, 3], uniforms[:3, 3] = target[:3, 3], 0.0, 0.5
    target[0, 4] = math.nan
    target[:, 5, ::2], draft[:, 6, 1::2] = math.nan, math.nan
    # 7: infinities   8: negative ones   9: the drafted token had no probability
    target[:, 7, 0], draft[:, 8] = math.inf, -0.1
    draft[0, 9, tokens[0, 9]] = 0.0
    # 10: the target gives the drafted token nothing   11: both do
    target[0, 10, tokens[0, 10]] = 0.0
    target[0, 11, tokens[0, 11]] = draft[0, 11, tokens[0, 11]] = 0.0
    r = _check(target, tokens, uniforms, draft)
    assert int(r.tokens[0, 2]) == -1 and int(r.accepted[3]) == 3 and int(r.tokens[3, 3]) == -1
    assert int(r.tokens[0, 4]) == -1 and int(r.accepted[10]) == 0 and int(r.accepted[11]) == 0
    assert int(r.accepted[9]) >= 1
    _check(target, tokens, uniforms)
    uniforms[:, 5] = math.nan
    _check(target, tokens, uniforms, draft)


def test_tokens_outside_the_vocabulary_are_refused():
    target, tokens, uniforms, draft = _inputs(4, 6, 50, "fp32")
    uniforms[:4] = 0.0  # everything else is taken
    tokens[0, 0], tokens[1, 1], tokens[2, 2], tokens[3, 3] = -1, 50, 2**40, -(2**62)
    for q in (draft, None):
        r = _check(target, tokens, uniforms, q)
        assert r.accepted.tolist() == [0, 1, 2, 3, 4, 4]


def test_lengths_are_taken_into_range_and_later_tokens_not_read():
    target, tokens, uniforms, draft = _inputs(5, 7, 30, "fp32")
    lengths = torch.tensor([0, 1, 2, 3, 4, 5, 3], device=DEV)
    want = _check(target, tokens, uniforms, draft, lengths)
    past = torch.arange(5, device=DEV)[:, None] >= lengths
    tokens = torch.where(past, 2**50, tokens)
    draft = torch.where(past[..., None], math.nan, draft)
    got = myelin.verify_draft(target, tokens, uniforms, draft, lengths=lengths)
    assert torch.equal(got.tokens, want.tokens) and torch.equal(got.accepted, want.accepted)
    wide = torch.tensor([-3, 1, 2, 3, 4, 900, 3], device=DEV)
    got = myelin.verify_draft(target, tokens, uniforms, draft, lengths=wide)
    assert torch.equal(got.tokens, want.tokens)
    got = myelin.verify_draft(target, tokens, uniforms, draft, lengths=wide.int())
    assert torch.equal(got.tokens, want.tokens)


@pytest.mark.parametrize("dtype", DTYPES)
def test_layouts(dtype):
    n, B, V = 3, 5, 4100
    g = torch.Generator().manual_seed(2)
    whole = torch.softmax(3 * torch.randn(B, n + 1, 2 * V + 5, generator=g), -1).to(DTYPES[dtype]).to(DEV)
    other = torch.softmax(3 * torch.randn(n, B, V + 3, generator=g), -1).to(DTYPES[dtype]).to(DEV)
    tokens = torch.randint(0, V, (B, n), generator=g).to(DEV).t()
    uniforms = torch.rand(B, n + 1, generator=g).to(DEV).t()
    swapped = whole.transpose(0, 1)
    for i, (p, q) in enumerate(((swapped[..., :V], other[..., :V]), (swapped[..., 1 : V + 1], other[..., 3:]),
                                (swapped[..., : 2 * V : 2], other[..., 1 : V + 1]),
                                (swapped[:, :1, :V].expand(n + 1, B, V), None),
                                (swapped[..., :V], other[:1, :1, :V].expand(n, B, V)))):
        _case(test="verify_layout", dtype=dtype, pair=i)
        a = _check(p, tokens, uniforms, q)
        b = myelin.verify_draft(p.contiguous(), tokens.contiguous(), uniforms.contiguous(),
                                None if q is None else q.contiguous())
        assert torch.equal(a.tokens, b.tokens)


def test_no_sequences():
    r = myelin.verify_draft(torch.empty(3, 0, 5, device=DEV), torch.empty(2, 0, dtype=torch.int64, device=DEV),
                            torch.empty(3, 0, device=DEV))
    assert r.accepted.shape == (0,) and r.tokens.shape == (3, 0)


def test_offsets_past_32_bits():
    _case(test="verify_large")
    n, B, V = 8, 2, 2**27
    p = torch.zeros(n + 1, B, V, dtype=torch.bfloat16, device=DEV)
    tokens = torch.full((n, B), V - 5, device=DEV)
    p[:, :, V - 5], p[:, :, V - 1] = 0.5, 0.25
    u = torch.zeros(n + 1, B, device=DEV)
    u[n] = torch.tensor([0.9, 0.5], device=DEV)
    r = myelin.verify_draft(p, tokens, u)
    assert r.accepted.tolist() == [n, n] and r.tokens[n].tolist() == [V - 1, V - 5]
    u[6, 1] = 0.5
    r = myelin.verify_draft(p, tokens, u)
    assert r.accepted.tolist() == [n, 6] and r.tokens[6:, 1].tolist() == [V - 1, -1, -1]


def test_refusals():
    p = torch.zeros(3, 2, 5, device=DEV)
    t = torch.zeros(2, 2, dtype=torch.int64, device=DEV)
    u = torch.zeros(3, 2, device=DEV)
    q = p[:2]
    n = torch.zeros(2, dtype=torch.int32, device=DEV)
    f = myelin.verify_draft
    for bad, message in ((lambda: f(p[0], t, u), "target_probs must be"), (lambda: f(p[:0], t[:0], u), "target_probs must"),
                         (lambda: f(p[..., :0], t, u), "target_probs must be"),
                         (lambda: f(p.half(), t, u), "float32 or bfloat16"), (lambda: f(p, t, u, p), "draft_probs must be"),
                         (lambda: f(p, t, u, q.bfloat16()), "dtype and device"), (lambda: f(p, t, u, q.cpu()), "dtype and"),
                         (lambda: f(p, t[:1], u), "draft_tokens must be"), (lambda: f(p, t.float(), u), "int64 or int32"),
                         (lambda: f(p, t, u[:2]), "uniforms must be"), (lambda: f(p, t, u.double()), "uniforms must be"),
                         (lambda: f(p, t.cpu(), u), "on the device"), (lambda: f(p, t, u.cpu()), "on the device"),
                         (lambda: f(p, t, u, lengths=n[:1]), "lengths must be"),
                         (lambda: f(p, t, u, lengths=n.cpu()), "lengths must be"),
                         (lambda: f(p, t, u, lengths=n.float()), "lengths must be")):
        with pytest.raises(ValueError, match=message):
            bad()
