"""Host-side behaviour of a draft model's operators: no CPU fallback, entry points
that check their arguments without launching, and no lost derivative."""

from __future__ import annotations

import ctypes
import math

import pytest
import torch
from torch.autograd import forward_ad

import myelin_amd as myelin
from myelin_amd import _lib, distillation, embedding, gated


def test_cpu_tensors_are_rejected():
    x, t = torch.zeros(3, 2, 4), torch.zeros(3, 2, dtype=torch.int64)
    for call in (lambda: myelin.gated_recurrence(x, x), lambda: myelin.gated_recurrence_step(x[0], x[0], x[0]),
                 lambda: myelin.token_embedding(t, x[0]), lambda: myelin.distillation_loss(x, x, torch.zeros_like(x).long()),
                 lambda: myelin.verify_draft(x, t[:2], x[..., 0])):
        with pytest.raises(ValueError, match="ROCm device"):
            call()


def test_recurrence_entry_points_validate():
    def fwd(x=16, dtype=0, strides=16, out=16, T=4, B=2, N=3):
        _lib.call("myelin_gated_recurrence_fwd", x, 16, dtype, strides, None, None, out, 16, None, T, B, N, None, 0, None)

    for kw, message in ((dict(dtype=1), "unsupported dtype"), (dict(T=0), "T must be positive"), (dict(B=-1), "not neg"),
                        (dict(N=-1), "not negative"), (dict(T=2**31), "too many"), (dict(B=2**30, N=2**30), "too many"),
                        (dict(x=None), "null pointer"), (dict(out=None), "null pointer"),
                        (dict(strides=None), "null pointer")):
        with pytest.raises(ValueError, match=message):
            fwd(**kw)
    # batch rows that a workgroup's 32-bit offsets do not reach
    for stride in (-1, 2**29, 2**62):
        strides = (ctypes.c_int64 * 6)(6, stride, 6, 3, 6, 3)
        with pytest.raises(ValueError, match="batch stride"):
            fwd(strides=strides)
        with pytest.raises(ValueError, match="batch stride"):
            _lib.call("myelin_gated_recurrence_bwd", 16, 16, 16, 0, strides, None, 16, None, 16, 16, 16, 4, 2, 3, None, 0,
                      None)
    fwd(x=None, B=0)  # nothing to do
    fwd(x=None, N=0)
    bwd = ("myelin_gated_recurrence_bwd", 16, 16, 16, 0, 16, None)
    with pytest.raises(ValueError, match="null pointer"):
        _lib.call(*bwd, None, None, 16, 16, 16, 4, 2, 3, None, 0, None)
    with pytest.raises(ValueError, match="unsupported dtype"):
        _lib.call(*bwd[:4], 7, *bwd[5:], 16, None, 16, 16, 16, 4, 2, 3, None, 0, None)
    with pytest.raises(ValueError, match="null pointer"):
        _lib.call("myelin_gated_recurrence_step", 16, 16, 0, 16, None, 16, 16, 2, 3, None)
    kept = _lib.load().myelin_gated_recurrence_kept_elems
    assert kept(1, 2, 3) == 6 and kept(8, 2, 3) == 6 and kept(9, 2, 3) == 12


def test_recurrence_workspace_is_checked():
    """A long sequence of few channels is split over time."""

    need = _lib.load().myelin_gated_recurrence_workspace_elems
    for dtype in (0, 2):
        for backward in (0, 1):
            n = need(dtype, 2**16, 1, 64, backward)
            if n:
                args = ([16, 16, dtype, 16, None, None, 16, 16, None] if not backward else
                        [16, 16, 16, dtype, 16, None, 16, None, 16, 16, 16])
                name = "myelin_gated_recurrence_" + ("bwd" if backward else "fwd")
                with pytest.raises(ValueError, match="workspace of"):
                    _lib.call(name, *args, 2**16, 1, 64, None, 0, None)
                with pytest.raises(ValueError, match="16-byte aligned"):
                    _lib.call(name, *args, 2**16, 1, 64, 8, n, None)


def test_embedding_entry_points_validate():
    def fwd(tokens=16, weight=16, dtype=0, ld=8, M=3, V=5, D=8, scale=1.0):
        _lib.call("myelin_token_embedding", tokens, weight, dtype, ld, 16, M, V, D, scale, 0, None)

    def bwd(tokens=16, dtype=0, gw=16, M=3, V=5, D=8, scale=1.0, ws=None, size=0):
        _lib.call("myelin_token_embedding_bwd", tokens, 16, dtype, gw, M, V, D, scale, 0, ws, size, None)

    for kw, message in ((dict(dtype=1), "unsupported dtype"), (dict(M=-1), "not negative"), (dict(V=0), "positive"),
                        (dict(D=0), "positive"), (dict(M=2**31), "too many"), (dict(V=2**31), "too many"),
                        (dict(scale=math.inf), "finite"), (dict(scale=math.nan), "finite"),
                        (dict(tokens=None), "null pointer")):
        for f in (fwd, bwd):
            with pytest.raises(ValueError, match=message):
                f(**kw)
    with pytest.raises(ValueError, match="row stride"):
        fwd(ld=7)
    with pytest.raises(ValueError, match="null pointer"):
        bwd(gw=None)
    fwd(tokens=None, M=0)
    need = _lib.load().myelin_token_embedding_bwd_workspace_bytes(100000, 1000, 64)
    if need:
        with pytest.raises(ValueError, match="workspace of"):
            bwd(M=100000, V=1000, D=64)
        with pytest.raises(ValueError, match="16-byte aligned"):
            bwd(M=100000, V=1000, D=64, ws=8, size=need)


def test_distillation_entry_points_validate():
    def fwd(x=16, dtype=0, ld=10, values=16, tokens=16, temperature=1.0, R=4, V=10, K=3):
        _lib.call("myelin_distillation_loss", x, dtype, ld, values, tokens, temperature, 16, None, 16, R, V, K, None, 0,
                  None)

    def bwd(x=16, dtype=0, ld=10, probs=16, tokens=16, temperature=1.0, R=4, V=10, K=3):
        _lib.call("myelin_distillation_loss_bwd", x, dtype, ld, tokens, probs, 16, 16, temperature, 16, R, V, K, None)

    for kw, message in ((dict(dtype=1), "unsupported dtype"), (dict(R=-1), "non-negative"), (dict(V=0), "V positive"),
                        (dict(V=2**31, ld=2**31), "below 2"), (dict(ld=9), "row stride"), (dict(K=0), "K must be"),
                        (dict(K=1025), "K must be"), (dict(temperature=0.0), "temperature must"),
                        (dict(temperature=math.nan), "temperature must"),
                        (dict(temperature=math.inf), "temperature must"), (dict(x=None), "null pointer"),
                        (dict(tokens=None), "null pointer")):
        for f in (fwd, bwd):
            with pytest.raises(ValueError, match=message):
                f(**kw)
    with pytest.raises(ValueError, match="null pointer"):
        bwd(probs=None)
    fwd(x=None, R=0)
    bwd(x=None, R=0)


def test_verification_entry_point_validates():
    def f(p=16, dtype=0, tokens=16, n=3, B=2, V=7, ws=16, size=10**6):
        _lib.call("myelin_verify_draft", p, None, dtype, 16, tokens, 16, None, 16, 16, n, B, V, ws, size, None)

    for kw, message in ((dict(dtype=1), "unsupported dtype"), (dict(n=-1), "not negative"), (dict(B=-1), "not neg"),
                        (dict(V=0), "V must be"), (dict(n=2**31), "too many"), (dict(B=2**24), "too many"),
                        (dict(V=2**31), "too many"), (dict(p=None), "null pointer"), (dict(tokens=None), "null pointer"),
                        (dict(ws=None), "workspace of"), (dict(size=8), "workspace of"),
                        (dict(ws=8), "16-byte aligned")):
        with pytest.raises(ValueError, match=message):
            f(**kw)
    f(p=None, B=0)


@pytest.fixture
def host_launches(monkeypatch):
    """Launches in plain torch, so that a call that lost a tangent would return a
    result."""

    monkeypatch.setattr(_lib, "require_device", lambda t, what: None)
    monkeypatch.setattr(gated, "_forward", lambda x, gate, state, lengths, keep: (
        (x * gate).sum(0), x + gate, None))
    monkeypatch.setattr(embedding, "_forward", lambda tokens, weight, scale, padding: weight[tokens] * scale)
    monkeypatch.setattr(distillation, "_forward", lambda x, values, tokens, temperature, keep: (x.sum(-1), values, x[:2]))


def _recurrence(x, gate, state):
    return myelin.gated_recurrence(x, gate, state)[1]


def _embedding(w):
    return myelin.token_embedding(torch.arange(3), w)


def _distillation(x):
    return myelin.distillation_loss(x, torch.ones(6, 2), torch.zeros(6, 2, dtype=torch.int64))


CASES = {
    "recurrence": (_recurrence, [(7, 2, 4), (7, 2, 4), (2, 4)]),
    "embedding": (_embedding, [(5, 3)]),
    "distillation": (_distillation, [(6, 20)]),
}
EACH = [(name, i) for name, (_, shapes) in CASES.items() for i in range(len(shapes))]


@pytest.mark.parametrize("name,which", EACH)
def test_a_tangent_is_not_lost(host_launches, name, which):
    f, shapes = CASES[name]
    xs = [torch.ones(s) for s in shapes]
    with forward_ad.dual_level():
        assert f(*xs) is not None  # no tangents: the call goes through
        xs[which] = forward_ad.make_dual(xs[which], torch.ones(shapes[which]))
        with pytest.raises(NotImplementedError, match="jvp"):
            f(*xs)
        with torch.no_grad(), pytest.raises(NotImplementedError, match="jvp"):
            f(*xs)


def test_tangents_of_a_step_and_of_the_teacher_are_refused(host_launches):
    with forward_ad.dual_level():
        for which in range(3):
            xs = [torch.ones(2, 4) for _ in range(3)]
            xs[which] = forward_ad.make_dual(xs[which], torch.ones(2, 4))
            with pytest.raises(ValueError, match="no forward-mode derivative"):
                myelin.gated_recurrence_step(*xs)
        values = forward_ad.make_dual(torch.ones(6, 2), torch.ones(6, 2))
        with pytest.raises(ValueError, match="no forward-mode derivative"):
            myelin.distillation_loss(torch.ones(6, 20), values, torch.zeros(6, 2, dtype=torch.int64))


@pytest.mark.parametrize("name", CASES)
def test_function_transforms_say_what_is_missing(host_launches, name):
    f, shapes = CASES[name]
    xs = [torch.ones(s) for s in shapes]
    first = lambda x: f(x, *xs[1:])  # noqa: E731
    for transform in (lambda: torch.func.vmap(first)(torch.ones(3, *shapes[0])),
                      lambda: torch.func.jvp(first, (xs[0],), (xs[0],)),
                      lambda: torch.func.grad(lambda x: first(x).sum())(xs[0])):
        with pytest.raises(RuntimeError, match="setup_context"):
            transform()


def test_names_are_public():
    for name in ("gated_recurrence", "gated_recurrence_step", "GatedRecurrence", "token_embedding", "TokenEmbedding",
                 "distillation_loss", "verify_draft", "VerifiedTokens"):
        assert name in myelin.__all__ and hasattr(myelin, name)
