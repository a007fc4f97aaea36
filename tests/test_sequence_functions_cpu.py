"""Forward-mode derivatives and function transforms of the sequence-model
operators, which have rules for neither, on the host: the launches are plain
torch here, so a call that lost a tangent would return a result."""

from __future__ import annotations

import pytest
import torch
from torch.autograd import forward_ad

import myelin_amd as myelin
from myelin_amd import _lib, attention, dropout, log_probs


@pytest.fixture(autouse=True)
def host_launches(monkeypatch):
    monkeypatch.setattr(_lib, "require_device", lambda t, what: None)
    monkeypatch.setattr(dropout, "_launch", lambda x, residual, *rest: x * 1.0)
    monkeypatch.setattr(attention, "_forward", lambda q, k, v, decay, state, lengths, scale: (
        torch.zeros(q.shape[1], q.shape[2], q.shape[3], v.shape[3]), (q.sum(-1, keepdim=True) * v)))

    def rows(x, targets, top, ignore_index):
        s = x.sum(-1)
        return s, s * 2.0, torch.stack((s, s)), None, None

    monkeypatch.setattr(log_probs, "_forward", rows)


def _attention(q, k, v, s):
    return myelin.decay_attention(q, k, v, torch.ones(2), s)[1]


def _dropout(x, r):
    return myelin.counter_dropout(x, 0.3, 5, residual=r)


def _log_probs(x):
    return myelin.token_log_probs(x, torch.zeros(6, dtype=torch.int64)).log_probs


CASES = {
    "attention": (_attention, [(7, 2, 2, 4), (7, 2, 2, 4), (7, 2, 2, 5), (2, 2, 4, 5)]),
    "dropout": (_dropout, [(5, 3), (5, 3)]),
    "log_probs": (_log_probs, [(6, 20)]),
}
EACH = [(name, i) for name, (_, shapes) in CASES.items() for i in range(len(shapes))]


@pytest.mark.parametrize("name,which", EACH)
def test_a_tangent_is_not_lost(name, which):
    f, shapes = CASES[name]
    xs = [torch.ones(s) for s in shapes]
    with forward_ad.dual_level():
        assert f(*xs) is not None  # no tangents: the call goes through
        xs[which] = forward_ad.make_dual(xs[which], torch.ones(shapes[which]))
        with pytest.raises(NotImplementedError, match="jvp"):
            f(*xs)
        with torch.no_grad(), pytest.raises(NotImplementedError, match="jvp"):
            f(*xs)


def test_a_tangent_of_the_decay_is_not_lost():
    q = torch.ones(7, 2, 2, 4)
    with forward_ad.dual_level():
        decay = forward_ad.make_dual(torch.ones(2), torch.ones(2))
        with pytest.raises(NotImplementedError, match="jvp"):
            myelin.decay_attention(q, q, q, decay)
        with pytest.raises(ValueError, match="no forward-mode derivative"):
            myelin.decay_attention_step(q[0], q[0], q[0], decay, torch.ones(2, 2, 4, 4))


@pytest.mark.parametrize("which", range(4))
def test_a_step_refuses_tangents(which):
    xs = [torch.ones(s) for s in ((2, 2, 4), (2, 2, 4), (2, 2, 5), (2, 2, 4, 5))]

    def step(q, k, v, s):
        return myelin.decay_attention_step(q, k, v, torch.ones(2), s)

    with forward_ad.dual_level():
        dual = list(xs)
        dual[which] = forward_ad.make_dual(xs[which], torch.ones(xs[which].shape))
        with pytest.raises(ValueError, match="no forward-mode derivative"):
            step(*dual)

    def only(x):
        return step(*[x if i == which else t for i, t in enumerate(xs)])[1]

    with pytest.raises(ValueError, match="no forward-mode derivative"):
        torch.func.jvp(only, (xs[which],), (torch.ones(xs[which].shape),))


@pytest.mark.parametrize("name", CASES)
def test_function_transforms_say_what_is_missing(name):
    f, shapes = CASES[name]
    xs = [torch.ones(s) for s in shapes]
    first = lambda x: f(x, *xs[1:])  # noqa: E731
    for transform in (lambda: torch.func.vmap(first)(torch.ones(3, *shapes[0])),
                      lambda: torch.func.jvp(first, (xs[0],), (xs[0],)),
                      lambda: torch.func.grad(lambda x: first(x).sum())(xs[0])):
        with pytest.raises(RuntimeError, match="setup_context"):
            transform()
