"""The sequence-model operators inside a forward-mode level, function transforms
and a compiled caller: the same bits, or an error that says what is missing."""

from __future__ import annotations

import pytest
import torch
from torch.autograd import forward_ad

import myelin_amd as myelin
from tests.test_gpu_sequence_functions import CASES, DEV, _leaf

pytestmark = pytest.mark.gpu


def _case(**kw):
    print("case:", " ".join(f"{k}={v}" for k, v in kw.items()), flush=True)


@pytest.mark.parametrize("name", CASES)
def test_forward_mode(name):
    _case(test="sequence_forward_mode", name=name)
    f, shapes = CASES[name]
    xs = [_leaf(*s, seed=i).requires_grad_() for i, s in enumerate(shapes)]

    def result():
        outs = f(*xs)
        diff = [o for o in outs if o.requires_grad]
        return [t.detach() for t in (*outs, *torch.autograd.grad(diff, xs, [torch.ones_like(o) for o in diff]))]

    want = result()
    with forward_ad.dual_level():
        for a, b in zip(want, result()):
            assert torch.equal(a, b)
        for i, x in enumerate(xs):
            dual = [forward_ad.make_dual(x, torch.ones_like(x)) if j == i else t for j, t in enumerate(xs)]
            with pytest.raises(NotImplementedError, match="jvp"):
                f(*dual)


def test_forward_mode_of_a_step():
    _case(test="sequence_forward_mode_step")
    q, k, v, s = _leaf(2, 2, 24), _leaf(2, 1, 24), _leaf(2, 1, 40), _leaf(2, 2, 24, 40)
    decay = torch.tensor([0.5, 0.9], device=DEV)
    want = myelin.decay_attention_step(q, k, v, decay, s)
    with forward_ad.dual_level():
        for a, b in zip(want, myelin.decay_attention_step(q, k, v, decay, s)):
            assert torch.equal(a, b)
        with pytest.raises(ValueError, match="no forward-mode derivative"):
            myelin.decay_attention_step(q, k, v, decay, forward_ad.make_dual(s, torch.ones_like(s)))
    # (vmap has no data to point at)
    with pytest.raises(RuntimeError, match="storage"):
        torch.func.vmap(lambda x: myelin.decay_attention_step(x, k, v, decay, s)[1])(torch.stack((q, q)))


@pytest.mark.parametrize("name", CASES)
def test_transforms(name):
    _case(test="sequence_transforms", name=name)
    f, shapes = CASES[name]
    xs = [_leaf(*s, seed=i) for i, s in enumerate(shapes)]
    first = lambda x: f(x, *xs[1:])[0]  # noqa: E731
    for transform in (lambda: torch.func.vmap(first)(torch.stack((xs[0], xs[0]))),
                      lambda: torch.func.jvp(first, (xs[0],), (xs[0],)),
                      lambda: torch.func.grad(lambda x: first(x).sum())(xs[0])):
        with pytest.raises(RuntimeError, match="setup_context"):
            transform()


@pytest.mark.parametrize("grad", [False, True])
@pytest.mark.parametrize("name", CASES)
def test_a_compiled_caller(name, grad):
    """The graph breaks at the operators; nothing changes."""

    _case(test="sequence_compiled", name=name, grad=grad)
    f, shapes = CASES[name]
    xs = [_leaf(*s, seed=i).requires_grad_(grad) for i, s in enumerate(shapes)]
    torch._dynamo.reset()
    compiled = torch.compile(lambda *a: [o * 2 if o.is_floating_point() else o for o in f(*a)], backend="eager")
    outs, got = f(*xs), compiled(*xs)
    for a, b in zip(outs, got):
        assert torch.equal(a * 2 if a.is_floating_point() else a, b)
    if grad:
        diff = [(a, b) for a, b in zip(outs, got) if a.requires_grad]
        want = torch.autograd.grad([a for a, _ in diff], xs, [torch.full_like(a, 2.0) for a, _ in diff])
        for a, b in zip(want, torch.autograd.grad([b for _, b in diff], xs, [torch.ones_like(b) for _, b in diff])):
            assert torch.equal(a, b)
