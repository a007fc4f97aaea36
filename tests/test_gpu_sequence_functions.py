"""The sequence-model operators' Python Functions, which tensor subclasses take,
against the C++ ones, which plain tensors do: the same bits, forward and
backward, and the same refusal of second derivatives.  Function transforms, for
which neither has a rule, raise."""

from __future__ import annotations

import pytest
import torch

import myelin_amd as myelin

pytestmark = pytest.mark.gpu
DEV = "cuda"


class Sub(torch.Tensor):
    pass


def _leaf(*shape, dtype=torch.float32, seed=0):
    g = torch.Generator().manual_seed(seed + len(shape) + sum(shape))
    return torch.randn(*shape, generator=g).to(dtype).to(DEV)


def _attention(q, k, v, s):
    decay = torch.tensor([0.5, 0.9], device=DEV)
    return myelin.decay_attention(q, k, v, decay, s, lengths=torch.tensor([70, 33], device=DEV))


def _dropout(x, r):
    return (myelin.counter_dropout(x, 0.3, 5, torch.tensor([9], device=DEV), residual=r, time_shared=True),)


def _log_probs(x):
    r = myelin.token_log_probs(x, torch.arange(6, device=DEV) - 1, top=3, ignore_index=-1)
    return r.log_probs, r.entropy, r.top_log_probs, r.top_tokens


CASES = {
    "attention": (_attention, [(70, 2, 2, 24), (70, 2, 1, 24), (70, 2, 1, 40), (2, 2, 24, 40)]),
    "dropout": (_dropout, [(5, 3, 50), (5, 3, 50)]),
    "log_probs": (_log_probs, [(6, 2000)]),
}


@pytest.mark.parametrize("name", CASES)
def test_subclasses_give_the_same_bits(name):
    print(f"case: test=sequence_functions name={name}", flush=True)
    f, shapes = CASES[name]
    leaves = [_leaf(*s, seed=i) for i, s in enumerate(shapes)]
    results = []
    for kind in (torch.Tensor, Sub):
        xs = [t.detach().clone().as_subclass(kind).requires_grad_() for t in leaves]
        with torch.no_grad():
            quiet = f(*xs)
        outs = f(*xs)
        diff = [o for o in outs if o.requires_grad]
        grads = torch.autograd.grad(diff, xs, [torch.ones_like(o) * 0.5 for o in diff])
        results.append([torch.Tensor(t.detach()) if t.is_floating_point() else t.as_subclass(torch.Tensor)
                        for t in (*quiet, *outs, *grads)])
        g = torch.autograd.grad(f(*xs)[0].sum(), xs[0], create_graph=True)[0]
        with pytest.raises(RuntimeError, match="once_differentiable"):
            g.sum().backward()
    assert len(results[0]) == len(results[1])
    for a, b in zip(*results):
        assert torch.equal(a, b)


@pytest.mark.parametrize("name", CASES)
def test_function_transforms_raise(name):
    f, shapes = CASES[name]
    leaves = [_leaf(3, *s) for s in shapes]
    with pytest.raises(Exception):
        torch.func.vmap(lambda *xs: f(*xs)[0])(*[t.requires_grad_() for t in leaves])
