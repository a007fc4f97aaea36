"""CounterDropout's choice of masks, on the host: ``counter_dropout`` itself is
the numpy generator here."""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch
import torch.utils.checkpoint

import myelin_amd as myelin
from myelin_amd import dropout
from tests.philox import words


def _keep(shape, p, seed, offset):
    n = math.prod(shape)
    return torch.from_numpy(words(0, n, seed, offset) >= np.uint64(int(p * 2**32))).reshape(shape)


@pytest.fixture(autouse=True)
def host_dropout(monkeypatch):
    """counter_dropout on host tensors; the masks of all calls, in order."""

    masks = []

    def counter_dropout(x, p, seed, offset=0, *, residual=None, time_shared=False):
        keep = _keep(x.shape, p, seed, int(offset))
        masks.append(keep)
        y = torch.where(keep, x / (1.0 - p), 0.0)
        return y if residual is None else y + residual

    monkeypatch.setattr(dropout, "counter_dropout", counter_dropout)
    return masks


def test_modules_without_a_seed_have_masks_of_their_own(host_dropout):
    """Masks of independent bits agree in p^2 + (1 - p)^2 of their elements: half
    of them here, within 5 standard deviations."""

    torch.manual_seed(3)
    x = torch.ones(4000)
    drops = [myelin.CounterDropout(0.5) for _ in range(3)]
    for drop in drops * 2:
        drop(x)
    for i, a in enumerate(host_dropout):
        for b in host_dropout[:i]:
            assert abs(int((a == b).sum()) - 2000) <= 5 * math.sqrt(1000)
    torch.manual_seed(3)
    drops[1](x)
    assert torch.equal(host_dropout[-1], host_dropout[0])  # torch's generator decides, not the module


def test_a_seed_fixes_the_masks(host_dropout):
    x = torch.ones(40)
    drop = myelin.CounterDropout(0.5, seed=8)
    for call in (1, 2, 3):
        torch.manual_seed(call)
        drop(x)
        assert torch.equal(host_dropout[-1], _keep((40,), 0.5, 8, call)) and int(drop.offset) == call
    again = myelin.CounterDropout(0.5, seed=8)
    again.load_state_dict(drop.state_dict())
    again(x)
    assert torch.equal(host_dropout[-1], _keep((40,), 0.5, 8, 4))


@pytest.mark.parametrize("seed", [None, 8])
def test_evaluation_draws_nothing(seed, host_dropout):
    x, r = torch.ones(4), torch.full((4,), 2.0)
    drop = myelin.CounterDropout(0.5, seed=seed).eval()
    before = torch.get_rng_state()
    assert torch.equal(drop(x), x) and torch.equal(drop(x, r), x + r)
    assert not host_dropout and int(drop.offset) == 0 and torch.equal(torch.get_rng_state(), before)


@pytest.mark.parametrize("reentrant", [False, True])
def test_a_checkpointed_layer_keeps_its_mask(reentrant, host_dropout):
    """Two checkpointed calls of one module, then the backward pass of both, which
    computes the second first: the gradient is the forward pass's own.  (Whole
    numbers, whose sums are exact in any order.)"""

    torch.manual_seed(5)
    drop = myelin.CounterDropout(0.5)
    x = torch.arange(1.0, 101.0).requires_grad_()
    square = lambda t: drop(t * t)  # noqa: E731
    a = torch.utils.checkpoint.checkpoint(square, x, use_reentrant=reentrant)
    b = torch.utils.checkpoint.checkpoint(square, x, use_reentrant=reentrant)
    (a.sum() + 3.0 * b.sum()).backward()
    first, second = host_dropout[:2]
    assert not torch.equal(first, second)
    assert torch.equal(x.grad, 4.0 * x.detach() * first + 12.0 * x.detach() * second)


@pytest.mark.parametrize("reentrant", [False, True])
def test_a_counted_mask_is_not_drawn_again(reentrant, host_dropout):
    drop = myelin.CounterDropout(0.5, seed=8)
    x = torch.randn(100, requires_grad=True)
    y = torch.utils.checkpoint.checkpoint(lambda t: drop(t * t), x, use_reentrant=reentrant)
    with pytest.raises(RuntimeError, match="leave the seed out"):
        y.sum().backward()
    assert int(drop.offset) == 1
    drop.eval()  # passes in a backward pass too
    y = torch.utils.checkpoint.checkpoint(lambda t: drop(t * t), x, use_reentrant=reentrant)
    y.sum().backward()
    assert torch.equal(x.grad, 2.0 * x.detach())
