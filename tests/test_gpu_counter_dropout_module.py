"""CounterDropout without a seed: masks from torch's generator of the device,
in eager calls and in a captured graph."""

from __future__ import annotations

import pytest
import torch
import torch.utils.checkpoint

import myelin_amd as myelin

pytestmark = pytest.mark.gpu
DEV = "cuda"


def test_masks_without_a_seed():
    """2^16 elements of which half are kept: independent masks agree in half of
    them, within 5 standard deviations (5 * 128)."""

    print("case: test=counter_dropout_drawn", flush=True)
    n = 2**16
    x, gy = torch.randn(n, device=DEV, requires_grad=True), torch.ones(n, device=DEV)
    drops = [myelin.CounterDropout(0.5).to(DEV) for _ in range(2)]
    torch.manual_seed(4)
    masks = []
    for drop in drops * 2:
        y = drop(x)
        (gx,) = torch.autograd.grad(y, x, gy)
        masks.append(gx != 0)
        assert torch.equal(y.detach(), torch.where(masks[-1], x.detach() * 2.0, 0.0))
    for i, a in enumerate(masks):
        for b in masks[:i]:
            assert abs(int((a == b).sum()) - n // 2) <= 5 * 128
    torch.manual_seed(4)
    assert torch.equal(drops[1](x) != 0, masks[0])


def test_a_captured_graph_draws_at_each_replay():
    print("case: test=counter_dropout_drawn_graph", flush=True)
    n = 2**16
    x, gy = torch.randn(n, device=DEV, requires_grad=True), torch.ones(n, device=DEV)
    drop = myelin.CounterDropout(0.5, time_shared=False).to(DEV)

    def body():
        y = drop(x)
        return y.detach(), torch.autograd.grad(y, x, gy)[0]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            body()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, gx = body()
    masks = []
    for _ in range(4):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, torch.where(gx != 0, x.detach() * 2.0, 0.0))
        masks.append(gx != 0)
        assert abs(int(masks[-1].sum()) - n // 2) <= 5 * 128
    for i, a in enumerate(masks):
        for b in masks[:i]:
            assert abs(int((a == b).sum()) - n // 2) <= 5 * 128


@pytest.mark.parametrize("reentrant", [False, True])
def test_a_checkpointed_layer_keeps_its_mask(reentrant):
    """The same bits as without checkpointing."""

    print(f"case: test=counter_dropout_checkpoint reentrant={reentrant}", flush=True)
    x, w = torch.randn(64, 512, device=DEV), torch.randn(512, 512, device=DEV)
    drops = [myelin.CounterDropout(0.5).to(DEV) for _ in range(2)]

    def layer(drop, t, weight):
        return drop(torch.tanh(t @ weight), t)

    def step(call):
        torch.manual_seed(6)
        leaves = [t.clone().requires_grad_() for t in (x, w)]
        y = call(drops[1], call(drops[0], leaves[0], leaves[1]), leaves[1])
        y.square().sum().backward()
        return y.detach(), [t.grad for t in leaves]

    y0, g0 = step(layer)
    y1, g1 = step(lambda *a: torch.utils.checkpoint.checkpoint(layer, *a, use_reentrant=reentrant))
    assert torch.equal(y0, y1)
    for a, b in zip(g0, g1):
        assert torch.equal(a, b)


def test_a_counted_mask_is_not_drawn_again():
    print("case: test=counter_dropout_checkpoint_counted", flush=True)
    drop = myelin.CounterDropout(0.5, seed=8).to(DEV)
    x = torch.randn(100, device=DEV, requires_grad=True)
    y = torch.utils.checkpoint.checkpoint(lambda t: drop(t * t), x, use_reentrant=False)
    with pytest.raises(RuntimeError, match="leave the seed out"):
        y.sum().backward()
    assert int(drop.offset) == 1
