"""counter_dropout: the mask word for word against the published generator, the
values against float64.

y is one product and at most one sum in fp32 of exact inputs, with 1 / (1 - p)
rounded to fp32: within 3 roundings of 2^-24 of |x / (1 - p)| + |residual|, then
rounded to the type.
"""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

import myelin_amd as myelin
from tests.philox import philox, words

pytestmark = pytest.mark.gpu
DEV = "cuda"
DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16}


def _case(**kw):
    print("case:", " ".join(f"{k}={v}" for k, v in kw.items()), flush=True)


def _keep(shape, p, seed, offset, shared=False):
    shape = shape[1:] if shared else shape
    n = math.prod(shape)
    return torch.from_numpy(words(0, n, seed, offset) >= np.uint64(int(p * 2**32))).reshape(shape)


def _check(y, x, p, seed, offset, residual=None, shared=False):
    """Bit for bit the fp32 product (and sum) rounded once, and that within its
    roundings of the definition in float64."""

    keep = _keep(x.shape, p, seed, offset, shared).expand(x.shape)
    x = x.detach().cpu()
    r = torch.zeros_like(x) if residual is None else residual.detach().cpu()
    scale = torch.tensor(1.0 / (1.0 - p) if p < 1.0 else 0.0, dtype=torch.float32)
    f = torch.where(keep, x.float() * scale, 0.0)
    f = f if residual is None else f + r.float()
    assert torch.equal(y.detach().cpu(), f.to(y.dtype))
    kept = torch.where(keep, x.double() / (1.0 - p) if p < 1.0 else 0.0, 0.0)
    want = kept + r.double()
    assert bool(((f.double() - want).abs() <= 3 * 2.0**-24 * (kept.abs() + r.double().abs())).all())


def test_generator_is_the_published_one():
    """The known answers that its authors publish with it."""

    assert philox((0, 0, 0, 0), (0, 0)) == [0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]
    assert philox((0xFFFFFFFF,) * 4, (0xFFFFFFFF,) * 2) == [0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD]
    assert philox((0x243F6A88, 0x85A308D3, 0x13198A2E, 0x03707344), (0xA4093822, 0x299F31D0)) == [
        0xD16CFE09, 0x94FDCCEB, 0x5001E420, 0x24126EA1]
    got = words(0, 8, 0x299F31D0A4093822, 0x0370734413198A2E)
    assert list(got[:4]) == philox((0, 0, 0x13198A2E, 0x03707344), (0xA4093822, 0x299F31D0))
    assert list(got[4:]) == philox((1, 0, 0x13198A2E, 0x03707344), (0xA4093822, 0x299F31D0))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(), (1,), (3,), (4,), (5,), (8,), (9,), (63,), (1000,), (4097,), (7, 33), (3, 5, 31),
                                   (2, 4, 64), (130, 3, 65), (1, 40000)])
@pytest.mark.parametrize("shared", [False, True])
def test_values_and_mask(shape, shared, dtype):
    if shared and not shape:
        return
    _case(test="dropout", shape=shape, shared=shared, dtype=dtype)
    g = torch.Generator().manual_seed(len(shape) + sum(shape))
    x = torch.randn(shape, generator=g).to(DTYPES[dtype]).to(DEV)
    res = torch.randn(shape, generator=g).to(DTYPES[dtype]).to(DEV)
    for p, seed, offset in ((0.1, 0, 0), (0.5, 2**62 + 12345, 2**33 + 7), (0.999, 17, 2**63 - 1)):
        y = myelin.counter_dropout(x, p, seed, offset, time_shared=shared)
        assert y.dtype == x.dtype and y.shape == x.shape
        _check(y, x, p, seed, offset, shared=shared)
        z = myelin.counter_dropout(x, p, seed, offset, residual=res, time_shared=shared)
        _check(z, x, p, seed, offset, res, shared=shared)


def test_none_and_all():
    x = torch.randn(1000, device=DEV)
    assert torch.equal(myelin.counter_dropout(x, 0.0, 1), x)
    x[5] = math.nan
    assert torch.equal(myelin.counter_dropout(x, 1.0, 1), torch.zeros_like(x))
    y = myelin.counter_dropout(torch.empty(0, 5, device=DEV), 0.5, 1)
    assert y.shape == (0, 5)
    assert myelin.counter_dropout(torch.empty(0, 5, device=DEV), 0.5, 1, time_shared=True).shape == (0, 5)


def test_dropped_infinities_and_nans_are_dropped():
    x = torch.full((4000,), math.inf, device=DEV)
    x[1::2] = math.nan
    keep = _keep((4000,), 0.5, 3, 4).to(DEV)
    y = myelin.counter_dropout(x, 0.5, 3, 4)
    assert bool((y[~keep] == 0).all()) and not bool(y[keep].isfinite().any())


@pytest.mark.parametrize("p", [0.1, 0.5, 0.9])
def test_share_of_kept_elements(p):
    """Within 5 standard deviations of the binomial's mean; seeds and offsets
    give masks that agree as independent ones do."""

    n = 1 << 20
    x = torch.ones(n, device=DEV)
    masks = [myelin.counter_dropout(x, p, s, o) != 0 for s, o in ((1, 0), (2, 0), (1, 1))]
    for m in masks:
        assert abs(int(m.sum()) - n * (1 - p)) <= 5 * math.sqrt(n * p * (1 - p))
    q = p * p + (1 - p) * (1 - p)
    for a, b in ((0, 1), (0, 2), (1, 2)):
        assert abs(int((masks[a] == masks[b]).sum()) - n * q) <= 5 * math.sqrt(n * q * (1 - q))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape,shared", [((6, 5, 33), False), ((6, 5, 33), True), ((4, 8, 64), True), ((1,), False)])
def test_gradients(shape, shared, dtype):
    """dx is the gradient under the same mask, the residual's the gradient; and
    y is linear, so a difference of two outputs is the product with dx."""

    _case(test="dropout_grad", shape=shape, shared=shared, dtype=dtype)
    g = torch.Generator().manual_seed(5)
    x, r, gy = (torch.randn(shape, generator=g).to(DTYPES[dtype]).to(DEV) for _ in range(3))
    x.requires_grad_()
    r.requires_grad_()
    y = myelin.counter_dropout(x, 0.3, 11, 22, residual=r, time_shared=shared)
    gx, gr = torch.autograd.grad(y, (x, r), gy, retain_graph=True)
    _check(gx, gy, 0.3, 11, 22, shared=shared)
    assert torch.equal(gr, gy) and gx.dtype == x.dtype
    # a gradient that is an expanded scalar
    (gs,) = torch.autograd.grad(y.sum(), x)
    _check(gs, torch.ones_like(x), 0.3, 11, 22, shared=shared)
    d = torch.randint(-4, 5, shape, generator=g).to(x.dtype).to(DEV)
    if dtype == "fp32":
        with torch.no_grad():
            a, b = (myelin.counter_dropout(v, 0.3, 11, 22, time_shared=shared).double() for v in (x + d, x - d))
        slope = float(((a - b) / 2 * gy.double()).sum())
        want = float((gx.double() * d.double()).sum())
        assert abs(slope - want) <= 1e-5 * float((gx.double() * d.double()).abs().sum() + 1)


def test_layouts_broadcasts_and_alignment():
    g = torch.Generator().manual_seed(6)
    for dt in DTYPES.values():
        base = torch.randn(64, 130, generator=g).to(dt).to(DEV)
        for x in (base.t(), base[:, 1:], base[1:, 3:68:2], base[:1].expand(64, 130), base.view(-1)[1:8320 - 7]):
            assert torch.equal(myelin.counter_dropout(x, 0.4, 9), myelin.counter_dropout(x.contiguous(), 0.4, 9))
        row = base[:1].clone().requires_grad_()
        y = myelin.counter_dropout(row.expand(64, 130), 0.4, 9)
        (gr,) = torch.autograd.grad(y.float().sum(), row)
        want = _keep((64, 130), 0.4, 9, 0).double().sum(0, keepdim=True) / 0.6
        # 64 terms of 1 / 0.6 summed by the expansion's own reduction
        assert float((gr.double().cpu() - want).abs().max()) <= (0.5 if dt == torch.bfloat16 else 1e-4)


def test_past_two_to_the_31_elements():
    """4 GiB of bf16: offsets pass 32 bits."""

    _case(test="dropout_large")
    n = 2**31 + 24
    x = torch.ones(n, dtype=torch.bfloat16, device=DEV)
    y = myelin.counter_dropout(x, 0.5, 77, 5)
    for first in (2**31 - 500, n - 1000):
        keep = torch.from_numpy(words(first, 1000 if first + 1000 <= n else n - first, 77, 5) >= np.uint64(2**31))
        assert torch.equal(y[first : first + keep.numel()].cpu() != 0, keep)


def test_offset_on_the_device_and_module_in_a_graph():
    _case(test="dropout_graph")
    x = torch.randn(6, 3, 50, device=DEV, requires_grad=True)
    gy = torch.randn(6, 3, 50, device=DEV)
    at = torch.tensor([41], device=DEV)
    assert torch.equal(myelin.counter_dropout(x, 0.5, 8, at), myelin.counter_dropout(x, 0.5, 8, 41))
    drop = myelin.CounterDropout(0.5, seed=8, time_shared=True).to(DEV)

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
    assert int(drop.offset) == 2
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, gx = body()
    for rep in range(3):
        graph.replay()
        torch.cuda.synchronize()
        offset = 3 + rep
        assert int(drop.offset) == offset
        assert torch.equal(y, myelin.counter_dropout(x.detach(), 0.5, 8, offset, time_shared=True))
        assert torch.equal(gx, myelin.counter_dropout(gy, 0.5, 8, offset, time_shared=True))
    drop.eval()
    assert torch.equal(drop(x), x) and torch.equal(drop(x, gy), x + gy) and int(drop.offset) == 5


def test_a_changed_offset_tensor_is_noticed():
    x = torch.randn(100, device=DEV, requires_grad=True)
    at = torch.zeros(1, dtype=torch.int64, device=DEV)
    y = myelin.counter_dropout(x, 0.5, 8, at)
    at += 1
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


def test_refusals():
    x = torch.zeros(4, 5, device=DEV)
    f = myelin.counter_dropout
    for bad, message in ((lambda: f(x, -0.1, 0), "p must be"), (lambda: f(x, 1.5, 0), "p must be"),
                         (lambda: f(x, math.nan, 0), "p must be"), (lambda: f(x, 0.5, -1), "seed must be"),
                         (lambda: f(x, 0.5, 2**63), "seed must be"), (lambda: f(x, 0.5, 0, -1), "offset must be"),
                         (lambda: f(x.double(), 0.5, 0), "float32 or bfloat16"),
                         (lambda: f(x, 0.5, 0, residual=x[:2]), "residual must match"),
                         (lambda: f(x, 0.5, 0, residual=x.bfloat16()), "device and dtype"),
                         (lambda: f(x, 0.5, 0, torch.zeros(1, device=DEV)), "one int64"),
                         (lambda: f(x, 0.5, 0, torch.zeros(2, dtype=torch.int64, device=DEV)), "one int64"),
                         (lambda: f(x[0, 0], 0.5, 0, time_shared=True), "time dimension"),
                         (lambda: myelin.CounterDropout(2.0), "p must be")):
        with pytest.raises(ValueError, match=message):
            bad()
