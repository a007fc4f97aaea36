"""distillation_loss where the teacher names tokens again and again, at up to 1024
places: the places of a token add up, and to look for them costs no more than to
compare each place with all others once.

A token's probability is a sum of up to K of its places' in their order, within K
2^-24 of it: the bound of test_gpu_distillation.py has that term.
"""

from __future__ import annotations

import math

import pytest
import torch

import myelin_amd as myelin
from tests.test_gpu_distillation import DEV, DTYPES, _case, _close, _reference, _run

pytestmark = pytest.mark.gpu

MAP = 1 << 15  # tokens that are equal modulo this are looked at together


def _tokens(kind, R, V, K, g):
    k = torch.arange(K)
    if kind == "one":
        row = torch.full((K,), V // 3)
    elif kind == "neighbours":
        row = k // 2
    elif kind == "far":  # each again in another 64 places
        row = k % max(40, K // 2)
    elif kind == "few":
        row = torch.randint(0, 5, (K,), generator=g) * (V // 5)
    else:  # distinct, but equal modulo MAP
        row = k // 2 + (k % 2) * MAP
    assert int(row.max()) < V
    return torch.stack([row.roll(r) for r in range(R)])


# a wave to a row; a workgroup to a row, of one tile and of more; rows in parts
SIZES = [(5, 600), (3, 3001), (257, 5000), (2, 40000)]
CASES = [(R, V, K, kind) for R, V in SIZES for K in (65, 128, 300, 1024)
         for kind in ("one", "neighbours", "far", "few")]
CASES += [(R, 34000, K, "alike") for R in (2, 257) for K in (65, 1024)]


@pytest.mark.parametrize("R,V,K,kind", CASES)
def test_repeated_tokens(R, V, K, kind):
    _case(test="distillation_repeats", R=R, V=V, K=K, kind=kind)
    g = torch.Generator().manual_seed(R + V + K)
    dtype = DTYPES["bf16" if K % 2 else "fp32"]
    tokens = _tokens(kind, R, V, K, g)
    values = 3.0 * torch.randn(R, K, generator=g)
    # empty places in either way, some of a token that others name, and one that
    # is 0 in float32
    values[0, 1::7], values[1, 0] = -math.inf, -300.0
    tokens[1, 2::5] = -1
    x = torch.randn(R, V, generator=g).to(dtype).to(DEV)
    weights = torch.randn(R, generator=g).to(DEV)
    tokens, values = tokens.to(DEV), values.to(DEV)
    want = _reference(x, values, tokens, 1.5, weights)
    loss, gx = _run(x, values, tokens, 1.5, weights)
    _close(loss, want[0], "loss")
    _close(gx, want[1], "gradient")
    again = _run(x, values, tokens, 1.5, weights)
    assert torch.equal(loss, again[0]) and torch.equal(gx, again[1])


def test_repeats_beside_a_token_out_of_range():
    """The row is NaN, the others are what they were."""

    g = torch.Generator().manual_seed(3)
    for V in (50, 6000):
        tokens = torch.randint(0, 10, (3, 200), generator=g).to(DEV)
        values = torch.randn(3, 200, generator=g).to(DEV)
        x, weights = torch.randn(3, V, generator=g).to(DEV), torch.ones(3, device=DEV)
        clean = _run(x, values, tokens, 1.0, weights)
        tokens[1, 77] = V
        loss, gx = _run(x, values, tokens, 1.0, weights)
        assert bool(loss[1].isnan()) and bool(gx[1].isnan().all())
        for row in (0, 2):
            assert torch.equal(loss[row], clean[0][row]) and torch.equal(gx[row], clean[1][row])


@pytest.mark.parametrize("V", [1000, 5000, 40000])
@pytest.mark.parametrize("kind", ["one", "neighbours"])
def test_repeats_take_no_milliseconds(V, kind):
    """1024 places compared with 1024, 64 at a time, are 2^14 comparisons of some ten
    instructions, well below a millisecond; one place after the other they are 2^20
    exchanges between lanes, up to 50 of them."""

    _case(test="distillation_repeats_time", V=V, kind=kind)
    g = torch.Generator().manual_seed(4)
    R, K = 4, 1024
    tokens = _tokens(kind, R, V, K, g).to(DEV)
    values = torch.randn(R, K, generator=g).to(DEV)
    leaf = torch.randn(R, V, generator=g).to(DEV).requires_grad_()
    times = []
    for _ in range(6):
        start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        torch.cuda.synchronize()
        start.record()
        myelin.distillation_loss(leaf, values, tokens)
        end.record()
        torch.cuda.synchronize()
        times.append(start.elapsed_time(end))
    print(f"{min(times) * 1e3:.0f} us", flush=True)
    assert min(times) < 2.0, times
