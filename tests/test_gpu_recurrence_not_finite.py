"""What a NaN of a gate, or an infinity or a NaN of an initial state, is part of in
gated_recurrence's results and gradients, and what not."""

from __future__ import annotations

import math

import pytest
import torch

from tests.test_gpu_gated_recurrence import DEV, DTYPES, _case, _inputs, _run

pytestmark = pytest.mark.gpu

# segments of one tile, workgroups of several, time cut, a wave to each 64 channels
SIZES = [(60, 2, 5), (900, 2, 70), (6000, 2, 3), (30, 2, 70000)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,B,N", SIZES)
def test_a_gate_that_is_nan(T, B, N, dtype):
    _case(test="recurrence_gate_nan", T=T, B=B, N=N, dtype=dtype)
    x, gate, s = _inputs(T, B, N, dtype)
    at, lengths = T // 2 + 3, torch.tensor([T, T // 2], device=DEV)
    g_out = torch.randn_like(x)
    clean = _run(x, gate, s, lengths, g_out, None)
    bad = gate.clone()
    bad[at, :, 1] = math.nan  # past the second sample's end
    final, out, grads = _run(x, bad, s, lengths, g_out, None)
    later, earlier, both = (torch.zeros_like(x, dtype=torch.bool) for _ in range(3))
    later[at:, 0, 1] = earlier[: at + 1, 0, 1] = both[:, 0, 1] = True
    for got, want, hit in ((out, clean[1], later), (final, clean[0], both[0]), (grads["x"], clean[2]["x"], earlier),
                           (grads["gate"], clean[2]["gate"], both), (grads["initial"], clean[2]["initial"], both[0])):
        assert torch.equal(got[~hit], want[~hit]) and bool(got[hit].isnan().all())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("value", [math.inf, math.nan])
@pytest.mark.parametrize("T,B,N", SIZES)
def test_an_initial_state_that_is_not_finite(T, B, N, value, dtype):
    _case(test="recurrence_state", T=T, B=B, N=N, value=value, dtype=dtype)
    x, gate, s = _inputs(T, B, N, dtype)
    lengths = torch.tensor([T, T // 2], device=DEV)
    g_out = torch.randn_like(x)
    clean = _run(x, gate, s, lengths, g_out, None)
    s = s.clone()
    s[0, 1] = value
    final, out, grads = _run(x, gate, s, lengths, g_out, None)
    hit = torch.zeros_like(x, dtype=torch.bool)
    hit[:, 0, 1] = True
    for got, want, there in ((out, clean[1], hit), (final, clean[0], hit[0]), (grads["gate"], clean[2]["gate"], hit)):
        assert torch.equal(got[~there], want[~there]) and not bool(got[there].isfinite().any())
    for name in ("x", "initial"):
        assert torch.equal(grads[name], clean[2][name])
