"""token_log_probs against its definition in float64.

Tolerances, for logits within +-100 (spread * normal): the sum of exponentials
is relatively good to about 64 roundings of fp32 (4e-6), so lse and log_probs
are to 1e-5 + 1e-6 |value| absolutely, the entropy, a quotient of two such sums
of terms up to ln V and more, to 1e-5 (1 + ln V), and the gradient to
3e-5 (|g_lp| + |g_ent| (1 + ln V)); a bf16 gradient has its rounding, 2^-8 of
the value, on top.
"""

from __future__ import annotations

import math

import pytest
import torch

import myelin_amd as myelin

pytestmark = pytest.mark.gpu
DEV = "cuda"
INF = math.inf
DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16}


def _case(**kw):
    print("case:", " ".join(f"{k}={v}" for k, v in kw.items()), flush=True)


def _logits(R, V, dtype, seed=0, spread=3.0):
    g = torch.Generator().manual_seed(seed * 7919 + R * 31 + V)
    return (spread * torch.randn(R, V, generator=g)).to(DTYPES[dtype]).to(DEV), g


def _reference(x, targets, top, ignore=-100):
    """(log_probs, entropy, top values, top tokens) in float64 on the CPU."""

    x = x.detach().double().cpu()
    R, V = x.shape
    lp, ent = torch.zeros(R, dtype=torch.float64), torch.zeros(R, dtype=torch.float64)
    tv = torch.full((R, top), -INF, dtype=torch.float64)
    ti = torch.full((R, top), -1)
    for r in range(R):
        t = None if targets is None else int(targets[r])
        if t == ignore:
            continue
        row = x[r]
        empty = bool((row == -INF).all())
        # about the maximum: a row of a type's lowest value is uniform
        log_p = row if empty else (row - row.max()) - torch.logsumexp(row - row.max(), 0)
        p = log_p.exp()
        ent[r] = 0.0 if empty else -torch.where(p > 0, p * log_p, 0.0).sum()
        if bool(row.isnan().any()):
            ent[r] = math.nan
        if t is not None:
            lp[r] = log_p[t] if 0 <= t < V else math.nan
        order = torch.argsort(-row, dim=0, stable=True)[:top]
        tv[r], ti[r] = log_p[order], order
    return lp, ent, tv, ti


def _close(got, want, tol, what):
    got = got.detach().double().cpu()
    assert torch.equal(got.isnan(), want.isnan()), f"{what}: NaN places"
    inf = want.isinf()
    assert torch.equal(got[inf], want[inf]) and torch.equal(got.isinf(), inf), f"{what}: infinities"
    fine = want.isfinite()
    tol = torch.as_tensor(tol, dtype=torch.float64).expand_as(want)[fine] + 1e-6 * want[fine].abs()
    err = (got[fine] - want[fine]).abs()
    assert bool((err <= tol).all()), f"{what}: worst {float((err / tol).max()):.3g} of the tolerance"


def _check(x, targets, top, ignore=-100):
    r = myelin.token_log_probs(x, targets, top=top, ignore_index=ignore)
    V = x.shape[-1]
    rows = x.reshape(-1, V)
    lp, ent, tv, ti = _reference(rows, None if targets is None else targets.reshape(-1).cpu(), top, ignore)
    assert (r.log_probs is None) == (targets is None)
    if targets is not None:
        assert r.log_probs.shape == x.shape[:-1] and r.log_probs.dtype == torch.float32
        _close(r.log_probs.reshape(-1), lp, 1e-5, "log_probs")
    _close(r.entropy.reshape(-1), ent, 1e-5 * (1 + math.log(V)), "entropy")
    if top:
        assert r.top_tokens.dtype == torch.int64 and r.top_tokens.shape == (*x.shape[:-1], top)
        assert torch.equal(r.top_tokens.reshape(-1, top).cpu(), ti), "top_tokens"
        _close(r.top_log_probs.reshape(-1, top), tv, 1e-5, "top_log_probs")
    else:
        assert r.top_log_probs is None and r.top_tokens is None
    return r


SIZES = [(1, 1), (3, 2), (7, 10), (300, 10), (5, 32), (5, 33), (9, 255), (4, 256), (2, 1000), (3, 1024), (3, 1025),
         (2, 4095), (2, 4096), (1, 4097), (3, 9001), (1, 70001), (600, 1500)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("R,V", SIZES)
def test_values_at_many_sizes(R, V, dtype):
    _case(test="log_probs_values", R=R, V=V, dtype=dtype)
    x, g = _logits(R, V, dtype)
    targets = torch.randint(0, V, (R,), generator=g).to(DEV)
    for top in sorted({0, 1, min(V, 5), min(V, 64)}):
        _check(x, targets, top)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("V", [10, 700, 5000, 20001])
def test_masked_logits_and_rows(V, dtype):
    _case(test="log_probs_masked", V=V, dtype=dtype)
    x, g = _logits(9, V, dtype)
    low = torch.finfo(x.dtype).min
    x[0, torch.arange(V) % 3 != 1] = -INF
    x[1, torch.arange(V) % 3 != 1] = low
    x[2] = -INF
    x[3] = low
    x[4, 1:] = -INF  # one token
    x[5, :-1] = -INF
    x[6] = 0.0
    targets = torch.randint(0, V // 3, (9,), generator=g) * 3 + 1
    targets[4], targets[5], targets[7] = 0, V - 1, -100
    targets = targets.to(DEV)
    for top in (0, 1, 7):
        _check(x, targets, top)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("V", [20, 3000])
def test_nan_and_infinity_stay_in_their_rows(V, dtype):
    _case(test="log_probs_nan", V=V, dtype=dtype)
    x, _ = _logits(4, V, dtype)
    x[1, V // 2] = math.nan
    x[2, V - 1] = INF
    targets = torch.tensor([0, 0, 0, 0], device=DEV)
    r = myelin.token_log_probs(x, targets)
    assert r.log_probs.isnan().tolist() == [False, True, True, False]
    assert r.entropy.isnan().tolist() == [False, True, True, False]
    _check(x[[0, 3]], targets[:2], 0)


@pytest.mark.parametrize("V", [10, 3000])
def test_large_offsets_lose_nothing(V):
    """Rows shifted by a large exact constant have the unshifted results: every
    shifted logit is exact, so only lse's own rounding (|lse| 2^-24) remains."""

    _case(test="log_probs_shift", V=V)
    x, g = _logits(4, V, "bf16")
    x = (x.float() * 64).round() / 64  # multiples of 1/64 below 64
    targets = torch.randint(0, V, (4,), generator=g).to(DEV)
    a, b = myelin.token_log_probs(x, targets), myelin.token_log_probs(x + 4096.0, targets)
    assert float((a.entropy - b.entropy).abs().max()) <= 1e-5 * (1 + math.log(V))
    assert float((a.log_probs - b.log_probs).abs().max()) <= 1e-5 + 4200 * 2**-23


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("R,V", [(3, 6000), (2, 1500), (600, 1100), (1, 50000)])
def test_ties_go_to_the_lowest_index(R, V, dtype):
    _case(test="log_probs_ties", R=R, V=V, dtype=dtype)
    g = torch.Generator().manual_seed(V)
    x = torch.randint(0, 4, (R, V), generator=g).to(DTYPES[dtype]).to(DEV)
    _check(x, None, 64)
    x.zero_()
    x[:, ::2] = -0.0  # equal to +0
    _check(x, None, 20)
    # the largest last, so that every tile brings better ones
    x.copy_(torch.arange(V, device=DEV).expand(R, V) if dtype == "fp32" else (torch.arange(V, device=DEV) // 200))
    _check(x / (1 + V // 64), None, 33)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("V", [11, 1031, 4200])
def test_layouts(V, dtype):
    """Rows that start anywhere, leading dimensions, transposed and expanded
    storage, narrow target types."""

    _case(test="log_probs_layouts", V=V, dtype=dtype)
    wide, g = _logits(6, 2 * V + 3, dtype)
    targets = torch.randint(0, V, (6,), generator=g).to(DEV)
    for shift in (0, 1, 2, 3):
        _check(wide[:, shift : shift + V], targets, 3)
    _check(wide[::2, V : 2 * V], targets[::2], 3)
    _check(wide[:, :V].t().contiguous().t(), targets.int(), 2)
    _check(wide[:, :V].view(2, 3, -1) if wide[:, :V].is_contiguous() else wide[:, :V].reshape(2, 3, V),
           targets.view(2, 3), 2)
    cut = wide.view(2, 3, -1)[:, 1:, 1 : V + 1]  # rows with no common stride
    _check(cut, targets.view(2, 3)[:, 1:], 2)
    _check(wide[:1, :V].expand(6, V), targets, 2)
    _check(wide[0, :V], targets[0], 1)


def test_no_rows():
    x = torch.empty(0, 17, device=DEV)
    r = myelin.token_log_probs(x, torch.empty(0, dtype=torch.int64, device=DEV), top=3)
    assert r.log_probs.shape == (0,) and r.top_tokens.shape == (0, 3)


@pytest.mark.parametrize("V", [10, 2000])
def test_targets_out_of_range_are_nan_and_read_nothing(V):
    _case(test="log_probs_bad_targets", V=V)
    x, _ = _logits(5, V, "fp32")
    x.requires_grad_()
    targets = torch.tensor([0, -1, V, 2**40, -100], device=DEV)
    r = myelin.token_log_probs(x, targets)
    assert r.log_probs.isnan().tolist() == [False, True, True, True, False]
    assert bool(r.entropy.isfinite().all())
    (g,) = torch.autograd.grad(r.log_probs.sum(), x)
    assert bool(g[[0, 4]].isfinite().all()) and bool(g[[1, 2, 3]].isnan().all())


def _grad_reference(x, targets, g_lp, g_ent, ignore=-100):
    x = x.detach().double().cpu()
    out = torch.zeros_like(x)
    for r in range(x.shape[0]):
        if int(targets[r]) == ignore or bool((x[r] == -INF).all()):
            continue
        log_p = x[r] - torch.logsumexp(x[r], 0)
        p = log_p.exp()
        each = torch.where(p > 0, p * log_p, 0.0)
        hit = torch.zeros_like(p)
        hit[int(targets[r])] = 1.0
        out[r] = float(g_lp[r]) * (hit - p) - float(g_ent[r]) * (each - p * each.sum())
    return out


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("R,V", [(1, 1), (7, 10), (300, 10), (5, 255), (3, 256), (4, 1000), (2, 4096), (3, 4104),
                                 (2, 9001)])
def test_gradient_is_the_formula(R, V, dtype):
    _case(test="log_probs_grad", R=R, V=V, dtype=dtype)
    x, g = _logits(R, V, dtype)
    if R > 2 and V > 1:
        x[1, ::2] = -INF
        x[2] = -INF
    x.requires_grad_()
    targets = torch.randint(0, V, (R,), generator=g)
    if R > 3:
        targets[3] = -100
    g_lp, g_ent = torch.randn(R, generator=g), torch.randn(R, generator=g)
    want = {"both": _grad_reference(x, targets, g_lp, g_ent),
            "log_probs": _grad_reference(x, targets, g_lp, 0 * g_ent),
            "entropy": _grad_reference(x, targets, 0 * g_lp, g_ent)}
    r = myelin.token_log_probs(x, targets.to(DEV), top=min(V, 2))
    for which, outs, gs in (("both", (r.log_probs, r.entropy), (g_lp, g_ent)), ("log_probs", (r.log_probs,), (g_lp,)),
                            ("entropy", (r.entropy,), (g_ent,))):
        (got,) = torch.autograd.grad(outs, x, tuple(t.to(DEV) for t in gs), retain_graph=True)
        assert got.dtype == x.dtype and got.shape == x.shape
        tol = (3e-5 * (g_lp.abs() + g_ent.abs() * (1 + math.log(V)))).double()[:, None]
        tol = tol + (2.0**-8 if dtype == "bf16" else 0.0) * want[which].abs()
        err = (got.double().cpu() - want[which]).abs()
        assert bool((err <= tol).all()), f"{which}: worst {float((err / tol).max()):.3g} of the tolerance"


@pytest.mark.parametrize("V", [10, 3001])
def test_gradient_is_the_difference_quotient(V):
    """Along random directions of unit entries, step 2^-6: the truncation is of
    order h^2 / 6 times a third derivative of order 1 a row, the rounding 2e-5 / h
    a row: 2e-3 a row in all."""

    _case(test="log_probs_difference", V=V)
    R, h = 4, 2.0**-6
    x, g = _logits(R, V, "fp32", spread=1.0)
    targets = torch.randint(0, V, (R,), generator=g).to(DEV)
    wide = torch.zeros(R, 2 * V, device=DEV)
    wide[:, 1 : V + 1] = x
    leaf = wide.requires_grad_()
    r = myelin.token_log_probs(leaf[:, 1 : V + 1], targets)
    (grad,) = torch.autograd.grad(r.log_probs.sum() + 0.5 * r.entropy.sum(), leaf)
    assert bool((grad[:, 0] == 0).all()) and bool((grad[:, V + 1 :] == 0).all())
    for seed in range(3):
        d = torch.randn(R, V, generator=torch.Generator().manual_seed(seed)).sign().to(DEV)

        def f(y):
            q = myelin.token_log_probs(y, targets)
            return float(q.log_probs.double().sum() + 0.5 * q.entropy.double().sum())

        slope = (f(x + h * d) - f(x - h * d)) / (2 * h)
        assert abs(slope - float((grad[:, 1 : V + 1].double() * d).sum())) <= 2e-3 * R


def test_second_derivatives_are_refused():
    x, _ = _logits(2, 10, "fp32")
    x.requires_grad_()
    r = myelin.token_log_probs(x, torch.tensor([1, 2], device=DEV))
    (g,) = torch.autograd.grad(r.log_probs.sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(g.sum(), x)


def test_refusals():
    x = torch.zeros(2, 10, device=DEV)
    t = torch.zeros(2, dtype=torch.int64, device=DEV)
    for bad, message in ((lambda: myelin.token_log_probs(x.half(), t), "float32 or bfloat16"),
                         (lambda: myelin.token_log_probs(x, t[:1]), "must match"),
                         (lambda: myelin.token_log_probs(x, t.float()), "int64 or int32"),
                         (lambda: myelin.token_log_probs(x, t.cpu()), "same device"),
                         (lambda: myelin.token_log_probs(x, t, top=11), "top must be"),
                         (lambda: myelin.token_log_probs(x, t, top=-1), "top must be"),
                         (lambda: myelin.token_log_probs(torch.zeros(3, 100, device=DEV), top=65), "top must be"),
                         (lambda: myelin.token_log_probs(x[:, :0], t), "V > 0")):
        with pytest.raises(ValueError, match=message):
            bad()


def test_other_stream_and_graph_replays():
    _case(test="log_probs_graph")
    x, g = _logits(3, 9001, "bf16")
    targets = torch.randint(0, 9001, (3,), generator=g).to(DEV)
    x.requires_grad_()

    def body():
        r = myelin.token_log_probs(x, targets)
        s = myelin.token_log_probs(x.detach(), targets, top=9)
        (gx,) = torch.autograd.grad((r.log_probs, r.entropy), x, (r.log_probs.detach(), r.entropy.detach()))
        return r.log_probs.detach(), r.entropy.detach(), s.top_log_probs, s.top_tokens, gx

    eager = [t.clone() for t in body()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            again = body()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    for a, b in zip(again, eager):
        assert torch.equal(a, b)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = body()
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(held, eager):
            assert torch.equal(a, b)
        _ = float((x.detach().float() * 2.0).sum())


@pytest.mark.parametrize("V", [62, 300])
def test_more_rows_than_one_launch_dimension(V):
    """Over 2^32 threads: rows past the first 2^32 / V are the same rows as alone."""

    R = (2**32 if V < 256 else 2**32 // 256 * V) // V + 5
    _case(test="log_probs_rows", R=R, V=V)
    x = torch.zeros(R, V, dtype=torch.bfloat16, device=DEV)
    rows = torch.tensor([0, 1, R // 2, R - 6, R - 5, R - 1], device=DEV)
    x[rows] = _logits(len(rows), V, "bf16")[0]
    targets = torch.zeros(R, dtype=torch.int64, device=DEV)
    targets[rows] = torch.arange(len(rows), device=DEV) * 7
    few = x[rows].clone().requires_grad_()
    want = myelin.token_log_probs(few, targets[rows])
    x.requires_grad_()
    got = myelin.token_log_probs(x, targets)
    (g,) = torch.autograd.grad(got[0].sum() + got[1].sum(), x)
    (w,) = torch.autograd.grad(want[0].sum() + want[1].sum(), few)
    for a, b in zip(got[:2], want[:2]):
        a = a.detach().abs()
        assert torch.equal(a[rows], b.abs())
        a[rows] = math.log(V)
        # every other row is uniform: log V, of terms that are exact but for its rounding
        assert bool(((a - math.log(V)).abs() < 1e-5 + 1e-6 * math.log(V)).all())
    assert torch.equal(g[rows], w)
