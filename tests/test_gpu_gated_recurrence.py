"""gated_recurrence and its step against the recurrence and its adjoint in float64,
one step after the other.

Tolerances are majorants of fp32's errors, formed beside the reference.  With e =
2^-24: a gate's two values carry at most 8 e (the exponential within 2 units in the
last place, one sum, a reciprocal within 1, one product, one difference), and each step adds its own
roundings and, where steps are joined in another order, those of the products of
decays: BASE = 16 e of the sum of absolute terms, carried on as the state is.  The
kernels of bfloat16 leave the rounding of the exponential's argument, |gate| e more.
An exponential below the least normal number is 0, so that a gate's smaller value is
within TINY = 2^-126 besides, times what it multiplies.  A result in bfloat16 adds
half a unit in its last place.
"""

from __future__ import annotations

import math

import pytest
import torch

import myelin_amd as myelin

pytestmark = pytest.mark.gpu
DEV = "cuda"
DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16}
BASE = 16 * 2.0**-24
TINY = 2.0**-126


def _case(**kw):
    print("case:", " ".join(f"{k}={v}" for k, v in kw.items()), flush=True)


def _half(dt):
    return torch.finfo(dt).eps / 2 if dt == torch.bfloat16 else 2.0**-24


def _reference(x, gate, state, lengths, g_out=None, g_state=None):
    """Values and, beside each, the bound of its fp32 error."""

    C = BASE if x.dtype == torch.float32 else BASE + gate.detach().double().cpu().abs().clamp(max=200.0) * 2.0**-24
    x, gate = x.detach().double().cpu(), gate.detach().double().cpu()
    T, B, N = x.shape
    C = torch.as_tensor(C, dtype=torch.float64).expand(T, B, N)
    live = torch.full((B, 1), T) if lengths is None else lengths.cpu().long().clamp(0, T)[:, None]
    a, b = torch.sigmoid(gate), torch.sigmoid(-gate)
    on = torch.arange(T)[:, None, None] < live
    a, b, x = torch.where(on, a, 1.0), torch.where(on, b, 0.0), torch.where(on, x, 0.0)
    h = torch.zeros(B, N, dtype=torch.float64) if state is None else state.detach().double().cpu()
    size, err = h.abs(), torch.zeros_like(h)
    hs, before, errs, sizes, errs_before = [], [], [], [], []
    for t in range(T):
        before.append(h)
        sizes.append(size)
        errs_before.append(err)
        h = a[t] * h + b[t] * x[t]
        tiny = TINY * (size + x[t].abs())
        size = a[t] * size + b[t] * x[t].abs()
        err = a[t] * err + torch.where(on[t], C[t] * size + tiny, 0.0)
        hs.append(h)
        errs.append(err)
    out = torch.where(on, torch.stack(hs), 0.0)
    r = {"state": (h, err), "out": (out, torch.where(on, torch.stack(errs), 0.0))}
    if g_out is None and g_state is None:
        return r
    zero = torch.zeros(B, N, dtype=torch.float64)
    g = zero if g_state is None else g_state.double().cpu()
    go = torch.zeros_like(x) if g_out is None else torch.where(on, g_out.double().cpu(), 0.0)
    size, err = g.abs(), zero
    gx, gg, ex, eg = ([None] * T for _ in range(4))
    for t in range(T - 1, -1, -1):
        g, size = g + go[t], size + go[t].abs()
        err = err + torch.where(on[t], C[t] * size + TINY * size, 0.0)
        d, dsize = before[t] - x[t], sizes[t] + x[t].abs()
        gx[t], ex[t] = b[t] * g, b[t] * (err + C[t] * size) + TINY * size
        gg[t] = b[t] * a[t] * g * d
        eg[t] = b[t] * a[t] * (err * dsize + size * (errs_before[t] + C[t] * dsize)) + TINY * size * dsize
        g, size, err = a[t] * g, a[t] * size, a[t] * err
    r["x"], r["gate"] = (torch.stack(gx), torch.stack(ex)), (torch.stack(gg), torch.stack(eg))
    r["initial"] = (g, err + C[0] * size)
    return r


def _close(got, want, what):
    value, bound = want
    dt = got.dtype
    got = got.detach().double().cpu()
    bound = bound + _half(dt) * (value.abs() + bound) + 1e-37
    bad = (got - value).abs() > bound
    worst = float(((got - value).abs() / bound).max()) if bad.numel() else 0.0
    assert not bool(bad.any()), f"{what}: {int(bad.sum())} elements, worst {worst:.2f} of the bound"


def _inputs(T, B, N, dtype, seed=0, tau=(1.5, 300.0)):
    g = torch.Generator().manual_seed(seed + 7 * T + 3 * B + N)
    x = torch.randn(T, B, N, generator=g)
    taus = torch.logspace(math.log2(tau[0]), math.log2(tau[1]), N, base=2.0)
    gate = torch.randn(T, B, N, generator=g) + torch.log(taus - 1.0)
    state = torch.randn(B, N, generator=g)
    return x.to(DTYPES[dtype]).to(DEV), gate.to(DTYPES[dtype]).to(DEV), state.to(DEV)


def _run(x, gate, state, lengths, g_out, g_state):
    leaves = [t.detach().clone().requires_grad_() for t in (x, gate)]
    s = None if state is None else state.detach().clone().requires_grad_()
    final, out = myelin.gated_recurrence(*leaves, s, lengths=lengths)
    wrt = leaves + ([] if s is None else [s])
    pairs = [(o, g) for o, g in ((out, g_out), (final, g_state)) if g is not None]
    grads = torch.autograd.grad([o for o, _ in pairs], wrt, [g for _, g in pairs])
    return final, out, dict(zip(("x", "gate", "initial"), grads))


SIZES = [(1, 1, 1), (1, 3, 5), (2, 1, 64), (15, 2, 3), (16, 1, 65), (17, 5, 33), (100, 4, 128), (255, 1, 7),
         (256, 2, 64), (257, 3, 130), (513, 1, 192), (700, 2, 31), (1025, 9, 63), (33, 300, 40), (3, 1, 5000)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,B,N", SIZES)
def test_sequences_and_gradients(T, B, N, dtype):
    _case(test="recurrence", T=T, B=B, N=N, dtype=dtype)
    x, gate, state = _inputs(T, B, N, dtype)
    g = torch.Generator().manual_seed(T + B + N)
    g_out = torch.randn(T, B, N, generator=g).to(x.dtype).to(DEV)
    g_state = torch.randn(B, N, generator=g).to(DEV)
    lengths = torch.randint(0, T + 1, (B,), generator=g)
    lengths[0] = T
    if B > 2:
        lengths[1], lengths[2] = 0, 1
    for s, ls in ((None, None), (state, lengths.to(DEV)), (state, lengths.int().to(DEV))):
        want = _reference(x, gate, s, ls, g_out, g_state)
        with torch.no_grad():
            final, out = myelin.gated_recurrence(x, gate, s, lengths=ls)
        assert final.dtype == torch.float32 and out.dtype == x.dtype and out.shape == x.shape
        _close(final, want["state"], "state")
        _close(out, want["out"], "out")
        final2, out2, grads = _run(x, gate, s, ls, g_out, g_state)
        assert torch.equal(final, final2.detach()) and torch.equal(out, out2.detach())
        for name, t in grads.items():
            assert t.dtype == (torch.float32 if name == "initial" else x.dtype)
            _close(t, want[name], f"gradient of {name}")


@pytest.mark.parametrize("T,B,N", [(5000, 1, 40), (9000, 2, 3), (4096, 1, 64), (40000, 1, 2)])
def test_long_sequences_of_few_channels(T, B, N):
    """Time is split over the chip."""

    for dtype in DTYPES:
        _case(test="recurrence_long", T=T, B=B, N=N, dtype=dtype)
        x, gate, state = _inputs(T, B, N, dtype, tau=(2.0, 2000.0))
        g = torch.Generator().manual_seed(T)
        g_out = torch.randn(T, B, N, generator=g).to(x.dtype).to(DEV)
        g_state = torch.randn(B, N, generator=g).to(DEV)
        lengths = torch.tensor([T - 777] + [13] * (B - 1)).to(DEV)
        for ls in (None, lengths):
            want = _reference(x, gate, state, ls, g_out, g_state)
            final, out, grads = _run(x, gate, state, ls, g_out, g_state)
            _close(final, want["state"], "state")
            _close(out, want["out"], "out")
            for name, t in grads.items():
                _close(t, want[name], f"gradient of {name}")


@pytest.mark.parametrize("which", ["out", "state"])
def test_one_gradient_alone(which):
    x, gate, state = _inputs(70, 3, 20, "fp32")
    g_out = torch.randn_like(x) if which == "out" else None
    g_state = torch.randn_like(state) if which == "state" else None
    want = _reference(x, gate, state, None, g_out, g_state)
    _, _, grads = _run(x, gate, state, None, g_out, g_state)
    for name, t in grads.items():
        _close(t, want[name], name)
    # one leaf alone
    leaves = {"x": x, "gate": gate, "initial": state}
    for name in leaves:
        args = [t.clone().requires_grad_(n == name) for n, t in leaves.items()]
        final, out = myelin.gated_recurrence(*args)
        root, g = (out, g_out) if which == "out" else (final, g_state)
        (t,) = torch.autograd.grad(root, args[list(leaves).index(name)], g)
        assert torch.equal(t, grads[name])


def test_gradients_are_the_differences_of_the_definition():
    """Along random directions, by central differences of the float64 definition:
    their own error, step^2 / 6 of a third derivative below the sum of absolute
    terms, is at most 1e-7 of it."""

    x, gate, state = _inputs(60, 2, 9, "fp32")
    g = torch.Generator().manual_seed(3)
    g_out, g_state = torch.randn(60, 2, 9, generator=g), torch.randn(2, 9, generator=g)
    want = _reference(x, gate, state, None, g_out, g_state)
    _, _, grads = _run(x, gate, state, None, g_out.to(DEV), g_state.to(DEV))
    leaves = [t.double().cpu() for t in (x, gate, state)]

    def value(args):
        r = _reference(*args, None)
        return float((r["out"][0] * g_out).sum() + (r["state"][0] * g_state).sum())

    step = 1e-4
    for i, name in enumerate(("x", "gate", "initial")):
        d = torch.randn(leaves[i].shape, generator=g, dtype=torch.float64)
        up, down = ([t + s * step * d if j == i else t for j, t in enumerate(leaves)] for s in (1, -1))
        slope = (value(up) - value(down)) / (2 * step)
        got = float((grads[name].double().cpu() * d).sum())
        v, bound = want[name]
        room = float(((bound + 2.0**-24 * v.abs()) * d.abs()).sum()) + 1e-6 * float((v * d).abs().sum())
        assert abs(got - slope) <= room, name


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,N", [(1, 1), (1, 64), (3, 5), (2, 1031), (256, 512), (7, 4098)])
def test_steps_continue_a_sequence(B, N, dtype):
    _case(test="recurrence_step", B=B, N=N, dtype=dtype)
    x, gate, state = _inputs(4, B, N, dtype)
    want = _reference(x, gate, state, None)
    s, mine = state, state.clone()
    for t in range(4):
        s, out = myelin.gated_recurrence_step(x[t], gate[t], s)
        same, out2 = myelin.gated_recurrence_step(x[t], gate[t], mine, out_state=mine)
        assert same is mine and torch.equal(s, mine) and torch.equal(out, out2) and out.dtype == x.dtype
        _close(out, (want["out"][0][t], want["out"][1][t]), "out")
    _close(s, want["state"], "state")
    # and a sequence continues the steps
    final, out = myelin.gated_recurrence(x, gate, s)
    again = _reference(x, gate, s, None)
    _close(final, again["state"], "state")


@pytest.mark.parametrize("dtype", DTYPES)
def test_layouts_are_read_in_place(dtype):
    """Halves of one projection, batch-major inputs, odd offsets, expanded rows."""

    T, B, N = 37, 3, 24
    g = torch.Generator().manual_seed(1)
    whole = torch.randn(T, B, 2 * N + 3, generator=g).to(DTYPES[dtype]).to(DEV)
    swapped = torch.randn(B, T, 2 * N, generator=g).to(DTYPES[dtype]).to(DEV).transpose(0, 1)
    row = torch.randn(1, 1, N, generator=g).to(DTYPES[dtype]).to(DEV)
    flat = torch.randn(T, N, B, generator=g).to(DTYPES[dtype]).to(DEV).transpose(1, 2)
    pairs = [(whole[..., :N], whole[..., N : 2 * N]), (whole[..., 1 : N + 1], whole[..., N + 3 :]),
             (swapped[..., :N], swapped[..., N:]), (row.expand(T, B, N), whole[..., :N]), (flat, row.expand(T, B, N))]
    g_out = torch.randn(B, T, N, generator=g).to(DTYPES[dtype]).to(DEV).transpose(0, 1)
    for i, (x, gate) in enumerate(pairs):
        _case(test="recurrence_layout", dtype=dtype, pair=i)
        a = myelin.gated_recurrence(x, gate)
        b = myelin.gated_recurrence(x.contiguous(), gate.contiguous())
        assert all(torch.equal(u, v) for u, v in zip(a, b))
        first = _run(x, gate, None, None, g_out, None)[2]
        xs, gs = x.detach().requires_grad_(), gate.detach().requires_grad_()
        second = torch.autograd.grad(myelin.gated_recurrence(xs, gs)[1], (xs, gs), g_out)
        assert all(torch.equal(u, v) for u, v in zip(first.values(), second))
        s = torch.randn(B, N, device=DEV)
        u, v = myelin.gated_recurrence_step(x[3], gate[3], s), myelin.gated_recurrence_step(
            x[3].contiguous(), gate[3].contiguous(), s)
        assert all(torch.equal(p, q) for p, q in zip(u, v))
    # a broadcast input's gradient is the sum over what it was read for
    r = row.detach().clone().requires_grad_()
    out = myelin.gated_recurrence(r.expand(T, B, N), whole[..., :N])[1]
    (gr,) = torch.autograd.grad(out, r, g_out)
    full = _run(row.expand(T, B, N), whole[..., :N], None, None, g_out, None)[2]["x"]
    want = full.double().sum((0, 1), keepdim=True)
    room = (T * B * _half(full.dtype) + _half(full.dtype)) * full.double().abs().sum((0, 1), keepdim=True)
    assert bool(((gr.double() - want).abs() <= room).all())


def test_an_expanded_gradient():
    x, gate, _ = _inputs(40, 2, 17, "fp32")
    xs = x.clone().requires_grad_()
    (a,) = torch.autograd.grad(myelin.gated_recurrence(xs, gate)[1].sum(), xs)
    (b,) = torch.autograd.grad(myelin.gated_recurrence(xs, gate)[1], xs, torch.ones_like(x))
    assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", DTYPES)
def test_gates_at_their_ends(dtype):
    """Gates of +-inf hold and replace exactly; far ones keep their accuracy."""

    T, N = 50, 8
    x = torch.randn(T, 1, N, device=DEV).to(DTYPES[dtype])
    gate = torch.full((T, 1, N), math.inf, device=DEV).to(DTYPES[dtype])
    s = torch.randn(1, N, device=DEV)
    final, out = myelin.gated_recurrence(x, gate, s)
    assert torch.equal(final, s) and torch.equal(out, s.to(x.dtype).expand(T, 1, N))
    final, out = myelin.gated_recurrence(x, -gate, s)
    assert torch.equal(out, x) and torch.equal(final, x[-1].float())
    leaf = x.clone().requires_grad_()
    (gx,) = torch.autograd.grad(myelin.gated_recurrence(leaf, -gate, s)[1], leaf, torch.ones_like(x))
    assert torch.equal(gx, torch.ones_like(x))
    for far in (-100.0, -30.0, 20.0, 88.0, 100.0):
        g = torch.full((T, 1, N), far, device=DEV).to(DTYPES[dtype])
        ones = torch.ones_like(x)
        want = _reference(x, g, s, None, ones, None)
        f, o, grads = _run(x, g, s, None, ones, None)
        _close(f, want["state"], far)
        _close(o, want["out"], far)
        for name, t in grads.items():
            _close(t, want[name], (far, name))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("value", [math.inf, -math.inf, math.nan])
@pytest.mark.parametrize("T,N", [(60, 5), (900, 70), (6000, 3)])
def test_what_is_not_finite_stays_in_its_steps(T, N, value, dtype):
    _case(test="recurrence_not_finite", T=T, N=N, value=value, dtype=dtype)
    x, gate, s = _inputs(T, 2, N, dtype)
    at, lengths = T // 2 + 3, torch.tensor([T, T // 2], device=DEV)
    g_out = torch.randn_like(x)
    clean = _run(x, gate, s, lengths, g_out, None)
    bad = x.clone()
    bad[at, :, 1] = value  # past the second sample's end
    final, out, grads = _run(bad, gate, s, lengths, g_out, None)
    hit = torch.zeros_like(x, dtype=torch.bool)
    hit[at:, 0, 1] = True
    assert torch.equal(out[~hit], clean[1][~hit]) and not bool(out[hit].isfinite().any())
    assert not bool(final[0, 1].isfinite()) and torch.equal(final[1], clean[0][1])
    assert torch.equal(grads["x"], clean[2]["x"])
    assert torch.equal(grads["gate"][~hit], clean[2]["gate"][~hit]) and not bool(grads["gate"][hit].isfinite().any())
    bad = g_out.clone()
    bad[at, :, 1] = value
    _, _, grads = _run(x, gate, s, lengths, bad, None)
    hit = torch.zeros_like(hit)
    hit[: at + 1, 0, 1] = True
    assert torch.equal(grads["x"][~hit], clean[2]["x"][~hit])
    assert not bool(grads["x"][at, 0, 1].isfinite()) and not bool(grads["x"][at - 1, 0, 1].isfinite())


def test_nothing_past_the_end_is_read_or_kept():
    """NaN behind every sample's end."""

    T, B, N = 300, 4, 33
    for dtype in DTYPES:
        x, gate, s = _inputs(T, B, N, dtype)
        lengths = torch.tensor([0, 1, 299, 300], device=DEV)
        past = torch.arange(T, device=DEV)[:, None, None] >= lengths[:, None]
        g_out = torch.randn_like(x)
        want = _run(x, gate, s, lengths, g_out, None)
        x, gate, g_out = (torch.where(past, math.nan, t) for t in (x, gate, g_out))
        got = _run(x, gate, s, lengths, g_out, None)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
        assert bool((got[1][past.expand_as(x)] == 0).all())
        for name in want[2]:
            assert torch.equal(got[2][name], want[2][name])
        # out of [0, T]
        a = myelin.gated_recurrence(x, gate, s, lengths=torch.tensor([-5, 1, 299, 300], device=DEV))
        assert torch.equal(a[1], want[1])
        b = myelin.gated_recurrence(x[..., :0], gate[..., :0], s[..., :0], lengths=lengths)
        assert b[0].shape == (B, 0) and b[1].shape == (T, B, 0)


def test_offsets_past_32_bits():
    T, N = 2100, 2**20
    _case(test="recurrence_large")
    g = torch.Generator(device=DEV).manual_seed(0)
    x = torch.empty(T, 1, N, dtype=torch.bfloat16, device=DEV).normal_(generator=g)
    gate = torch.empty_like(x).normal_(generator=g)
    final, out = myelin.gated_recurrence(x, gate)
    some = torch.tensor([0, 1, 77777, N - 1], device=DEV)
    want = _reference(x[..., some], gate[..., some], None, None)
    _close(out[..., some], want["out"], "out")
    _close(final[..., some], want["state"], "state")


def test_refusals():
    x = torch.zeros(4, 2, 3, device=DEV)
    s = torch.zeros(2, 3, device=DEV)
    f, one = myelin.gated_recurrence, myelin.gated_recurrence_step
    n = torch.zeros(2, dtype=torch.int32, device=DEV)
    for bad, message in ((lambda: f(x[0], x[0]), "must be shaped"), (lambda: f(x, x[:, :, :2]), "gate must have"),
                         (lambda: f(x, x.bfloat16()), "gate must have"), (lambda: f(x.half(), x.half()), "float32 or"),
                         (lambda: f(x[:0], x[:0]), "at least one"), (lambda: f(x, x, s[:1]), "initial_state must be"),
                         (lambda: f(x, x, s.bfloat16()), "initial_state must be"),
                         (lambda: f(x, x, s.cpu()), "initial_state must be"),
                         (lambda: f(x, x, lengths=n[:1]), "lengths must be"),
                         (lambda: f(x, x, lengths=n.cpu()), "lengths must be"),
                         (lambda: f(x, x, lengths=n.float()), "lengths must be"),
                         (lambda: one(x, x, s), "must be shaped"), (lambda: one(x[0], x[0], s[0]), "state must be"),
                         (lambda: one(x[0], x[0], s.clone().requires_grad_()), "no gradient"),
                         (lambda: one(x[0], x[0], s, out_state=s.t().contiguous().t()), "contiguous"),
                         (lambda: one(x[0], x[0], s, out_state=s[:1]), "out_state must be"),
                         (lambda: one(x[0], x[0], s, out_state=s.clone().requires_grad_()), "written in place"),
                         (lambda: myelin.GatedRecurrence(3, 4, taus=(0.5, 2.0)), "taus must be"),
                         (lambda: myelin.GatedRecurrence(3, 4, taus=(8.0, 2.0)), "taus must be")):
        with pytest.raises(ValueError, match=message):
            bad()
    base = torch.zeros(9, device=DEV)
    with pytest.raises(ValueError, match="overlap"):
        one(x[0], x[0], base[:6].view(2, 3), out_state=base[2:8].view(2, 3))


def test_a_state_advanced_in_place_is_noticed():
    x, gate, s = _inputs(5, 2, 6, "fp32")
    xs = x.clone().requires_grad_()
    state = torch.ones(2, 6, device=DEV)
    w = torch.ones(2, 6, device=DEV, requires_grad=True)
    y = (w * state).sum()
    myelin.gated_recurrence_step(x[0], gate[0], state, out_state=state)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()
    final, out = myelin.gated_recurrence(xs, gate, s)
    out.sum().backward()
    assert xs.grad is not None


def test_module():
    _case(test="recurrence_module")
    torch.manual_seed(0)
    m = myelin.GatedRecurrence(12, 20, taus=(4.0, 64.0)).to(DEV)
    taus = 1.0 / (1.0 - torch.sigmoid(m.synapse.bias[20:].detach().double()))
    assert abs(float(taus[0]) - 4.0) < 1e-4 and abs(float(taus[-1]) - 64.0) < 1e-2
    x = torch.randn(30, 3, 12, device=DEV)
    lengths = torch.tensor([30, 7, 0], device=DEV)
    final, out = m(x, lengths=lengths)
    both = m.synapse(x)
    want = myelin.gated_recurrence(both[..., :20].contiguous(), both[..., 20:].contiguous(), lengths=lengths)
    assert torch.equal(final, want[0]) and torch.equal(out, want[1])
    out.square().sum().backward()
    assert all(p.grad is not None and bool(p.grad.isfinite().all()) for p in m.parameters())
    with torch.no_grad():
        whole, _ = m(x)
        s = torch.zeros(3, 20, device=DEV)
        for t in range(30):
            s, y = m.step(x[t], s, out_state=s)
    # (the projection of 3 rows and of 90 may differ in its sums' last bits)
    assert float((s - whole).abs().max()) <= 1e-5


def test_a_state_that_overlaps_the_inputs_is_refused():
    """Its elements would be written while others still read them as inputs."""

    base = torch.zeros(16, device=DEV)
    x, free, s = base[:6].view(2, 3), base[6:12].view(2, 3), torch.zeros(2, 3, device=DEV)
    other = torch.zeros(2, 3, device=DEV)
    for a, b, name in ((x, other, "x"), (other, x, "gate"), (base[:10].view(2, 5)[:, :3], other, "x")):
        with pytest.raises(ValueError, match=f"must not overlap {name}"):
            myelin.gated_recurrence_step(a, b, s, out_state=base[4:10].view(2, 3))
    new, out = myelin.gated_recurrence_step(x, other, s + 1, out_state=free)  # beside them
    assert torch.equal(free, out) and torch.equal(new, free) and torch.equal(free, torch.full_like(s, 0.5))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,B,N", [(150, 301, 64), (129, 5, 3301), (75, 150, 257), (50, 33, 2200), (41, 5, 27001)])
def test_workgroups_that_share_a_cu(T, B, N, dtype):
    """With more channels than the CUs have workgroups for at once, fewer waves to
    each go over several tiles."""

    test_sequences_and_gradients(T, B, N, dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,B,N", [(1, 3, 50001), (16, 70, 1999), (33, 131100, 1), (64, 33, 4003), (65, 33, 4003)])
def test_few_steps_of_many_channels(T, B, N, dtype):
    """A wave to 64 channels, up to 64 steps; the last workgroup has waves without any."""

    test_sequences_and_gradients(T, B, N, dtype)
