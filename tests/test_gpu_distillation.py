"""distillation_loss and its gradient against the definition in float64.

With e = 2^-24 and V logits a row: the sum of exponentials is within (V / 64 + 64) e
of itself by its additions (a lane's own, then pairs), and each exponential within
(4 + 2 |d|) e by its own error and its argument's rounding, d = (x - m) /
temperature; that is |d| <= 2^7 where it counts.  So log s carries at most S = (V /
64 + 64 + 260) e; a log probability adds 4 e |log q|, and the loss is a sum of K
terms p (log p - log q), p within 300 e: K e + 300 e + ... of their absolute sum.
A gradient is g / temperature (q - p), p within 300 e of itself.  q = e^(d - log s)
takes the roundings of x - m, of 1 / temperature, of their product and of the
difference into its exponent, 4 |d| e, beside S: a temperature of 0.1 puts tokens at
|d| of some hundreds.  Below the least normal number 2^-126 it is 0.
"""

from __future__ import annotations

import math

import pytest
import torch

import myelin_amd as myelin

pytestmark = pytest.mark.gpu
DEV = "cuda"
DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16}
E = 2.0**-24


def _case(**kw):
    print("case:", " ".join(f"{k}={v}" for k, v in kw.items()), flush=True)


def _reference(x, values, tokens, temperature, g=None):
    """(loss, bound), and (gradient, bound) for row gradients g."""

    x, v = x.detach().double().cpu() / temperature, values.double().cpu() / temperature
    t = tokens.cpu().long()
    R, V = x.shape
    K = t.shape[1]
    there = (t != -1) & (v != -math.inf)
    v = torch.where(there, v, -math.inf)
    none = ~there.any(-1)
    p = torch.where(none[:, None], 0.0, torch.softmax(v, -1))
    nothing = (x == -math.inf).all(-1)
    log_q = torch.where(nothing[:, None], -math.inf, torch.log_softmax(x, -1))
    at = torch.where(there, t, 0).clamp(0, V - 1)
    lq = log_q.gather(-1, at)
    used = there & (p > 0)
    terms = torch.where(used, p * (torch.log(p) - lq), 0.0)
    sizes = torch.where(used, p * (torch.log(p).abs() + lq.abs() + 1.0), 0.0)
    bad = (there & ((t < 0) | (t >= V))).any(-1)
    loss = torch.where(bad, math.nan, terms.sum(-1))
    S = (V / 64 + 64 + 260) * E
    bound = sizes.sum(-1) * (K * E + 600 * E + S)
    if g is None:
        return (loss, bound), None
    full = torch.zeros(R, V, dtype=torch.float64).scatter_add_(-1, at, torch.where(there, p, 0.0))
    q = torch.exp(log_q)
    rate = (g.double().cpu() / temperature)[:, None]
    grad = torch.where((none | nothing)[:, None], 0.0, rate * (q - full))
    grad = torch.where(bad[:, None], math.nan, grad)
    far = torch.where(x > -math.inf, (x.amax(-1, keepdim=True) - x), 0.0)
    room = rate.abs() * ((q + full) * (S + (300 + K) * E) + q * 4 * far * E + 2.0**-126)
    return (loss, bound), (grad, room)


def _close(got, want, what):
    value, bound = want
    dt = got.dtype
    got = got.detach().double().cpu()
    same = (got == value) | (got.isnan() & value.isnan())
    half = torch.finfo(dt).eps / 2
    room = bound + half * (value.abs() + bound) + 1e-37
    # (a bfloat16 below the least normal number is rounded to a multiple of 2^-133)
    room = room + (2.0**-134 if dt == torch.bfloat16 else 0.0)
    bad = ~(same | ((got - value).abs() <= room))
    assert not bool(bad.any()), f"{what}: {int(bad.sum())}, worst {float(((got - value).abs() / room)[bad].max()):.2f}"


def _teacher(R, V, K, g, spread=3.0):
    full = spread * torch.randn(R, V, generator=g)
    top = torch.topk(full, K)
    return full, top.values.to(DEV), top.indices.to(DEV)


def _run(x, values, tokens, temperature, g):
    leaf = x.detach().requires_grad_()
    loss = myelin.distillation_loss(leaf, values, tokens, temperature=temperature)
    (gx,) = torch.autograd.grad(loss, leaf, g)
    assert gx.dtype == x.dtype and gx.shape == x.shape and loss.dtype == torch.float32
    return loss, gx


SIZES = [(1, 1, 1), (3, 2, 2), (5, 10, 3), (2, 64, 64), (7, 255, 8), (4, 1000, 20), (2, 4096, 64), (3, 4097, 65),
         (1, 100003, 20), (9, 33000, 100), (600, 50, 5), (2, 5000, 1000), (130, 8200, 7), (1, 1500, 1024)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("R,V,K", SIZES)
def test_losses_and_gradients(R, V, K, dtype):
    _case(test="distillation", R=R, V=V, K=K, dtype=dtype)
    g = torch.Generator().manual_seed(R + V + K)
    full, values, tokens = _teacher(R, V, K, g)
    x = (0.7 * full + torch.randn(R, V, generator=g)).to(DTYPES[dtype]).to(DEV)
    weights = torch.randn(R, generator=g).to(DEV)
    order = torch.randperm(K, generator=g).to(DEV)
    for temperature in (1.0, 2.5, 0.1):
        want = _reference(x, values, tokens, temperature, weights)
        with torch.no_grad():
            quiet = myelin.distillation_loss(x, values, tokens, temperature=temperature)
        loss, gx = _run(x, values, tokens, temperature, weights)
        assert torch.equal(quiet, loss.detach())
        _close(loss, want[0], "loss")
        _close(gx, want[1], "gradient")
        # in any order, up to a constant, int32
        loss, gx = _run(x, values[:, order] - 5.0, tokens[:, order].int(), temperature, weights)
        shifted = _reference(x, values[:, order] - 5.0, tokens[:, order], temperature, weights)
        _close(loss, shifted[0], "loss in another order")
        _close(gx, shifted[1], "gradient in another order")


def test_a_student_that_is_the_teacher():
    g = torch.Generator().manual_seed(0)
    x = torch.randn(20, 30, generator=g).to(DEV)
    top = torch.topk(x, 30)
    loss, gx = _run(x, top.values, top.indices, 1.0, torch.ones(20, device=DEV))
    assert float(loss.detach().abs().max()) <= 30 * 20 * E * 5 and float(gx.abs().max()) <= 700 * E


def test_token_log_probs_gives_the_teacher():
    """Its alternatives, ignored rows among them, as they are."""

    g = torch.Generator().manual_seed(1)
    teacher = torch.randn(6, 4, 500, generator=g).to(DEV)
    x = torch.randn(6, 4, 500, generator=g).to(DEV)
    targets = torch.randint(0, 500, (6, 4), generator=g).to(DEV)
    targets[2, 1] = targets[5, 3] = -100
    r = myelin.token_log_probs(teacher, targets, top=9)
    weights = torch.randn(6, 4, generator=g).to(DEV)
    loss, gx = _run(x, r.top_log_probs, r.top_tokens, 1.5, weights)
    assert loss.shape == (6, 4) and loss[2, 1].item() == 0.0 == loss[5, 3].item()
    assert not bool(gx[2, 1].any()) and bool(gx[2, 2].any())
    want = _reference(x.view(24, 500), r.top_log_probs.view(24, 9), r.top_tokens.view(24, 9), 1.5, weights.view(24))
    _close(loss.view(24), want[0], "loss")
    _close(gx.view(24, 500), want[1], "gradient")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("V", [40, 700, 5000, 100000])
def test_masks_and_empty_places(V, dtype):
    _case(test="distillation_masks", V=V, dtype=dtype)
    g = torch.Generator().manual_seed(V)
    K, R = 6, 9
    full, values, tokens = _teacher(R, V, K, g)
    x = torch.randn(R, V, generator=g).to(DTYPES[dtype]).to(DEV)
    lowest = torch.finfo(DTYPES[dtype]).min
    # 0: the teacher's second token is masked for the student
    x[0, tokens[0, 1]] = -math.inf
    # 1: a token that the teacher does not name is
    other = next(i for i in range(V) if i not in tokens[1].tolist())
    x[1, other] = -math.inf
    # 2: nothing is allowed   3: everything has the type's lowest value
    x[2], x[3] = -math.inf, lowest
    # 4: some places are empty in either way, one with a token that would be outside
    tokens[4, 0], values[4, 3] = -1, -math.inf
    tokens[4, 3] = V + 7
    # 5: all are   6: the masked token has no probability
    tokens[5, :3], values[5, 3:] = -1, -math.inf
    x[6, tokens[6, 2]], values[6, 2] = -math.inf, -math.inf
    # 7: one token alone   8: lowest values for all but the teacher's tokens
    tokens[7, 1:] = -1
    keep = x[8, tokens[8]]
    x[8] = lowest
    x[8, tokens[8]] = keep
    weights = torch.randn(R, generator=g).to(DEV)
    loss, gx = _run(x, values, tokens, 1.0, weights)
    want = _reference(x, values, tokens, 1.0, weights)
    assert float(loss[0]) == math.inf and float(loss[2]) == math.inf and float(loss[5]) == 0.0
    assert not bool(gx[2].any()) and not bool(gx[5].any())
    _close(loss, want[0], "loss")
    _close(gx, want[1], "gradient")


@pytest.mark.parametrize("V", [30, 9000, 70000])
def test_what_is_not_finite_stays_in_its_row(V):
    g = torch.Generator().manual_seed(V)
    _, values, tokens = _teacher(8, V, 5, g)
    x = torch.randn(8, V, generator=g).to(DEV)
    weights = torch.ones(8, device=DEV)
    clean = _run(x, values, tokens, 1.0, weights)
    x[1, V // 2], x[2, V - 1] = math.nan, math.inf
    values[3, 2], values[4, 0] = math.nan, math.inf
    tokens[5, 4], tokens[6, 1] = V, -2
    loss, gx = _run(x, values, tokens, 1.0, weights)
    for row in (1, 2, 3, 4, 5, 6):
        assert bool(loss[row].isnan()), row
        assert bool(gx[row].isnan().any()), row
    for row in (5, 6):
        assert bool(gx[row].isnan().all())
    for row in (0, 7):
        assert torch.equal(loss[row], clean[0][row]) and torch.equal(gx[row], clean[1][row])


def test_a_token_named_twice():
    """The two places' probabilities add."""

    for V in (20, 6000):
        x = torch.randn(3, V, device=DEV)
        tokens = torch.tensor([[4, 7, 4, 4], [9, 9, 9, 9], [0, 1, 2, 3]], device=DEV)
        values = torch.randn(3, 4, device=DEV)
        weights = torch.tensor([1.0, -2.0, 0.0], device=DEV)
        loss, gx = _run(x, values, tokens, 1.0, weights)
        want = _reference(x, values, tokens, 1.0, weights)
        _close(loss, want[0], "loss")
        _close(gx, want[1], "gradient")
        assert not bool(gx[2].any())
        # the first of the two places with a probability that is 0 in float32
        values = torch.tensor([[-300.0, 0.0, 1.0, -400.0]] * 3, device=DEV)
        tokens = torch.tensor([[4, 4, 7, 4], [7, 4, 4, 7], [5, 9, 9, 9]], device=DEV)
        loss, gx = _run(x, values, tokens, 1.0, weights)
        want = _reference(x, values, tokens, 1.0, weights)
        _close(loss, want[0], "loss")
        _close(gx, want[1], "gradient")


@pytest.mark.parametrize("shift", [-1e4, 1e4, 3e38])
def test_far_logits(shift):
    """Logits far from 0: differences count.  (A row of them has few values.)"""

    g = torch.Generator().manual_seed(5)
    x = (torch.randn(4, 3000, generator=g) + shift).to(DEV)
    _, values, tokens = _teacher(4, 3000, 6, g)
    weights = torch.ones(4, device=DEV)
    want = _reference(x, values + (shift if abs(shift) < 1e5 else 0), tokens, 1.0, weights)
    loss, gx = _run(x, values + (shift if abs(shift) < 1e5 else 0), tokens, 1.0, weights)
    _close(loss, want[0], "loss")
    _close(gx, want[1], "gradient")


def test_gradients_are_the_differences_of_the_definition():
    """Central differences of step h: h^2 / 6 of a third derivative, at most 1 of
    the direction's cubes."""

    g = torch.Generator().manual_seed(6)
    R, V, K, h = 3, 60, 7, 1e-3
    _, values, tokens = _teacher(R, V, K, g)
    x = torch.randn(R, V, generator=g).to(DEV)
    weights = torch.randn(R, generator=g).to(DEV)
    _, gx = _run(x, values, tokens, 2.0, weights)
    d = torch.randn(R, V, generator=g, dtype=torch.float64)
    up, down = (_reference(x.cpu().double() + s * h * d, values, tokens, 2.0)[0][0] for s in (1, -1))
    slope = ((up - down) / (2 * h) * weights.cpu().double()).sum()
    got = (gx.double().cpu() * d).sum()
    assert abs(float(slope - got)) <= h * h * float(d.abs().pow(3).sum()) + 1e-5


@pytest.mark.parametrize("dtype", DTYPES)
def test_layouts(dtype):
    g = torch.Generator().manual_seed(7)
    base = torch.randn(12, 4200, generator=g).to(DTYPES[dtype]).to(DEV)
    weights = torch.randn(12, generator=g).to(DEV)
    for x in (base[:, :4096], base[:, 1:4098], base[:, 3:900], base[:, ::2], base[:, 7:50]):
        V = x.shape[1]
        values = torch.randn(12, 10, generator=g).to(DEV)[:, ::2]
        tokens = torch.randint(0, V, (5, 12), generator=g).to(DEV).t()
        a, b = _run(x, values, tokens, 1.0, weights), _run(x.contiguous(), values.contiguous(), tokens.contiguous(), 1.0,
                                                           weights)
        want = _reference(x, values, tokens, 1.0, weights)
        for u, v in zip(a, want):
            _close(u, v, V)
        for u, v in zip(b, want):
            _close(u, v, V)
    x = base[:, :100].reshape(3, 4, 100)
    tokens = torch.randint(0, 100, (3, 4, 6), generator=g).to(DEV)
    values = torch.randn(3, 4, 6, generator=g).to(DEV)
    loss = myelin.distillation_loss(x.transpose(0, 1), values.transpose(0, 1), tokens.transpose(0, 1))
    assert loss.shape == (4, 3)
    flat = myelin.distillation_loss(x.reshape(12, 100), values.view(12, 6), tokens.view(12, 6)).view(3, 4)
    assert torch.equal(loss, flat.t())
    one = myelin.distillation_loss(x[1, 2], values[1, 2], tokens[1, 2])
    assert one.shape == () and torch.equal(one, flat[1, 2])
    # a bfloat16 teacher, an expanded gradient
    leaf = x.reshape(12, 100).detach().requires_grad_()
    low = values.view(12, 6).bfloat16()
    (a,) = torch.autograd.grad(myelin.distillation_loss(leaf, low, tokens.view(12, 6)).sum(), leaf)
    (b,) = torch.autograd.grad(myelin.distillation_loss(leaf, low.float(), tokens.view(12, 6)), leaf,
                               torch.ones(12, device=DEV))
    assert torch.equal(a, b)


def test_no_rows():
    x = torch.empty(0, 10, device=DEV, requires_grad=True)
    loss = myelin.distillation_loss(x, torch.empty(0, 3, device=DEV), torch.empty(0, 3, dtype=torch.int64, device=DEV))
    assert loss.shape == (0,)
    (gx,) = torch.autograd.grad(loss.sum(), x)
    assert gx.shape == (0, 10)


def test_offsets_past_32_bits():
    _case(test="distillation_large")
    R, V = 16500, 131072
    x = torch.empty(R, V, dtype=torch.bfloat16, device=DEV).normal_(generator=torch.Generator(device=DEV).manual_seed(0))
    tokens = torch.tensor([[5, V - 1, 70000]], device=DEV).expand(R, 3)
    values = torch.tensor([[1.0, 2.0, 0.0]], device=DEV).expand(R, 3)
    weights = torch.ones(R, device=DEV)
    loss, gx = _run(x, values, tokens, 1.0, weights)
    some = torch.tensor([0, R - 200, R - 1], device=DEV)
    want = _reference(x[some], values[some], tokens[some], 1.0, weights[some])
    _close(loss[some], want[0], "loss")
    _close(gx[some], want[1], "gradient")


def test_refusals():
    x = torch.zeros(4, 10, device=DEV)
    v = torch.zeros(4, 3, device=DEV)
    t = torch.zeros(4, 3, dtype=torch.int64, device=DEV)
    f = myelin.distillation_loss
    for bad, message in ((lambda: f(x[:, :0], v, t), "V > 0"), (lambda: f(x.half(), v, t), "float32 or bfloat16"),
                         (lambda: f(x, v.double(), t), "float32 or bfloat16"), (lambda: f(x, v[:2], t[:2]), "rows of"),
                         (lambda: f(x, v[0], t[0]), "rows of"), (lambda: f(x, v, t[:, :2]), "teacher_tokens must match"),
                         (lambda: f(x, v[:, :0], t[:, :0]), "places a row"),
                         (lambda: f(x, v.repeat(1, 400), t.repeat(1, 400)), "places a row"),
                         (lambda: f(x, v.cpu(), t), "same device"), (lambda: f(x, v, t.cpu()), "same device"),
                         (lambda: f(x, v, t.float()), "int64 or int32"),
                         (lambda: f(x, v.clone().requires_grad_(), t), "pass teacher_logits detached"),
                         (lambda: f(x, v, t, temperature=0.0), "temperature must"),
                         (lambda: f(x, v, t, temperature=-1.0), "temperature must"),
                         (lambda: f(x, v, t, temperature=math.inf), "temperature must"),
                         (lambda: f(x, v, t, temperature=math.nan), "temperature must")):
        with pytest.raises(ValueError, match=message):
            bad()
