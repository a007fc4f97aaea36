"""decay_attention, its gradients and its single step against the recurrence in
float64.

Tolerances.  Let A be the same result on the inputs' absolute values: the sum of
the magnitudes of every term.  fp32: each term has a few roundings and its sum a
few hundred, of random sign: within 256 * 2^-24 of A.  bf16 inputs are exact, but
a partial product may be rounded to bf16 (2^-8) before it is multiplied again, and
the result is: 2^-8 (A + |value|) on top.  States are fp32 for either type, their
terms rounded to no less than 16 bits: 2^-16 A on top for bf16.
"""

from __future__ import annotations

import math

import pytest
import torch

import myelin_amd as myelin

pytestmark = pytest.mark.gpu
DEV = "cuda"
DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16}


def _case(**kw):
    print("case:", " ".join(f"{k}={v}" for k, v in kw.items()), flush=True)


def _inputs(T, B, H, Hk, Dk, Dv, dtype, seed=0, state=True):
    g = torch.Generator().manual_seed(seed * 7919 + T * 31 + B * 7 + H + Dk * 3 + Dv)
    dt = DTYPES[dtype]
    q, k = (torch.randn(T, B, h, Dk, generator=g).to(dt).to(DEV) for h in (H, Hk))
    v, go = (torch.randn(T, B, h, Dv, generator=g).to(dt).to(DEV) for h in (Hk, H))
    s, gs = (torch.randn(B, H, Dk, Dv, generator=g).to(DEV) for _ in range(2))
    taus = torch.logspace(0.3, 3, H, dtype=torch.float64)
    decay = (1 - 1 / taus).float().to(DEV)
    return q, k, v, decay, s if state else None, go, gs


def _reference(q, k, v, decay, state, lengths, scale, g_out=None, g_state=None, device="cpu"):
    """The recurrence and its adjoint: (state, out, gq, gk, gv, gstate)."""

    T, B, H, Dk = q.shape
    Hk, Dv = v.shape[-2:]
    q, k, v, d = (t.detach().double().to(device) for t in (q, k, v, decay))
    n = torch.full((B,), T) if lengths is None else lengths.cpu().long().clamp(0, T)
    live = (torch.arange(T)[:, None] < n[None]).to(device)[..., None, None]  # [T, B, 1, 1]
    q, k, v = (torch.where(live, t, 0.0) for t in (q, k, v))
    k, v = (t.repeat_interleave(H // Hk, 2) for t in (k, v))
    fade = torch.where(live[..., None], d[:, None, None], 1.0)  # [T, B, H, 1, 1]
    S = torch.zeros(B, H, Dk, Dv, dtype=torch.float64, device=device) if state is None else state.detach().double().to(device)
    out = torch.zeros(T, B, H, Dv, dtype=torch.float64, device=device)
    grads = g_out is not None
    gq, gk, gv = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    if grads:
        g_out = torch.where(live, g_out.detach().double().to(device), 0.0)
    for t in range(T):
        S = fade[t] * S + k[t][..., None] * v[t][..., None, :]
        out[t] = scale * (q[t][..., None] * S).sum(-2)
        if grads:
            gq[t] = scale * (S * g_out[t][..., None, :]).sum(-1)
    if not grads:
        return S, out
    G = g_state.detach().double().to(device) if g_state is not None else torch.zeros_like(S)
    for t in range(T - 1, -1, -1):
        G = G + scale * q[t][..., None] * g_out[t][..., None, :]
        gk[t] = torch.where(live[t], (G * v[t][..., None, :]).sum(-1), 0.0)
        gv[t] = torch.where(live[t], (G * k[t][..., None]).sum(-2), 0.0)
        G = fade[t] * G
    gk, gv = (t.view(T, B, Hk, H // Hk, -1).sum(3) for t in (gk, gv))
    return S, out, gq, gk, gv, G


NAMES = ("state", "out", "gq", "gk", "gv", "gstate")


def _close(name, got, want, size, dtype):
    got, want, size = got.detach().double().cpu(), want.cpu(), size.cpu()
    tol = 256 * 2.0**-24 * size
    if dtype == "bf16":
        tol = tol + (2.0**-16 * size if "state" in name else 2.0**-8 * (size + want.abs()))
    err = (got - want).abs()
    assert got.shape == want.shape, f"{name}: shape"
    assert bool(torch.isfinite(got).all()), f"{name}: not finite"
    assert bool((err <= tol + 1e-30).all()), f"{name}: worst {float((err / (tol + 1e-30)).max()):.3g} of the tolerance"


def _check(q, k, v, decay, state, lengths, dtype, go=None, gs=None, scale=None, device="cpu"):
    sc = q.shape[-1] ** -0.5 if scale is None else scale
    leaves = [t.detach().requires_grad_() if go is not None and t is not None else t for t in (q, k, v, state)]
    q, k, v, state = leaves
    final, out = myelin.decay_attention(q, k, v, decay, state, lengths=lengths, scale=scale)
    assert out.dtype == q.dtype and final.dtype == torch.float32
    got = [final, out]
    if go is not None:
        wrt = [t for t in leaves if t is not None]
        got += torch.autograd.grad((final, out), wrt, (gs, go))
    args = (q, k, v, decay, state)
    want = _reference(*args, lengths, sc, go, gs, device)
    ab = lambda t: None if t is None else t.detach().abs()  # noqa: E731
    # NaN where nothing is read stays out of the magnitudes too
    size = _reference(*(ab(t) for t in args), lengths, abs(sc), ab(go), ab(gs), device)
    for name, g, w, z in zip(NAMES, got, want, size):
        _close(name, g, w, z, dtype)
    return got


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T", [1, 2, 15, 16, 17, 63, 64, 65, 127, 128, 129, 300, 517])
def test_lengths_of_time(T, dtype):
    _case(test="attention_T", T=T, dtype=dtype)
    q, k, v, d, s, go, gs = _inputs(T, 2, 3, 3, 24, 40, dtype)
    _check(q, k, v, d, None, None, dtype, go, gs)
    _check(q, k, v, d, s, None, dtype, go, gs)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("Dk,Dv", [(1, 1), (1, 128), (128, 1), (7, 9), (16, 16), (17, 33), (32, 64), (64, 32), (65, 66),
                                   (96, 100), (127, 128), (128, 127), (128, 128)])
def test_widths(Dk, Dv, dtype):
    _case(test="attention_widths", Dk=Dk, Dv=Dv, dtype=dtype)
    q, k, v, d, s, go, gs = _inputs(150, 2, 2, 1, Dk, Dv, dtype)
    _check(q, k, v, d, s, None, dtype, go, gs)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,H,Hk", [(1, 1, 1), (3, 4, 4), (2, 4, 2), (1, 6, 1), (40, 8, 2)])
def test_shared_heads_and_ragged_lengths(B, H, Hk, dtype):
    _case(test="attention_heads", B=B, H=H, Hk=Hk, dtype=dtype)
    T = 140
    q, k, v, d, s, go, gs = _inputs(T, B, H, Hk, 32, 48, dtype)
    n = torch.randint(0, T + 1, (B,), generator=torch.Generator().manual_seed(B))
    n[0] = 70
    if B > 2:
        n[1], n[2] = 0, 1
    if B > 6:  # taken into [0, T]
        n[3], n[4], n[5], n[6] = T, T + 100, -5, 64
    for kind in (torch.int32, torch.int64):
        _check(q, k, v, d, s, n.to(kind).to(DEV), dtype, go, gs)
    _check(q, k, v, d, None, n.to(DEV), dtype, go, gs)


@pytest.mark.parametrize("dtype", DTYPES)
def test_steps_past_a_length_are_not_read(dtype):
    _case(test="attention_padding", dtype=dtype)
    T, B = 200, 4
    q, k, v, d, s, go, gs = _inputs(T, B, 2, 1, 40, 24, dtype)
    n = torch.tensor([0, 1, 64, 131], device=DEV)
    clean = _check(q, k, v, d, s, n, dtype, go, gs)
    pad = (torch.arange(T, device=DEV)[:, None] >= n).view(T, B, 1, 1)
    for bad in (math.nan, math.inf):
        dirty = [torch.where(pad, torch.full((), bad, dtype=t.dtype, device=DEV), t).requires_grad_() for t in (q, k, v)]
        state = s.clone().requires_grad_()
        final, out = myelin.decay_attention(*dirty, d, state, lengths=n)
        grads = torch.autograd.grad((final, out), (*dirty, state),
                                    (gs, torch.where(pad, torch.full((), bad, dtype=go.dtype, device=DEV), go)))
        for name, a, b in zip(NAMES, (final, out, *grads), clean):
            assert torch.equal(a, b), name
        for t in (out, *grads[:3]):
            assert bool((t[pad.expand_as(t)] == 0).all())


@pytest.mark.parametrize("dtype", DTYPES)
def test_decays_from_nothing_to_everything(dtype):
    _case(test="attention_decays", dtype=dtype)
    q, k, v, _, s, go, gs = _inputs(200, 2, 6, 6, 20, 30, dtype)
    d = torch.tensor([0.0, 1e-30, 1e-3, 0.5, 1.0 - 2.0**-20, 1.0], device=DEV)
    _check(q, k, v, d, s, None, dtype, go, gs)
    _check(q, k, v, d, s, torch.tensor([3, 130], device=DEV), dtype, go, gs, scale=-2.5)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("Dk,Dv", [(64, 64), (20, 36)])
def test_layouts(Dk, Dv, dtype):
    """Batch-major and head-major storage, slices that start anywhere, expanded
    inputs, transposed widths."""

    _case(test="attention_layouts", Dk=Dk, Dv=Dv, dtype=dtype)
    T, B, H = 70, 3, 2
    q, k, v, d, s, go, gs = _inputs(T, B, H, H, Dk, Dv, dtype)
    plain = _check(q, k, v, d, s, None, dtype, go, gs)

    def same(views, what):
        leaves = [t.detach().requires_grad_() for t in views]
        state = s.clone().requires_grad_()
        final, out = myelin.decay_attention(*leaves, d, state)
        grads = torch.autograd.grad((final, out), (*leaves, state), (gs, go))
        for name, a, b in zip(NAMES, (final, out, *grads), plain):
            assert torch.equal(a, b), f"{what}: {name}"

    same([t.transpose(0, 1).contiguous().transpose(0, 1) for t in (q, k, v)], "batch-major")
    same([t.permute(1, 2, 0, 3).contiguous().permute(2, 0, 1, 3) for t in (q, k, v)], "head-major")
    same([t.transpose(2, 3).contiguous().transpose(2, 3) for t in (q, k, v)], "transposed widths")
    for shift in (1, 4, 8):
        wide = [torch.zeros(*t.shape[:-1], t.shape[-1] + 16, dtype=t.dtype, device=DEV) for t in (q, k, v)]
        views = []
        for w, t in zip(wide, (q, k, v)):
            w[..., shift : shift + t.shape[-1]] = t
            views.append(w[..., shift : shift + t.shape[-1]])
        same(views, f"slices at {shift}")
    packed = torch.cat((q, k, v), -1)  # one projection's output
    same(list(packed.split((Dk, Dk, Dv), -1)), "split projection")
    # one key for all steps and samples, a gradient that is an expanded scalar
    k1 = k[:1, :1].detach().clone().requires_grad_()
    final, out = myelin.decay_attention(q, k1.expand(T, B, H, Dk), v, d, s)
    (g1,) = torch.autograd.grad(out.sum(), k1)
    want = _reference(q, k1.expand(T, B, H, Dk), v, d, s, None, Dk**-0.5, torch.ones_like(go))
    size = _reference(q.abs(), k1.abs().expand(T, B, H, Dk), v.abs(), d, s.abs(), None, Dk**-0.5, torch.ones_like(go))
    _close("gk", g1, want[3].sum((0, 1), keepdim=True), size[3].sum((0, 1), keepdim=True), dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,B,H,Hk,Dk,Dv", [(5000, 1, 2, 2, 64, 64), (3001, 2, 1, 1, 128, 100), (4100, 1, 2, 1, 33, 20)])
def test_long_sequences(T, B, H, Hk, Dk, Dv, dtype):
    _case(test="attention_long", T=T, B=B, H=H, Dk=Dk, Dv=Dv, dtype=dtype)
    q, k, v, d, s, go, gs = _inputs(T, B, H, Hk, Dk, Dv, dtype)
    _check(q, k, v, d, s, None, dtype, go, gs, device=DEV)
    n = torch.tensor([T - 300, 700][:B], device=DEV)
    _check(q, k, v, d, None, n, dtype, go, gs, device=DEV)


@pytest.mark.parametrize("T", [37, 1300])
def test_gradients_are_difference_quotients(T):
    """out and state are linear in each of q, k, v and the initial state, so the
    difference over 2 along d is exact: (f(x + d) - f(x - d)) / 2 = f'(x) d, but
    for the roundings of two results: 512 * 2^-24 of their terms' magnitudes."""

    _case(test="attention_differences", T=T)
    q, k, v, decay, s, go, gs = _inputs(T, 2, 4, 2, 20, 28, "fp32")
    n = torch.tensor([T, T - 20], device=DEV)
    leaves = {"q": q, "k": k, "v": v, "s": s}
    for t in leaves.values():
        t.requires_grad_()

    def f(x):
        final, out = myelin.decay_attention(x["q"], x["k"], x["v"], decay, x["s"], lengths=n)
        return final, out

    grads = dict(zip(leaves, torch.autograd.grad(f(leaves), list(leaves.values()), (gs, go))))
    with torch.no_grad():
        for name, x in leaves.items():
            d = torch.randn(x.shape, generator=torch.Generator().manual_seed(3)).to(DEV)
            up, down = f({**leaves, name: x + d}), f({**leaves, name: x - d})
            slope = sum(float(((a.double() - b.double()) / 2 * g.double()).sum()) for a, b, g in zip(up, down, (gs, go)))
            size = sum(float((a.double().abs() * g.double().abs()).sum()) for a, g in zip(up, (gs, go)))
            assert abs(slope - float((grads[name].double() * d.double()).sum())) <= 512 * 2.0**-24 * size, name


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,H,Hk,Dk,Dv", [(1, 1, 1, 1, 1), (2, 3, 1, 7, 9), (5, 4, 2, 64, 64), (3, 2, 2, 128, 128),
                                          (2, 2, 2, 33, 30), (300, 2, 2, 16, 100), (2, 4, 1, 128, 20)])
def test_single_steps(B, H, Hk, Dk, Dv, dtype):
    """One step against its formula; several against the whole sequence."""

    _case(test="attention_step", B=B, H=H, Dk=Dk, Dv=Dv, dtype=dtype)
    T = 5
    q, k, v, d, s, _, _ = _inputs(T, B, H, Hk, Dk, Dv, dtype)
    sc = Dk**-0.5
    state = s.clone()
    for t in range(T):
        before = state
        state, out = myelin.decay_attention_step(q[t], k[t], v[t], d, state)
        assert torch.equal(before, s) or t > 0  # the given state is kept
        one = (q[t : t + 1], k[t : t + 1], v[t : t + 1])
        want = _reference(*one, d, before, None, sc)
        size = _reference(*(x.abs() for x in one), d, before.abs(), None, sc)
        _close("state", state, want[0], size[0], dtype)
        _close("out", out, want[1][0], size[1][0], dtype)
    whole = _reference(q, k, v, d, s, None, sc)
    size = _reference(q.abs(), k.abs(), v.abs(), d, s.abs(), None, sc)
    _close("state", state, whole[0], size[0], dtype)
    inplace = s.clone()
    kept = inplace.data_ptr()
    for t in range(T):
        inplace, out = myelin.decay_attention_step(q[t], k[t], v[t], d, inplace, out_state=inplace)
    assert inplace.data_ptr() == kept and torch.equal(inplace, state)
    # strided rows, a state that starts off a multiple of 16 bytes
    room = torch.zeros(s.numel() + 1, device=DEV)
    off = room[1:].view_as(s).copy_(s)
    a = myelin.decay_attention_step(q[0], k[0], v[0], d, off)
    b = myelin.decay_attention_step(q[0].transpose(0, 1).contiguous().transpose(0, 1), k[0], v[0], d, s)
    _close("state", a[0], b[0].double(), b[0].double().abs(), "fp32")
    _close("out", a[1], b[1].double(), _reference(*(x[:1].abs() for x in (q, k, v)), d, s.abs(), None, sc)[1][0], dtype)


@pytest.mark.parametrize("dtype", DTYPES)
def test_a_prompt_continues_where_another_ended(dtype):
    q, k, v, d, s, _, _ = _inputs(333, 2, 2, 2, 48, 48, dtype)
    _case(test="attention_continued", dtype=dtype)
    whole = _reference(q, k, v, d, s, None, 48**-0.5)
    size = _reference(q.abs(), k.abs(), v.abs(), d, s.abs(), None, 48**-0.5)
    state, outs = s, []
    for a, b in ((0, 100), (100, 101), (101, 333)):
        state, out = myelin.decay_attention(q[a:b], k[a:b], v[a:b], d, state)
        outs.append(out)
    _close("state", state, whole[0], size[0], dtype)
    _close("out", torch.cat(outs), whole[1], size[1], dtype)


def test_partial_gradients():
    """Only one output's gradient, only some inputs'."""

    q, k, v, d, s, go, gs = _inputs(90, 2, 2, 2, 16, 16, "fp32")
    _case(test="attention_partial")
    both = _reference(q, k, v, d, s, None, 0.25, go, gs)
    size = _reference(q.abs(), k.abs(), v.abs(), d, s.abs(), None, 0.25, go.abs(), gs.abs())
    k.requires_grad_()
    final, out = myelin.decay_attention(q, k, v, d, s)
    (gk,) = torch.autograd.grad((final, out), k, (gs, go), retain_graph=True)
    _close("gk", gk, both[3], size[3], "fp32")
    (a,) = torch.autograd.grad(final, k, gs, retain_graph=True)
    (b,) = torch.autograd.grad(out, k, go, retain_graph=True)
    _close("gk", a + b, both[3], size[3], "fp32")
    g = torch.autograd.grad(out, k, go, create_graph=True)[0]
    with pytest.raises(RuntimeError):
        torch.autograd.grad(g.sum(), k)


def test_runs_are_repeatable_on_other_streams_and_in_graphs():
    _case(test="attention_graph")
    q, k, v, d, s, go, gs = _inputs(700, 2, 4, 2, 64, 40, "bf16")
    n = torch.tensor([700, 350], dtype=torch.int32, device=DEV)
    leaves = [t.requires_grad_() for t in (q, k, v, s)]

    def body():
        final, out = myelin.decay_attention(q, k, v, d, s, lengths=n)
        grads = torch.autograd.grad((final, out), leaves, (gs, go))
        with torch.no_grad():
            step = myelin.decay_attention_step(q[0], k[0], v[0], d, final.detach())
        return [final.detach(), out.detach(), *grads, *step]

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
        _ = float((q.detach().float() * 2.0).sum())


def test_module():
    with pytest.raises(ValueError, match="taus"):
        myelin.DecayAttention([])
    with pytest.raises(ValueError, match="taus"):
        myelin.DecayAttention([4.0, 0.5])
    m = myelin.DecayAttention([1.0, 2.0, math.inf]).to(DEV)
    assert m.decay.tolist() == [0.0, 0.5, 1.0]
    q, k, v, _, s, _, _ = _inputs(6, 2, 3, 3, 8, 8, "fp32")
    final, out = m(q, k, v, s)
    want = myelin.decay_attention(q, k, v, m.decay, s)
    assert torch.equal(final, want[0]) and torch.equal(out, want[1])
    a, b = m.step(q[0], k[0], v[0], s), myelin.decay_attention_step(q[0], k[0], v[0], m.decay, s)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_no_samples():
    q, k, v, d, s, _, _ = _inputs(6, 2, 3, 3, 8, 8, "fp32")
    final, out = myelin.decay_attention(q[:, :0], k[:, :0], v[:, :0], d, s[:0])
    assert final.shape == (0, 3, 8, 8) and out.shape == (6, 0, 3, 8)


def test_refusals():
    q, k, v, d, s, _, _ = _inputs(6, 2, 4, 2, 8, 8, "fp32")
    f, g = myelin.decay_attention, myelin.decay_attention_step
    wide = torch.zeros(6, 2, 2, 129, device=DEV)
    one = (q[0], k[0], v[0])
    for bad, message in (
            (lambda: f(q[0], k, v, d), "q must be shaped"), (lambda: f(q.half(), k.half(), v.half(), d), "float32 or"),
            (lambda: f(q, k.bfloat16(), v, d), "same dtype"), (lambda: f(q, k.cpu(), v, d), "ROCm device"),
            (lambda: f(q, k[:5], v, d), "time and batch sizes"), (lambda: f(q, k, v[:, :, :1], d), "same heads"),
            (lambda: f(q[..., :7], k, v, d), "same width"), (lambda: f(q[:, :, :3], k, v, d[:3]), "multiple"),
            (lambda: f(q, k, wide, d), "width must be"), (lambda: f(q[:0], k[:0], v[:0], d), "one timestep"),
            (lambda: f(q, k, v, d[:2]), "decay must be"), (lambda: f(q, k, v, d.double()), "decay must be"),
            (lambda: f(q, k, v, d.clone().requires_grad_()), "constant of the heads"),
            (lambda: f(q, k, v, d, s[:1]), "initial_state must be"),
            (lambda: f(q, k, v, d, s.bfloat16()), "initial_state must be"),
            (lambda: f(q, k, v, d, lengths=torch.ones(3, dtype=torch.int32, device=DEV)), "lengths must be"),
            (lambda: f(q, k, v, d, lengths=torch.ones(2, device=DEV)), "int32 or int64"),
            (lambda: f(q, k, v, d, scale=0.0), "scale must be"), (lambda: f(q, k, v, d, scale=math.inf), "scale must"),
            (lambda: g(q, k, v, d, s), "q must be shaped"), (lambda: g(*one, d, s[:, :2]), "state must be"),
            (lambda: g(*one, d, s.clone().requires_grad_()), "no gradient"),
            (lambda: g(*one, d, s, out_state=s.transpose(2, 3)), "contiguous"),
            (lambda: g(*one, d, s, out_state=s[:1]), "out_state must be")):
        with pytest.raises(ValueError, match=message):
            bad()
    room = torch.zeros(s.numel() + 4, device=DEV)
    with pytest.raises(ValueError, match="not overlap"):
        g(*one, d, room[: s.numel()].view_as(s), out_state=room[4:].view_as(s))


@pytest.mark.parametrize("bad", [math.nan, math.inf])
@pytest.mark.parametrize("which", ["q", "k", "v", "go"])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,Dk,Dv", [(100, 20, 36), (300, 128, 128)])
def test_a_value_reaches_no_step_before_it(T, Dk, Dv, dtype, which, bad):
    """A NaN or an infinity in one step: outputs before it, and gradients that it
    is not part of, are those of the formula, also within its chunk."""

    _case(test="attention_causal", T=T, Dk=Dk, Dv=Dv, dtype=dtype, which=which, bad=bad)
    q, k, v, d, s, go, gs = _inputs(T, 1, 2, 1, Dk, Dv, dtype)
    clean = dict(q=q, k=k, v=v, go=go)
    dirty = {n: t.clone() for n, t in clean.items()}
    at = 77
    dirty[which][at, 0, 0, Dk // 3] = bad
    leaves = [dirty[n].requires_grad_() for n in ("q", "k", "v")] + [s.clone().requires_grad_()]
    final, out = myelin.decay_attention(*leaves[:3], d, leaves[3])
    got = (final, out, *torch.autograd.grad((final, out), leaves, (gs, dirty["go"])))
    scale = Dk**-0.5
    want = _reference(*leaves[:3], d, s, None, scale, dirty["go"], gs)
    size = _reference(q.abs(), k.abs(), v.abs(), d, s.abs(), None, scale, go.abs(), gs.abs())
    for name, a, w, z in zip(NAMES, got, want, size):
        a = a.detach().double().cpu()
        if "state" not in name:
            # the formula's sums over a whole step: NaN in all that it is part of
            w = torch.where(w.isfinite().all(-1, keepdim=True), w, math.nan) if name[0] == "g" else w
        ok = w.isfinite()
        _close(name, torch.where(ok, a, 0.0), torch.where(ok, w, 0.0), z, dtype)
    first = dict(q=(1, slice(0, at)), k=(1, slice(0, at)), v=(1, slice(0, at)), go=(3, slice(at + 1, T)))[which]
    assert bool(got[first[0]][first[1]].isfinite().all())
    if which in ("q", "go"):  # gradients of later steps, and of every other step's q
        assert bool(got[3][at + 1 :].isfinite().all()) and bool(got[4][at + 1 :].isfinite().all())
    if which in ("k", "v"):
        assert bool(got[2][:at].isfinite().all())


@pytest.mark.parametrize("kind", [torch.Tensor, torch.nn.Parameter])
def test_a_state_advanced_in_place_is_noticed(kind):
    """The backward pass of a sequence reads its initial state again."""

    _case(test="attention_state_version", kind=kind.__name__)
    q, k, v, d, s, go, _ = _inputs(20, 2, 2, 2, 8, 8, "fp32")
    if kind is torch.nn.Parameter:
        s = torch.nn.Parameter(s, requires_grad=False)
    q.requires_grad_()
    _, out = myelin.decay_attention(q, k, v, d, s)
    _, kept = myelin.decay_attention(q, k, v, d, s[:, :])
    with torch.no_grad():
        other, _ = myelin.decay_attention_step(q[0], k[0], v[0], d, s)  # a new tensor: nothing has changed
        assert other is not s
        torch.autograd.grad(out, q, go, retain_graph=True)
        myelin.decay_attention_step(q[0], k[0], v[0], d, s, out_state=s)
    for o in (out, kept):
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            torch.autograd.grad(o, q, go)
    with torch.inference_mode():  # tensors without a version
        a, b = (t.clone() for t in (s.detach(), s.detach()))
        one = (q[0].clone(), k[0].clone(), v[0].clone(), d.clone())
        new, _ = myelin.decay_attention_step(*one, a)
        myelin.decay_attention_step(*one, b, out_state=b)
        assert torch.equal(new, b)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,H,Hk,Dk,Dv", [(300, 2, 2, 128, 128), (2100, 2, 1, 64, 40)])
def test_gradients_do_not_depend_on_which_are_asked_for(T, H, Hk, Dk, Dv, dtype):
    _case(test="attention_which_gradients", T=T, Dk=Dk, Dv=Dv, dtype=dtype)
    q, k, v, d, s, go, gs = _inputs(T, 2, H, Hk, Dk, Dv, dtype)
    every = None
    for wanted in ((0, 1, 2, 3), (0, 1, 2), (0,), (1, 3)):
        leaves = [t.clone().requires_grad_(i in wanted) for i, t in enumerate((q, k, v, s))]
        final, out = myelin.decay_attention(*leaves[:3], d, leaves[3])
        grads = dict(zip(wanted, torch.autograd.grad((final, out), [leaves[i] for i in wanted], (gs, go))))
        every = every or grads
        for i, g in grads.items():
            assert torch.equal(g, every[i]), NAMES[2 + i]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("scale", [1e-30, 1e-39, -3e-42])
@pytest.mark.parametrize("T", [70, 1300])
def test_small_scales(T, scale, dtype):
    """Nothing is divided by the scale: a state's gradient of 1e9 passes through at
    any.  (Terms that the scale makes smaller than 2^-126 may be lost: 1e-38 of
    sums that are held to 1e-30.)"""

    _case(test="attention_small_scale", T=T, scale=scale, dtype=dtype)
    q, k, v, d, s, go, gs = _inputs(T, 2, 2, 1, 24, 40, dtype)
    _check(q, k, v, d, s, None, dtype, go, gs * 1e9, scale=scale)


def test_few_heads_use_the_whole_chip():
    """A long prompt of 2 heads has an eighth of the work of 16, which fill the
    chip, and more of its time in launches: held to 0.4 of theirs (0.26 measured;
    on two of the eight XCDs 0.54)."""

    _case(test="attention_few_heads")

    def microseconds(heads):
        q, k, v, d, _, _, _ = _inputs(32768, 1, heads, heads, 128, 128, "bf16", state=False)
        times = []
        for _ in range(8):
            start, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
            start.record()
            for _ in range(10):
                myelin.decay_attention(q, k, v, d)
            end.record()
            torch.cuda.synchronize()
            times.append(start.elapsed_time(end) * 100.0)
        return min(times)

    with torch.no_grad():
        few, many = microseconds(2), microseconds(16)
    print(f"2 heads {few:.0f} us, 16 heads {many:.0f} us", flush=True)
    assert few <= 0.4 * many


@pytest.mark.parametrize("bad", [math.nan, math.inf])
@pytest.mark.parametrize("which", ["q", "k", "v", "go"])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,Dk,Dv", [(100, 20, 36), (300, 128, 128)])
def test_a_value_is_not_lost(T, Dk, Dv, dtype, which, bad):
    """A NaN or an infinity in one step: wherever the formula has one, in its own
    chunk and in later ones, the results have."""

    _case(test="attention_not_lost", T=T, Dk=Dk, Dv=Dv, dtype=dtype, which=which, bad=bad)
    q, k, v, d, s, go, gs = _inputs(T, 1, 2, 1, Dk, Dv, dtype)
    dirty = {n: t.clone() for n, t in dict(q=q, k=k, v=v, go=go).items()}
    at = 77
    dirty[which][at, 0, 0, Dk // 3] = bad
    leaves = [dirty[n].requires_grad_() for n in ("q", "k", "v")] + [s.clone().requires_grad_()]
    final, out = myelin.decay_attention(*leaves[:3], d, leaves[3])
    got = (final, out, *torch.autograd.grad((final, out), leaves, (gs, dirty["go"])))
    want = _reference(*leaves[:3], d, s, None, Dk**-0.5, dirty["go"], gs)
    reached = {"q": ("out", "gk", "gv", "gstate"), "k": ("state", "out", "gq", "gv"), "v": ("state", "out", "gq", "gk"),
               "go": ("gq", "gk", "gv", "gstate")}[which]
    for name, a, w in zip(NAMES, got, want):
        strange = ~w.isfinite()
        assert bool(strange.any()) == (name in reached), name
        assert not bool((a.detach().cpu().isfinite() & strange).any()), name


@pytest.mark.parametrize("T,H,Hk,Dk,Dv", [(300, 2, 2, 128, 128), (517, 4, 2, 50, 75), (1400, 2, 1, 64, 96), (40, 2, 2, 128, 20)])
def test_bf16_results_are_rounded_once(T, H, Hk, Dk, Dv):
    """Half a unit of bf16's 8 bits is 2^-8.  What is multiplied again holds two bf16
    parts, 2^-16 off, at most twice in a term (the values summed into a state, and the
    state), and the sums are fp32's, 2^-16 of the terms' magnitudes A: in all below
    2^-14 A, beside the result's own rounding, 2^-8 of it."""

    _case(test="attention_rounded_once", T=T, Dk=Dk, Dv=Dv)
    q, k, v, d, s, go, gs = _inputs(T, 2, H, Hk, Dk, Dv, "bf16")
    for state, gstate in ((s, gs), (None, None)):
        leaves = [t if t is None else t.detach().requires_grad_() for t in (q, k, v, state)]
        final, out = myelin.decay_attention(*leaves[:3], d, leaves[3])
        grads = (go,) if gstate is None else (go, gstate)
        got = torch.autograd.grad((out, final)[: len(grads)], leaves[:3], grads)
        args, scale = (q, k, v, d, state), Dk**-0.5
        want = _reference(*args, None, scale, go, gstate)
        ab = lambda t: None if t is None else t.abs()  # noqa: E731
        size = _reference(*(ab(t) for t in args), None, scale, go.abs(), ab(gstate))
        for name, a, w, z in zip(NAMES[1:], (out, *got), want[1:], size[1:]):
            tol = 2.0**-8 * w.abs() + 2.0**-14 * z
            assert bool(((a.detach().double().cpu() - w).abs() <= tol).all()), name
