"""A draft model's operators in every way that they are called: tensor subclasses
(the Python Functions) against plain tensors (the C++ ones), second derivatives and
transforms that are refused, a compiled caller, captured graphs, other streams."""

from __future__ import annotations

import pytest
import torch
from torch.autograd import forward_ad

import myelin_amd as myelin

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _case(**kw):
    print("case:", " ".join(f"{k}={v}" for k, v in kw.items()), flush=True)


class Sub(torch.Tensor):
    pass


def _leaf(*shape, seed=0):
    g = torch.Generator().manual_seed(seed + len(shape) + sum(shape))
    return torch.randn(*shape, generator=g).to(DEV)


def _recurrence(x, gate, s):
    return myelin.gated_recurrence(x, gate, s, lengths=torch.full((2,), x.shape[0] - 5, device=x.device))


def _embedding(w):
    return (myelin.token_embedding(torch.arange(200, device=w.device).view(50, 4) % 7, w, scale=2.0, padding_index=3),)


def _distillation(x):
    tokens = torch.arange(24, device=x.device).view(6, 4)
    return (myelin.distillation_loss(x, (tokens % 5).float(), tokens, temperature=1.5),)


CASES = {
    "recurrence": (_recurrence, [(70, 2, 24), (70, 2, 24), (2, 24)]),
    "recurrence_long": (_recurrence, [(5000, 2, 3), (5000, 2, 3), (2, 3)]),
    "embedding": (_embedding, [(7, 40)]),
    "distillation": (_distillation, [(6, 2000)]),
    "distillation_wide": (_distillation, [(6, 50000)]),
}


@pytest.mark.parametrize("name", CASES)
def test_subclasses_give_the_same_bits(name):
    _case(test="draft_functions", name=name)
    f, shapes = CASES[name]
    leaves = [_leaf(*s, seed=i) for i, s in enumerate(shapes)]
    results = []
    for kind in (torch.Tensor, Sub):
        xs = [t.detach().clone().as_subclass(kind).requires_grad_() for t in leaves]
        with torch.no_grad():
            quiet = f(*xs)
        outs = f(*xs)
        grads = torch.autograd.grad(outs, xs, [torch.ones_like(o) * 0.5 for o in outs])
        # a part of the gradients
        alone = [torch.autograd.grad(f(*[t if j == i else t.detach() for j, t in enumerate(xs)])[-1].sum(), x)[0]
                 for i, x in enumerate(xs)]
        results.append([torch.Tensor(t.detach()) for t in (*quiet, *outs, *grads, *alone)])
        g = torch.autograd.grad(f(*xs)[0].sum(), xs[0], create_graph=True)[0]
        with pytest.raises(RuntimeError, match="once_differentiable"):
            g.sum().backward()
    assert len(results[0]) == len(results[1])
    for a, b in zip(*results):
        assert torch.equal(a, b)


def test_verified_subclasses():
    p = torch.softmax(_leaf(4, 3, 500), -1)
    t, u = torch.randint(0, 500, (3, 3), device=DEV), torch.rand(4, 3, device=DEV)
    a, b = myelin.verify_draft(p, t, u, p[:3]), myelin.verify_draft(p.as_subclass(Sub), t, u, p[:3])
    assert torch.equal(a.tokens, torch.Tensor(b.tokens).long()) and torch.equal(a.accepted, torch.Tensor(b.accepted).long())
    # probabilities that come out of a model with gradients
    c = myelin.verify_draft(p.clone().requires_grad_(), t, u, p[:3].clone().requires_grad_())
    assert torch.equal(a.tokens, c.tokens) and not c.tokens.requires_grad


@pytest.mark.parametrize("name", CASES)
def test_forward_mode(name):
    _case(test="draft_forward_mode", name=name)
    f, shapes = CASES[name]
    xs = [_leaf(*s, seed=i).requires_grad_() for i, s in enumerate(shapes)]

    def result():
        outs = f(*xs)
        return [t.detach() for t in (*outs, *torch.autograd.grad(outs, xs, [torch.ones_like(o) for o in outs]))]

    want = result()
    with forward_ad.dual_level():
        for a, b in zip(want, result()):
            assert torch.equal(a, b)
        for i, x in enumerate(xs):
            dual = [forward_ad.make_dual(x, torch.ones_like(x)) if j == i else t for j, t in enumerate(xs)]
            with pytest.raises(NotImplementedError, match="jvp"):
                f(*dual)


@pytest.mark.parametrize("grad", [False, True])
@pytest.mark.parametrize("name", CASES)
def test_a_compiled_caller(name, grad):
    """The graph breaks at the operators; nothing changes."""

    _case(test="draft_compiled", name=name, grad=grad)
    f, shapes = CASES[name]
    xs = [_leaf(*s, seed=i).requires_grad_(grad) for i, s in enumerate(shapes)]
    torch._dynamo.reset()
    compiled = torch.compile(lambda *a: [o * 2 for o in f(*a)], backend="eager")
    outs, got = f(*xs), compiled(*xs)
    for a, b in zip(outs, got):
        assert torch.equal(a * 2, b)
    if grad:
        want = torch.autograd.grad(outs, xs, [torch.full_like(a, 2.0) for a in outs])
        for a, b in zip(want, torch.autograd.grad(got, xs, [torch.ones_like(b) for b in got])):
            assert torch.equal(a, b)


def _everything(xs):
    """One pass through all of them: results that depend on every input."""

    x, gate, s, w, logits = xs
    state, out = _recurrence(x, gate, s)
    (rows,) = _embedding(w)
    (loss,) = _distillation(logits)
    grads = torch.autograd.grad((state, out, rows, loss), xs, [torch.ones_like(t) for t in (state, out, rows, loss)])
    p = torch.softmax(logits.detach(), -1).view(3, 2, -1)
    tokens = torch.arange(4, device=x.device).view(2, 2) * 3
    u = (s.detach()[:2, :3].t().contiguous().sigmoid() * 0.5).contiguous()
    v = myelin.verify_draft(p, tokens, u, torch.roll(p[:2], 1, 0))
    step_state, step_out = myelin.gated_recurrence_step(x.detach()[0], gate.detach()[0], s.detach())
    return [t.detach() for t in (state, out, rows, loss, *grads, v.accepted, v.tokens, step_state, step_out)]


def _inputs(T=300, V=20000, seed=0):
    g = torch.Generator().manual_seed(seed)
    shapes = [(T, 2, 24), (T, 2, 24), (2, 24), (7, 40), (6, V)]
    return [torch.randn(*s, generator=g).to(DEV).requires_grad_() for s in shapes]


@pytest.mark.parametrize("T,V", [(300, 3000), (6000, 60000)])
def test_captured_and_replayed(T, V):
    """Every replay, with the program's own work between them, gives the eager bits
    of the inputs that are there then; two graphs with workspaces of one pool do not
    disturb each other."""

    _case(test="draft_graph", T=T, V=V)
    xs = _inputs(T, V)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            _everything(xs)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    first, second = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(first):
        got = _everything(xs)
    with torch.cuda.graph(second, pool=first.pool()):
        other = _everything(xs)
    for rep in range(4):
        with torch.no_grad():
            for t, new in zip(xs, _inputs(T, V, seed=rep)):
                t.copy_(new)
        want = _everything(xs)
        torch.cuda.synchronize()
        first.replay()
        kept = [t.clone() for t in got]
        second.replay()
        torch.cuda.synchronize()
        for i, (a, b, c) in enumerate(zip(want, kept, other)):
            assert torch.equal(a, b) and torch.equal(a, c), (rep, i)
        torch.randn(1000, 1000, device=DEV).sum().item()


def test_two_streams_at_once():
    _case(test="draft_streams")
    sets = [_inputs(3000, 30000, seed=i) for i in range(2)]
    want = [_everything(xs) for xs in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    got = [[], []]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(_everything(sets[i]))
    torch.cuda.synchronize()
    for i in range(2):
        for run in got[i]:
            assert all(torch.equal(a, b) for a, b in zip(run, want[i]))


def test_the_same_bits_on_every_run():
    xs = _inputs(5000, 40000, seed=7)
    want = _everything(xs)
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(_everything(xs), want))


def test_losses_in_the_rows_shape_may_be_changed_in_place():
    g = torch.Generator().manual_seed(3)
    logits, teacher = torch.randn(4, 3, 50, generator=g), torch.randn(4, 3, 5, generator=g)
    tokens = torch.randint(0, 50, (4, 3, 5), generator=g).to(DEV)
    mask = (torch.arange(12) % 3 > 0).float().view(4, 3).to(DEV)
    for lead in ((4, 3), (12,), (2, 2, 3), (4, 3, 1)):
        x = logits.to(DEV).view(*lead, 50).clone().requires_grad_()
        loss = myelin.distillation_loss(x, teacher.to(DEV).view(*lead, 5), tokens.view(*lead, 5))
        assert loss.shape == lead
        loss.mul_(mask.view(lead))
        loss.sum().backward()
        y = logits.to(DEV).view(12, 50).clone().requires_grad_()
        rows = myelin.distillation_loss(y, teacher.to(DEV).view(12, 5), tokens.view(12, 5))
        rows.backward(mask.view(12))
        assert torch.equal(x.grad.view(12, 50), y.grad)
    one = logits[0, 0].to(DEV).requires_grad_()
    loss = myelin.distillation_loss(one, teacher[0, 0].to(DEV), tokens[0, 0])
    assert loss.shape == ()
    loss.backward()
    assert one.grad.shape == (50,)
    # rows that are not one after the other in memory
    wide = logits.to(DEV).transpose(0, 1).clone().transpose(0, 1).requires_grad_()
    myelin.distillation_loss(wide, teacher.to(DEV), tokens).sum().backward()
    flat = logits.to(DEV).requires_grad_()
    myelin.distillation_loss(flat, teacher.to(DEV), tokens).sum().backward()
    assert torch.equal(wide.grad, flat.grad)
