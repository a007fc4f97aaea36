"""A draft model's operators together, as examples/spiking_draft.py uses them beside
the spiking sequence model."""

from __future__ import annotations

import pytest
import torch

import myelin_amd as myelin
from examples.spiking_draft import DraftModel, distil, speculate
from examples.spiking_sequence import SpikingSequenceModel, generate, sequences

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _models(tokens):
    torch.manual_seed(0)
    return SpikingSequenceModel(tokens, width=64).to(DEV), DraftModel(tokens, width=32).to(DEV)


def test_distillation_runs_and_reaches_every_parameter():
    print("case: test=spiking_draft_train", flush=True)
    teacher, draft = _models(20)
    before = [p.detach().clone() for p in draft.parameters()]
    losses = distil(draft, teacher, 20, updates=3, steps=24, batch=8, top=5, temperature=2.0)
    assert len(losses) == 3 and all(torch.isfinite(torch.tensor(losses)))
    for p, old in zip(draft.parameters(), before):
        assert p.grad is not None and bool(p.grad.isfinite().all()) and bool(p.grad.any())
        assert not torch.equal(p, old)
    assert all(p.grad is None for p in teacher.parameters())


def test_gradients_are_those_of_plain_torch():
    """The model's loss in float64 from the formulas.  Its fp32 gradients are sums of
    some thousand products; 1e-4 of a tensor's largest is a hundred times what their
    roundings come to."""

    print("case: test=spiking_draft_gradients", flush=True)
    _, draft = _models(20)
    T, B, K = 12, 3, 4
    g = torch.Generator().manual_seed(2)
    data = torch.randint(0, 20, (T, B), generator=g).to(DEV)
    lengths = torch.tensor([12, 5, 0], device=DEV)
    values = torch.randn(T, B, K, generator=g).to(DEV)
    alternatives = torch.rand(T, B, 20, generator=g).argsort(-1)[..., :K].to(DEV)
    past = torch.arange(T, device=DEV)[:, None] >= lengths
    alternatives = torch.where(past[..., None], -1, alternatives)
    loss = myelin.distillation_loss(draft(data, lengths), values, alternatives, temperature=1.5).sum()
    grads = torch.autograd.grad(loss, list(draft.parameters()))

    leaves = {n: p.detach().double().cpu().requires_grad_() for n, p in draft.named_parameters()}
    x = leaves["embedding.weight"][data.cpu()]
    both = x @ leaves["memory.synapse.weight"] + leaves["memory.synapse.bias"]
    u, gate = both.split(32, -1)
    h, rows = torch.zeros(B, 32, dtype=torch.float64), []
    for t in range(T):
        a = torch.sigmoid(gate[t])
        on = (lengths.cpu() > t)[:, None]
        h = torch.where(on, a * h + (1 - a) * u[t], h)
        rows.append(torch.where(on, h, 0.0))
    logits = torch.stack(rows) @ leaves["readout.weight"] + leaves["readout.bias"]
    log_q = torch.log_softmax(logits / 1.5, -1)
    p = torch.softmax(values.double().cpu() / 1.5, -1)
    picked = log_q.gather(-1, alternatives.cpu().clamp(min=0))
    want = (p * (p.log() - picked)).sum(-1)[~past.cpu()].sum()
    assert abs(loss.item() - want.item()) <= 1e-5 * abs(want.item())
    for (n, leaf), got in zip(leaves.items(), grads):
        (w,) = torch.autograd.grad(want, leaf, retain_graph=True)
        assert float((got.double().cpu() - w).abs().max()) <= 1e-4 * float(w.abs().max()), n


def test_the_most_probable_tokens_are_the_teacher_s_own():
    """Whatever the draft model drafts, and however many of it are taken."""

    print("case: test=spiking_draft_greedy", flush=True)
    teacher, draft = _models(20)
    prompt = sequences(20, 6, 5, torch.Generator().manual_seed(3)).to(DEV)
    want, _ = generate(teacher, prompt, 12)
    got, _ = speculate(teacher, draft, prompt, 12, ahead=3, greedy=True)
    assert torch.equal(got, want.cpu())


def test_drawn_tokens_are_tokens():
    print("case: test=spiking_draft_drawn", flush=True)
    teacher, draft = _models(20)
    prompt = sequences(20, 6, 5, torch.Generator().manual_seed(3)).to(DEV)
    got, taken = speculate(teacher, draft, prompt, 10, ahead=3)
    assert got.shape == (10, 5) and bool(((got >= 0) & (got < 20)).all()) and 0.0 <= taken <= 3.0
    again, _ = speculate(teacher, draft, prompt, 10, ahead=3)
    assert torch.equal(got, again)


def test_steps_give_the_sequence_s_logits():
    """(The projections of 5 rows and of 100 may differ in their sums' last bits.)"""

    print("case: test=spiking_draft_steps", flush=True)
    _, draft = _models(20)
    data = sequences(20, 20, 5, torch.Generator().manual_seed(4)).to(DEV)
    with torch.no_grad():
        whole = draft(data)
        state, rows = draft.begin(5, DEV), []
        for tokens in data:
            logits, state = draft.step(tokens, state)
            rows.append(logits)
    assert float((torch.stack(rows) - whole).abs().max()) <= 1e-5 * float(whole.abs().max())
