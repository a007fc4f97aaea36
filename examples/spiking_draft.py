"""A small draft model beside the spiking sequence model: distilled from its top
logits, then drafting tokens that the spiking model verifies.

    tokens -> TokenEmbedding -> GatedRecurrence -> logits

The spiking model looks at several drafted tokens a turn; those it agrees with are
taken, so that the result has its distribution (or, asked for the most probable
tokens, is what it gives alone).

    python examples/spiking_draft.py
"""

from __future__ import annotations

import pathlib
import sys

import torch
from torch import nn

sys.path.insert(0, str(pathlib.Path(__file__).resolve().parents[1]))

import myelin_amd as myelin  # noqa: E402
from examples.spiking_sequence import SpikingSequenceModel, sequences, train  # noqa: E402


class DraftModel(nn.Module):
    def __init__(self, tokens: int, width: int = 64) -> None:
        super().__init__()
        self.embedding = myelin.TokenEmbedding(tokens, width)
        self.memory = myelin.GatedRecurrence(width, width, taus=(2.0, 32.0))
        self.readout = myelin.LinearSynapse(width, tokens)
        for synapse in (self.memory.synapse, self.readout):
            fan_in = synapse.weight.shape[0]
            nn.init.uniform_(synapse.weight, -(3.0 / fan_in) ** 0.5, (3.0 / fan_in) ** 0.5)

    def forward(self, tokens: torch.Tensor, lengths: torch.Tensor | None = None) -> torch.Tensor:
        """Logits ``[T, B, tokens]`` of the next token, for ``tokens [T, B]``."""

        _, hidden = self.memory(self.embedding(tokens), lengths=lengths)
        return self.readout(hidden)

    def begin(self, batch: int, device) -> torch.Tensor:
        return torch.zeros(batch, self.memory.features, device=device)

    @torch.no_grad()
    def step(self, tokens: torch.Tensor, state: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
        """Logits ``[B, tokens]`` after one more token of each sample, and the state
        after it."""

        state, hidden = self.memory.step(self.embedding(tokens), state)
        return self.readout(hidden[None])[0], state


def distil(draft: DraftModel, teacher: SpikingSequenceModel, tokens: int, updates: int, steps: int = 64,
           batch: int = 32, top: int = 8, temperature: float = 1.0, device: str = "cuda") -> list[float]:
    """Losses of the updates: the divergence of the draft model from the teacher's
    ``top`` alternatives, over the steps that each sample has."""

    generator = torch.Generator().manual_seed(5)
    optimiser = torch.optim.Adam(draft.parameters(), lr=5e-3)
    teacher.eval()
    losses = []
    for _ in range(updates):
        data = sequences(tokens, steps, batch, generator).to(device)
        lengths = torch.randint(steps // 2, steps + 1, (batch,), generator=generator).to(device)
        past = torch.arange(steps, device=device)[:, None] >= lengths
        with torch.no_grad():
            # (a row whose target is ignored has no alternatives, and so no loss)
            offered = myelin.token_log_probs(teacher(data, lengths), data.masked_fill(past, -100), top=top)
        rows = myelin.distillation_loss(draft(data, lengths), offered.top_log_probs, offered.top_tokens,
                                        temperature=temperature)
        loss = rows.sum() / lengths.sum()
        optimiser.zero_grad()
        loss.backward()
        optimiser.step()
        losses.append(float(loss.detach()))
    return losses


def _pick(states: list[torch.Tensor], at: torch.Tensor) -> torch.Tensor:
    """Of a state after each step, each sample's after step ``at``."""

    return torch.stack(states)[at, torch.arange(at.numel(), device=at.device)]


@torch.no_grad()
def speculate(teacher: SpikingSequenceModel, draft: DraftModel, prompt: torch.Tensor, count: int, ahead: int = 4,
              greedy: bool = False, seed: int = 0) -> tuple[torch.Tensor, float]:
    """``count`` tokens after ``prompt [T, B]``, ``[count, B]``, and how many drafted
    tokens a turn were taken."""

    teacher.eval()
    device, batch = prompt.device, prompt.shape[1]
    generator = torch.Generator(device=device).manual_seed(seed)
    large, small = teacher.begin(batch, device), draft.begin(batch, device)
    for tokens in prompt[:-1]:
        _, large = teacher.step(tokens, large)
        _, small = draft.step(tokens, small)
    last = prompt[-1]
    out: list[list[int]] = [[] for _ in range(batch)]
    turns, taken = 0, 0
    while min(map(len, out)) < count:
        # the draft model goes ahead, one step more than it drafts
        drafted, chances, small_states, tokens = [], [], [], last
        for i in range(ahead + 1):
            logits, small = draft.step(tokens, small)
            small_states.append(small)
            if i == ahead:
                break
            if greedy:
                tokens = logits.argmax(-1)
            else:
                chances.append(torch.softmax(logits, -1))
                tokens = torch.multinomial(chances[-1], 1, generator=generator)[:, 0]
            drafted.append(tokens)
        # the large one takes the same steps
        rows, membranes, memories = [], [], []
        membrane, memory = large
        for tokens in (last, *drafted):
            logits, (membrane, memory) = teacher.step(tokens, (membrane, memory.clone()))
            rows.append(nn.functional.one_hot(logits.argmax(-1), logits.shape[-1]).float() if greedy
                        else torch.softmax(logits, -1))
            membranes.append(membrane.membrane)
            memories.append(memory)
        uniforms = torch.rand(ahead + 1, batch, generator=generator, device=device)
        result = myelin.verify_draft(torch.stack(rows), torch.stack(drafted), uniforms,
                                     None if greedy else torch.stack(chances))
        at = result.accepted
        last = result.tokens.gather(0, at[None])[0]
        large = (myelin.LIFState(_pick(membranes, at)), _pick(memories, at))
        small = _pick(small_states, at)
        for b, (n, tokens) in enumerate(zip(at.tolist(), result.tokens.t().tolist())):
            out[b] += tokens[: n + 1]
        turns += batch
        taken += int(at.sum())
    return torch.tensor([row[:count] for row in out]).t(), taken / turns


def main() -> None:
    tokens, device = 50, "cuda"
    torch.manual_seed(0)
    teacher = SpikingSequenceModel(tokens).to(device)
    print(f"teacher: loss {train(teacher, tokens, 200)[-1]:.3f}", flush=True)
    draft = DraftModel(tokens).to(device)
    losses = distil(draft, teacher, tokens, 150)
    print(f"draft: divergence {losses[0]:.3f} -> {losses[-1]:.3f}", flush=True)
    prompt = sequences(tokens, 8, 4, torch.Generator().manual_seed(2)).to(device)
    for greedy in (True, False):
        result, taken = speculate(teacher, draft, prompt, 24, greedy=greedy)
        print(f"{'most probable' if greedy else 'drawn'}: {taken:.2f} of 4 drafted tokens a turn taken")
        for b in range(prompt.shape[1]):
            print("  ", prompt[:, b].tolist(), "->", result[:, b].tolist())


if __name__ == "__main__":
    main()
