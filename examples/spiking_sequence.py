"""A small spiking sequence model: trained on whole sequences, then asked for
tokens one at a time.

    embedding -> LinearSurrogateLIF -> q, k, v -> DecayAttention -> projection
              -> CounterDropout (+ spikes) -> logits -> token_log_probs

The LIF layer's leak and the attention's decays are the model's memory: training
and the prompt run over all time steps at once, generation carries the membrane
and the attention's states from step to step.

    python examples/spiking_sequence.py
"""

from __future__ import annotations

import pathlib
import sys

import torch
from torch import nn

sys.path.insert(0, str(pathlib.Path(__file__).resolve().parents[1]))

import myelin_amd as myelin  # noqa: E402


class SpikingSequenceModel(nn.Module):
    def __init__(self, tokens: int, width: int = 128, heads: int = 4, kv_heads: int = 2, key: int = 16,
                 value: int = 32, dropout: float = 0.1) -> None:
        super().__init__()
        self.shapes = [(heads, key), (kv_heads, key), (kv_heads, value)]
        self.embedding = nn.Embedding(tokens, width)
        self.hidden = myelin.LinearSurrogateLIF(width, width, surrogate=myelin.fast_sigmoid_surrogate,
                                                surrogate_slope=5.0, stream_synapse=True)
        self.qkv = myelin.LinearSynapse(width, sum(h * d for h, d in self.shapes))
        self.attention = myelin.DecayAttention([4.0 * 4.0**i for i in range(heads)])
        self.project = myelin.LinearSynapse(heads * value, width)
        self.dropout = myelin.CounterDropout(dropout, seed=1)
        self.readout = myelin.LinearSynapse(width, tokens)
        for synapse in (self.hidden.synapse, self.qkv, self.project, self.readout):
            fan_in = synapse.weight.shape[0]
            nn.init.uniform_(synapse.weight, -(3.0 / fan_in) ** 0.5, (3.0 / fan_in) ** 0.5)

    def heads(self, spikes: torch.Tensor) -> list[torch.Tensor]:
        """Queries, keys and values: views of one projection."""

        parts = self.qkv(spikes).split([h * d for h, d in self.shapes], -1)
        return [p.unflatten(-1, shape) for p, shape in zip(parts, self.shapes)]

    def answer(self, spikes: torch.Tensor, mixed: torch.Tensor) -> torch.Tensor:
        return self.readout(self.dropout(self.project(mixed.flatten(-2)), spikes))

    def forward(self, tokens: torch.Tensor, lengths: torch.Tensor | None = None) -> torch.Tensor:
        """Logits ``[T, B, tokens]`` of the next token, for ``tokens [T, B]``."""

        spikes = self.hidden(self.embedding(tokens))
        _, mixed = self.attention(*self.heads(spikes), lengths=lengths)
        return self.answer(spikes, mixed)

    def begin(self, batch: int, device) -> tuple[myelin.LIFState, torch.Tensor]:
        """The states before the first token."""

        (heads, key), (_, _), (_, value) = self.shapes
        width = self.embedding.embedding_dim
        return (myelin.LIFState(torch.zeros(batch, width, device=device)),
                torch.zeros(batch, heads, key, value, device=device))

    @torch.no_grad()
    def step(self, tokens: torch.Tensor, states) -> tuple[torch.Tensor, tuple]:
        """Logits ``[B, tokens]`` after one more token of each sample, and the
        states after it (the attention's is updated in place)."""

        membrane, memory = states
        cell = self.hidden.unroll.cell
        membrane, spikes = myelin.surrogate_lif_forward(
            self.hidden.synapse(self.embedding(tokens)[None]), membrane, cell.params,
            surrogate=myelin.surrogate_name(cell.surrogate), surrogate_slope=cell.surrogate_slope)
        q, k, v = (t[0] for t in self.heads(spikes))
        memory, mixed = self.attention.step(q, k, v, memory, out_state=memory)
        return self.answer(spikes, mixed[None])[0], (membrane, memory)


def sequences(tokens: int, steps: int, batch: int, generator: torch.Generator) -> torch.Tensor:
    """``[steps, batch]`` tokens that step through a fixed cycle of all of them,
    with a random jump now and then."""

    cycle = torch.randperm(tokens, generator=torch.Generator().manual_seed(0))
    place = torch.randint(0, tokens, (batch,), generator=generator)
    rows = []
    for _ in range(steps):
        jump = torch.rand(batch, generator=generator) < 0.05
        place = torch.where(jump, torch.randint(0, tokens, (batch,), generator=generator), (place + 1) % tokens)
        rows.append(cycle[place])
    return torch.stack(rows)


def train(model: SpikingSequenceModel, tokens: int, updates: int, steps: int = 64, batch: int = 32,
          device: str = "cuda") -> list[float]:
    """Losses of the updates: mean negative log probability of the next token,
    less a little entropy; samples end at lengths of their own."""

    generator = torch.Generator().manual_seed(1)
    optimiser = torch.optim.Adam(model.parameters(), lr=3e-3)
    losses = []
    for _ in range(updates):
        data = sequences(tokens, steps + 1, batch, generator).to(device)
        lengths = torch.randint(steps // 2, steps + 1, (batch,), generator=generator).to(device)
        past = torch.arange(steps, device=device)[:, None] >= lengths
        targets = data[1:].masked_fill(past, -100)
        result = myelin.token_log_probs(model(data[:-1], lengths), targets)
        loss = -(result.log_probs.sum() + 1e-3 * result.entropy.sum()) / lengths.sum()
        optimiser.zero_grad()
        loss.backward()
        optimiser.step()
        losses.append(float(loss.detach()))
    return losses


@torch.no_grad()
def generate(model: SpikingSequenceModel, prompt: torch.Tensor, count: int, alternatives: int = 3):
    """``count`` most probable tokens after ``prompt [T, B]``, with the log
    probabilities of each step's alternatives: ``[count, B]``, ``[count, B,
    alternatives]``."""

    model.eval()
    states = model.begin(prompt.shape[1], prompt.device)
    for tokens in prompt:
        logits, states = model.step(tokens, states)
    chosen, offered = [], []
    for _ in range(count):
        result = myelin.token_log_probs(logits, top=alternatives)
        tokens = result.top_tokens[:, 0]
        chosen.append(tokens)
        offered.append(result.top_log_probs)
        logits, states = model.step(tokens, states)
    return torch.stack(chosen), torch.stack(offered)


def main() -> None:
    tokens, device = 50, "cuda"
    torch.manual_seed(0)
    model = SpikingSequenceModel(tokens).to(device)
    losses = train(model, tokens, 200)
    for i in range(0, len(losses), 40):
        print(f"update {i:4d}  loss {losses[i]:.3f}", flush=True)
    print(f"update {len(losses) - 1:4d}  loss {losses[-1]:.3f}", flush=True)
    prompt = sequences(tokens, 8, 2, torch.Generator().manual_seed(2)).to(device)
    chosen, offered = generate(model, prompt, 12)
    for b in range(prompt.shape[1]):
        print("prompt", prompt[:, b].tolist(), "->", chosen[:, b].tolist())
        print("  first step's alternatives:", [f"{p:.2f}" for p in offered[0, b].exp().tolist()])


if __name__ == "__main__":
    main()
