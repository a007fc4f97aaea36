"""The sequence-model operators together, as examples/spiking_sequence.py uses
them beside the LIF layer."""

from __future__ import annotations

import math

import pytest
import torch

from examples.spiking_sequence import SpikingSequenceModel, generate, sequences, train

pytestmark = pytest.mark.gpu
DEV = "cuda"


def test_training_lowers_the_loss_and_generation_follows_the_cycle():
    print("case: test=spiking_sequence_train", flush=True)
    torch.manual_seed(0)
    tokens = 20
    model = SpikingSequenceModel(tokens, width=64).to(DEV)
    losses = train(model, tokens, 120, steps=40, batch=32)
    assert losses[0] > 0.8 * math.log(tokens)
    # nineteen steps of twenty follow the cycle: an entropy of 0.35 nats
    assert sum(losses[-10:]) / 10 < 0.5 * math.log(tokens)
    prompt = sequences(tokens, 6, 4, torch.Generator().manual_seed(3)).to(DEV)
    chosen, offered = generate(model, prompt, 10)
    assert chosen.shape == (10, 4) and offered.shape == (10, 4, 3)
    cycle = torch.randperm(tokens, generator=torch.Generator().manual_seed(0)).tolist()
    follows = {a: b for a, b in zip(cycle, cycle[1:] + cycle[:1])}
    rows = [prompt[-1].tolist()] + chosen.tolist()
    right = sum(follows[a] == b for x, y in zip(rows, rows[1:]) for a, b in zip(x, y))
    assert right >= 30  # of 40; by chance 2


def test_steps_give_the_sequence_s_logits():
    """A spike may flip where the two ways' currents differ in their last bits:
    nearly all rows agree to rounding."""

    print("case: test=spiking_sequence_steps", flush=True)
    torch.manual_seed(1)
    model = SpikingSequenceModel(30, width=64).to(DEV).eval()
    data = sequences(30, 50, 5, torch.Generator().manual_seed(4)).to(DEV)
    with torch.no_grad():
        whole = model(data)
        states = model.begin(5, DEV)
        rows = []
        for tokens in data:
            logits, states = model.step(tokens, states)
            rows.append(logits)
    err = (torch.stack(rows) - whole).abs().amax(-1)
    assert float((err <= 1e-4 * float(whole.abs().max())).float().mean()) >= 0.9
