"""token_embedding at the ends of the 64-bit numbers: padding is a number that was
given, and without one no token is padding."""

from __future__ import annotations

import pytest
import torch

import myelin_amd as myelin

pytestmark = pytest.mark.gpu
DEV = "cuda"
LEAST, MOST = -(2**63), 2**63 - 1


@pytest.mark.parametrize("padding", [None, 0, -1, MOST, -MOST])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V,D", [(7, 5), (300, 64), (5000, 200)])
def test_tokens_at_the_ends_of_the_numbers(V, D, dtype, padding):
    """Small tables, a workgroup to a position, and a sort."""

    for repeat in (1, 2000):
        print(f"case: test=embedding_numbers V={V} D={D} dtype={dtype} padding={padding} repeat={repeat}", flush=True)
        weight = torch.randn(V, D, device=DEV).to(dtype).requires_grad_()
        tokens = torch.tensor([LEAST, 0, -1, V - 1, V, MOST, -MOST, 2], device=DEV).repeat(repeat)
        y = myelin.token_embedding(tokens, weight, scale=2.0, padding_index=padding)
        hole = torch.zeros_like(tokens, dtype=torch.bool) if padding is None else tokens == padding
        inside = (tokens >= 0) & (tokens < V) & ~hole
        rows = weight.detach()[tokens.clamp(0, V - 1)] * 2  # exact
        assert torch.equal(y[inside], rows[inside]) and not bool(y[hole].any())
        assert bool(y[~inside & ~hole].isnan().all())
        # ones: sums of whole numbers, 2 or 4000 = 125 * 2^5, exact in both types
        (g,) = torch.autograd.grad(y, weight, torch.ones_like(y))
        count = torch.bincount(tokens[inside], minlength=V).float()
        assert torch.equal(g, (2.0 * count).to(dtype)[:, None].expand(V, D))
