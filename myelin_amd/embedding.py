"""The embeddings of tokens, scaled, and the gradient of their table
(``csrc/embedding.hip``): what a sequence model reads its tokens with."""

from __future__ import annotations

import math
from typing import Any

import torch
from torch import nn

from myelin_amd import _lib, autograd
from myelin_amd.packing import _device_of

_TYPES = (torch.float32, torch.bfloat16)
NO_PADDING = -(2**63)  # for the kernels: no token is padding, this one neither


def _forward(tokens, weight, scale, padding):
    V, D = weight.shape
    M = tokens.numel()
    out = torch.empty((*tokens.shape, D), dtype=weight.dtype, device=weight.device)
    with _device_of(weight):
        _lib.call("myelin_token_embedding", tokens.data_ptr(), weight.data_ptr(), _lib.DT[weight.dtype],
                  weight.stride(0), out.data_ptr(), M, V, D, scale, padding, _lib.stream(weight.device))
    return out


class HipTokenEmbeddingFunction(torch.autograd.Function):
    """Saves the tokens, by reference, and nothing else."""

    @staticmethod
    def forward(ctx: Any, weight, tokens, scale, padding):
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(tokens)
        ctx.meta = (scale, padding, *weight.shape)
        return _forward(tokens, weight, scale, padding)

    @staticmethod
    @autograd.differentiated_once
    def backward(ctx: Any, g):
        if g is None:
            return (None,) * 4
        (tokens,) = ctx.saved_tensors
        scale, padding, V, D = ctx.meta
        M = tokens.numel()
        g = g.contiguous()
        gw = torch.empty((V, D), dtype=g.dtype, device=g.device)
        need = _lib.load().myelin_token_embedding_bwd_workspace_bytes(M, V, D)
        ws = torch.empty(need, dtype=torch.uint8, device=g.device) if need else None
        with _device_of(g):
            _lib.call("myelin_token_embedding_bwd", tokens.data_ptr(), g.data_ptr(), _lib.DT[g.dtype], gw.data_ptr(), M,
                      V, D, scale, padding, _lib.ptr(ws), need, _lib.stream(g.device))
        return gw, None, None, None


def token_embedding(
    tokens: torch.Tensor,
    weight: torch.Tensor,
    *,
    scale: float = 1.0,
    padding_index: int | None = None,
) -> torch.Tensor:
    """``scale * weight[tokens]``, a float32 product rounded to the weight's type: ``[..., D]``.

    ``tokens [...]`` int64 or int32, ``weight [V, D]`` float32 or bfloat16.  Tokens
    equal to ``padding_index`` (any number above -2^63, also one outside the table)
    give zeros and no gradient; any other token outside ``[0, V)`` gives a row of NaN
    and no gradient (nothing is read out of range).

    Differentiable in the weight.  A row's gradient is the float32 sum over its tokens,
    in an order that their positions alone decide (the same bits on every run),
    scaled and rounded once.
    """

    if weight.ndim != 2 or 0 in weight.shape:
        raise ValueError(f"weight must be shaped [V, D], neither 0; got {tuple(weight.shape)}")
    _lib.require_device(weight, "weight")
    if weight.dtype not in _TYPES:
        raise ValueError(f"weight must be float32 or bfloat16; got {weight.dtype}")
    if tokens.device != weight.device:
        raise ValueError("tokens must be on the same device as weight")
    if tokens.dtype not in (torch.int64, torch.int32):
        raise ValueError(f"tokens must be int64 or int32; got {tokens.dtype}")
    scale = float(scale)
    if not math.isfinite(scale) or abs(scale) > torch.finfo(torch.float32).max:
        raise ValueError(f"scale must be finite in float32; got {scale}")
    if padding_index is not None and not -(2**63) < padding_index < 2**63:
        raise ValueError(f"padding_index must fit 64 bits; got {padding_index}")
    padding = NO_PADDING if padding_index is None else padding_index
    if (weight.shape[0] > 1 and weight.stride(0) < weight.shape[1]) or (
            weight.stride(1) != 1 and weight.shape[1] > 1):
        weight = weight.contiguous()
    if autograd.plain(weight):
        return autograd.native().token_embedding(weight, tokens, scale, padding)
    return HipTokenEmbeddingFunction.apply(weight, tokens.to(torch.int64).contiguous(), scale, padding)


class TokenEmbedding(nn.Module):
    """A table of ``tokens`` embeddings of ``width``, drawn from a unit normal
    distribution as ``nn.Embedding``'s, looked up by :func:`token_embedding`."""

    def __init__(self, tokens: int, width: int, scale: float = 1.0, padding_index: int | None = None) -> None:
        super().__init__()
        self.scale = scale
        self.padding_index = padding_index
        self.weight = nn.Parameter(torch.randn(tokens, width))

    def forward(self, tokens: torch.Tensor) -> torch.Tensor:
        return token_embedding(tokens, self.weight, scale=self.scale, padding_index=self.padding_index)
