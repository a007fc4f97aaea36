"""Distillation from a teacher's top logits (``csrc/distillation.hip``): the loss
of a student that learns from the alternatives of another model, as
:func:`~myelin_amd.token_log_probs` gives them, and its gradient."""

from __future__ import annotations

import math
from typing import Any

import torch

from myelin_amd import _lib, autograd
from myelin_amd.packing import _device_of

MAX_TOP = 1024
_TYPES = (torch.float32, torch.bfloat16)


def _forward(x, values, tokens, temperature, keep):
    """(loss, probs, stats) of rows ``x [R, V]``; probs where a gradient is wanted."""

    R, V = x.shape
    K = tokens.shape[1]
    dev = x.device
    loss = torch.empty(R, dtype=torch.float32, device=dev)
    stats = torch.empty((2, R), dtype=torch.float32, device=dev)
    probs = torch.empty((R, K), dtype=torch.float32, device=dev) if keep else None
    need = _lib.load().myelin_distillation_loss_workspace_bytes(R, V)
    ws = torch.empty(need, dtype=torch.uint8, device=dev) if need else None
    with _device_of(x):
        _lib.call("myelin_distillation_loss", x.data_ptr(), _lib.DT[x.dtype], x.stride(0), values.data_ptr(),
                  tokens.data_ptr(), temperature, loss.data_ptr(), _lib.ptr(probs), stats.data_ptr(), R, V, K,
                  _lib.ptr(ws), need, _lib.stream(dev))
    return loss, probs, stats


class HipDistillationLossFunction(torch.autograd.Function):
    """Saves the logits and the teacher's tokens, by reference, the teacher's
    probabilities and two numbers a row."""

    @staticmethod
    def forward(ctx: Any, x, values, tokens, temperature):
        ctx.set_materialize_grads(False)
        loss, probs, stats = _forward(x, values, tokens, temperature, ctx.needs_input_grad[0])
        ctx.save_for_backward(x, tokens, probs, stats)
        ctx.temperature = temperature
        return loss

    @staticmethod
    @autograd.differentiated_once
    def backward(ctx: Any, g):
        if g is None:
            return (None,) * 4
        x, tokens, probs, stats = ctx.saved_tensors
        R, V = x.shape
        gx = torch.empty((R, V), dtype=x.dtype, device=x.device)
        g = g.contiguous()
        with _device_of(x):
            _lib.call("myelin_distillation_loss_bwd", x.data_ptr(), _lib.DT[x.dtype], x.stride(0), tokens.data_ptr(),
                      probs.data_ptr(), stats.data_ptr(), g.data_ptr(), ctx.temperature, gx.data_ptr(), R, V,
                      tokens.shape[1], _lib.stream(x.device))
        return gx, None, None, None


def distillation_loss(
    logits: torch.Tensor,
    teacher_logits: torch.Tensor,
    teacher_tokens: torch.Tensor,
    *,
    temperature: float = 1.0,
) -> torch.Tensor:
    """``sum_k p_k (log p_k - log q[token_k])`` of each row, float32 in the rows'
    shape: the divergence of the student's ``q = softmax(logits / temperature)``
    from the teacher's ``p = softmax(teacher_logits / temperature)`` over its
    ``K`` tokens.

    ``logits [..., V]`` float32 or bfloat16; ``teacher_logits [..., K]`` float32 or
    bfloat16, up to a constant of the row (log probabilities are as good), a
    constant of the training; ``teacher_tokens [..., K]`` int64 or int32, in any
    order, ``K`` at most 1024.  ``token_log_probs(..., top=K)`` gives both.
    Differentiable in the logits.

    A place of token -1 or value ``-inf`` is empty; a row of empty places (one
    whose target was ignored) is not read and gives 0 and no gradient.  Other
    tokens outside ``[0, V)`` make the row's loss and gradient NaN (nothing is read
    out of range).  A token named twice counts twice.  Logits of ``-inf`` are
    masked tokens: the loss is ``+inf`` where the teacher gives one of them a
    probability; a row of nothing but ``-inf`` has loss ``+inf`` and no gradient.
    """

    if logits.ndim == 0 or logits.shape[-1] == 0:
        raise ValueError(f"logits must be shaped [..., V] with V > 0; got {tuple(logits.shape)}")
    _lib.require_device(logits, "logits")
    if logits.dtype not in _TYPES or teacher_logits.dtype not in _TYPES:
        raise ValueError(f"logits and teacher_logits must be float32 or bfloat16; got {logits.dtype} and "
                         f"{teacher_logits.dtype}")
    lead, V = logits.shape[:-1], logits.shape[-1]
    if teacher_logits.ndim != logits.ndim or teacher_logits.shape[:-1] != lead:
        raise ValueError(f"teacher_logits must be shaped [..., K] with the rows of logits; got "
                         f"{tuple(teacher_logits.shape)} and {tuple(logits.shape)}")
    K = teacher_logits.shape[-1]
    if not 1 <= K <= MAX_TOP:
        raise ValueError(f"teacher_logits must have [1, {MAX_TOP}] places a row; got {K}")
    if teacher_tokens.shape != teacher_logits.shape:
        raise ValueError(f"teacher_tokens must match teacher_logits; got {tuple(teacher_tokens.shape)} and "
                         f"{tuple(teacher_logits.shape)}")
    if teacher_logits.device != logits.device or teacher_tokens.device != logits.device:
        raise ValueError("teacher_logits and teacher_tokens must be on the same device as logits")
    if teacher_tokens.dtype not in (torch.int64, torch.int32):
        raise ValueError(f"teacher_tokens must be int64 or int32; got {teacher_tokens.dtype}")
    if teacher_logits.requires_grad:
        raise ValueError("the teacher is a constant and has no gradient; pass teacher_logits detached")
    autograd.refuse_tangents("distillation_loss", teacher_logits)
    temperature = float(temperature)
    if not (2.0**-64 <= temperature <= 2.0**64):
        raise ValueError(f"temperature must be positive and finite, within 2**-64 and 2**64; got {temperature}")
    if autograd.plain(logits):
        return autograd.native().distillation_loss(logits, teacher_logits, teacher_tokens, temperature)
    values = teacher_logits.reshape(-1, K).float().contiguous()
    tokens = teacher_tokens.reshape(-1, K).to(torch.int64).contiguous()
    x = logits if logits.ndim == 2 else logits.reshape(-1, V)
    if (x.shape[0] > 1 and x.stride(0) < V) or x.stride(1) != 1:
        x = x.contiguous()
    loss = HipDistillationLossFunction.apply(x, values, tokens, temperature)
    return loss if len(lead) == 1 else loss.view(lead)
