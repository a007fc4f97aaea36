"""Log probabilities of given tokens (or classes), with entropy, top
alternatives and the gradient (``csrc/log_probs.hip``): the loss of a readout
while training, what it answers with afterwards."""

from __future__ import annotations

from typing import Any, NamedTuple

import torch

from myelin_amd import _lib, autograd
from myelin_amd.packing import _device_of

MAX_TOP = 64
_TYPES = (torch.float32, torch.bfloat16)


class TokenLogProbs(NamedTuple):
    """Results of :func:`token_log_probs`, float32, in the rows' shape."""

    log_probs: torch.Tensor | None
    entropy: torch.Tensor
    top_log_probs: torch.Tensor | None
    top_tokens: torch.Tensor | None


def _forward(x, targets, top, ignore_index):
    """(log_probs, entropy, stats, top_log_probs, top_tokens) of rows ``x [R, V]``."""

    R, V = x.shape
    dev = x.device
    log_probs = None if targets is None else torch.empty(R, dtype=torch.float32, device=dev)
    entropy = torch.empty(R, dtype=torch.float32, device=dev)
    stats = torch.empty((2, R), dtype=torch.float32, device=dev)
    top_lp = top_tok = None
    if top:
        top_lp = torch.empty((R, top), dtype=torch.float32, device=dev)
        top_tok = torch.empty((R, top), dtype=torch.int64, device=dev)
    need = _lib.load().myelin_token_log_probs_workspace_bytes(R, V, top)
    ws = torch.empty(need, dtype=torch.uint8, device=dev) if need else None
    with _device_of(x):
        _lib.call("myelin_token_log_probs", x.data_ptr(), _lib.DT[x.dtype], x.stride(0), _lib.ptr(targets),
                  ignore_index, _lib.ptr(log_probs), entropy.data_ptr(), stats.data_ptr(), _lib.ptr(top_lp),
                  _lib.ptr(top_tok), R, V, top, _lib.ptr(ws), need, _lib.stream(dev))
    return log_probs, entropy, stats, top_lp, top_tok


class HipTokenLogProbsFunction(torch.autograd.Function):
    """Saves the logits, by reference, and two numbers a row."""

    @staticmethod
    def forward(ctx: Any, x, targets, top, ignore_index):
        ctx.set_materialize_grads(False)
        log_probs, entropy, stats, top_lp, top_tok = _forward(x, targets, top, ignore_index)
        ctx.save_for_backward(x, targets, stats, entropy)
        ctx.ignore_index = ignore_index
        if top:
            ctx.mark_non_differentiable(top_lp, top_tok)
        return log_probs, entropy, top_lp, top_tok

    @staticmethod
    @autograd.differentiated_once
    def backward(ctx: Any, g_lp, g_ent, _g_top=None, _g_tok=None):
        if g_lp is None and g_ent is None:
            return None, None, None, None
        x, targets, stats, entropy = ctx.saved_tensors
        R, V = x.shape
        gx = torch.empty((R, V), dtype=x.dtype, device=x.device)
        g_lp, g_ent = (None if g is None else g.contiguous() for g in (g_lp, g_ent))
        with _device_of(x):
            _lib.call("myelin_token_log_probs_bwd", x.data_ptr(), _lib.DT[x.dtype], x.stride(0), _lib.ptr(targets),
                      ctx.ignore_index, stats.data_ptr(), entropy.data_ptr(), _lib.ptr(g_lp), _lib.ptr(g_ent),
                      gx.data_ptr(), R, V, _lib.stream(x.device))
        return gx, None, None, None


def token_log_probs(
    logits: torch.Tensor,
    targets: torch.Tensor | None = None,
    *,
    top: int = 0,
    ignore_index: int = -100,
) -> TokenLogProbs:
    """Log probabilities of ``targets`` under ``softmax(logits)``, entropies and
    the ``top`` most probable alternatives of each row.

    ``logits [..., V]`` float32 or bfloat16, ``targets [...]`` int64 or int32;
    without targets ``log_probs`` is ``None``, with ``top=0`` the alternatives
    are.  ``top`` is at most ``min(64, V)``; equal logits go to the lower index.
    ``log_probs`` and ``entropy`` are differentiable, the alternatives are not.

    A row whose target is ``ignore_index`` gives 0, 0, ``-inf`` and -1 and no
    gradient; any other target outside ``[0, V)`` gives NaN (nothing is read
    out of range).  Logits of ``-inf`` or a type's lowest value are masked
    tokens; a row of nothing but ``-inf`` has log probability ``-inf``, entropy
    0 and no gradient.
    """

    if logits.ndim == 0 or logits.shape[-1] == 0:
        raise ValueError(f"logits must be shaped [..., V] with V > 0; got {tuple(logits.shape)}")
    _lib.require_device(logits, "logits")
    if logits.dtype not in _TYPES:
        raise ValueError(f"logits must be float32 or bfloat16; got {logits.dtype}")
    lead, V = logits.shape[:-1], logits.shape[-1]
    if not 0 <= top <= min(MAX_TOP, V):
        raise ValueError(f"top must be in [0, min({MAX_TOP}, V)]; got {top} with V = {V}")
    if targets is not None:
        if targets.shape != lead:
            raise ValueError(f"targets must match logits.shape[:-1]; got {tuple(targets.shape)} and {tuple(lead)}")
        if targets.device != logits.device:
            raise ValueError("targets must be on the same device as logits")
        if targets.dtype not in (torch.int64, torch.int32):
            raise ValueError(f"targets must be int64 or int32; got {targets.dtype}")
        if targets.ndim != 1:
            targets = targets.reshape(-1)
        targets = targets.to(torch.int64).contiguous()
    x = logits if logits.ndim == 2 else logits.reshape(-1, V)
    if (x.shape[0] > 1 and x.stride(0) < V) or x.stride(1) != 1:
        x = x.contiguous()
    if autograd.plain(x):
        results = iter(autograd.native().token_log_probs(x, targets, top, ignore_index))
        log_probs = None if targets is None else next(results)
        entropy = next(results)
        top_lp, top_tok = (next(results), next(results)) if top else (None, None)
    else:
        log_probs, entropy, top_lp, top_tok = HipTokenLogProbsFunction.apply(x, targets, top, ignore_index)
    if len(lead) == 1:
        return TokenLogProbs(log_probs, entropy, top_lp, top_tok)
    return TokenLogProbs(
        None if log_probs is None else log_probs.view(lead),
        entropy.view(lead),
        None if top_lp is None else top_lp.view(*lead, top),
        None if top_tok is None else top_tok.view(*lead, top),
    )
