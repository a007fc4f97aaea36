"""Verification of drafted tokens (``csrc/verification.hip``): a small model drafts
some tokens, the large one looks at all of them at once, and those that it agrees
with are taken, so that the result has the large model's distribution."""

from __future__ import annotations

import ctypes
from typing import NamedTuple

import torch

from myelin_amd import _lib, autograd
from myelin_amd.packing import _device_of

_TYPES = (torch.float32, torch.bfloat16)


class VerifiedTokens(NamedTuple):
    """Results of :func:`verify_draft`, int64."""

    accepted: torch.Tensor
    tokens: torch.Tensor


def _verify(target, draft, tokens, uniforms, lengths):
    rows, B, V = target.shape
    dev = target.device
    accepted = torch.empty(B, dtype=torch.int64, device=dev)
    out = torch.empty((rows, B), dtype=torch.int64, device=dev)
    strides = [*target.stride()[:2], *(draft.stride()[:2] if draft is not None else (0, 0))]
    need = _lib.load().myelin_verify_draft_workspace_bytes(B, V)
    ws = torch.empty(need, dtype=torch.uint8, device=dev) if need else None
    with _device_of(target):
        _lib.call("myelin_verify_draft", target.data_ptr(), _lib.ptr(draft), _lib.DT[target.dtype],
                  (ctypes.c_int64 * 4)(*strides), tokens.data_ptr(), uniforms.data_ptr(), _lib.ptr(lengths),
                  accepted.data_ptr(), out.data_ptr(), rows - 1, B, V, _lib.ptr(ws), need, _lib.stream(dev))
    return accepted, out


def _rows(t: torch.Tensor) -> torch.Tensor:
    """``t`` with unit stride in its last dimension."""

    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


def verify_draft(
    target_probs: torch.Tensor,
    draft_tokens: torch.Tensor,
    uniforms: torch.Tensor,
    draft_probs: torch.Tensor | None = None,
    *,
    lengths: torch.Tensor | None = None,
) -> VerifiedTokens:
    """Which of ``n`` drafted tokens of each sequence are taken, and the token after
    them.

    Time-major: ``target_probs [n + 1, B, V]`` are the target's probabilities before
    each drafted token and after the last, ``draft_probs [n, B, V]`` those that the
    drafted tokens were drawn from (``None``: they were chosen, not drawn), float32
    or bfloat16, any strides; ``draft_tokens [n, B]`` int64 or int32; ``uniforms
    [n + 1, B]`` float32 in [0, 1).  ``lengths [B]`` (int32 or int64 on the device,
    taken into [0, n]) gives each sequence's drafted tokens; later ones are not read.

    Token ``i`` is taken while ``uniforms[i] * draft_probs[i, token] <
    target_probs[i, token]``.  The first that is not is replaced by a draw from
    ``max(target_probs[i] - draft_probs[i], 0)``; where all are taken the next is a
    draw from the target's row after them.  A draw with ``u = uniforms[n]`` is the
    lowest token whose cumulative weight is above ``u`` times the sum of all.  All of
    it is computed in float64.

    Returns ``accepted [B]`` and ``tokens [n + 1, B]``: the taken tokens, the drawn
    one, then -1.

    Weights that are not positive and finite (NaN among them) count as 0.  Where
    nothing is left after a refusal the draw is from the target's row; where that
    has nothing either, the token is -1.  A drafted token outside ``[0, V)`` is
    refused, nothing is read out of range.  Numbers ``u`` that are not below 1 draw
    the last token with a weight.
    """

    if target_probs.ndim != 3 or target_probs.shape[0] == 0 or target_probs.shape[2] == 0:
        raise ValueError(f"target_probs must be shaped [n + 1, B, V] with V > 0; got {tuple(target_probs.shape)}")
    _lib.require_device(target_probs, "target_probs")
    rows, B, V = target_probs.shape
    if target_probs.dtype not in _TYPES:
        raise ValueError(f"target_probs must be float32 or bfloat16; got {target_probs.dtype}")
    if draft_probs is not None:
        if draft_probs.shape != (rows - 1, B, V):
            raise ValueError(f"draft_probs must be shaped [n, B, V] = {(rows - 1, B, V)}; got "
                             f"{tuple(draft_probs.shape)}")
        if draft_probs.dtype != target_probs.dtype or draft_probs.device != target_probs.device:
            raise ValueError("draft_probs must have the dtype and device of target_probs")
    if draft_tokens.shape != (rows - 1, B):
        raise ValueError(f"draft_tokens must be shaped [n, B] = {(rows - 1, B)}; got {tuple(draft_tokens.shape)}")
    if draft_tokens.dtype not in (torch.int64, torch.int32):
        raise ValueError(f"draft_tokens must be int64 or int32; got {draft_tokens.dtype}")
    if uniforms.shape != (rows, B) or uniforms.dtype != torch.float32:
        raise ValueError(f"uniforms must be float32 of shape [n + 1, B] = {(rows, B)}; got {uniforms.dtype}, "
                         f"{tuple(uniforms.shape)}")
    if draft_tokens.device != target_probs.device or uniforms.device != target_probs.device:
        raise ValueError("draft_tokens and uniforms must be on the device of target_probs")
    if lengths is not None:
        if lengths.shape != (B,) or lengths.device != target_probs.device:
            raise ValueError(f"lengths must be shaped [B] on the device of target_probs; got {tuple(lengths.shape)}")
        if lengths.dtype not in (torch.int32, torch.int64):
            raise ValueError(f"lengths must be int32 or int64; got {lengths.dtype}")
        if lengths.dtype == torch.int64:
            lengths = lengths.clamp(0, rows - 1).to(torch.int32)
        lengths = lengths.contiguous()
    if autograd.plain(target_probs, draft_tokens, uniforms) and (draft_probs is None or autograd.plain(draft_probs)):
        return VerifiedTokens(*autograd.native().verify_draft(target_probs, draft_probs, draft_tokens, uniforms,
                                                              lengths))
    return VerifiedTokens(*_verify(
        _rows(target_probs.detach()), None if draft_probs is None else _rows(draft_probs.detach()),
        draft_tokens.to(torch.int64).contiguous(), uniforms.detach().contiguous(), lengths))
