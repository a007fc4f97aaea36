"""Linear attention with a decay for each head (``csrc/decay_attention.hip``):
a memory addressed by content that leaks as a membrane does.

A head keeps a matrix ``S_t = d S_{t-1} + k_t v_t^T`` and answers a query with
``scale * S_t^T q_t``; the decay ``d = 1 - 1 / tau`` is a constant of the head,
as ``LIFParams``' time constants are of a layer.  Prompts and training run over
whole sequences (:func:`decay_attention`), generation one step at a time
(:func:`decay_attention_step`); both carry the same state, so either continues
the other.
"""

from __future__ import annotations

import ctypes
import math
from typing import Any, Sequence

import torch
from torch import nn

from myelin_amd import _lib, autograd
from myelin_amd.packing import _device_of

MAX_DIM = 128
_TYPES = (torch.float32, torch.bfloat16)


def _strides(*tensors):
    """Host array of the strides of all but each tensor's last dimension."""

    s = [x for t in tensors for x in t.stride()[:-1]]
    return (ctypes.c_int64 * len(s))(*s)


def _rows(t: torch.Tensor) -> torch.Tensor:
    """``t`` with unit stride in its last dimension."""

    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


def _workspace(q, sizes, backward):
    n = _lib.load().myelin_decay_attention_workspace_elems(_lib.DT[q.dtype], *sizes, backward)
    return (torch.empty(n, dtype=torch.float32, device=q.device) if n else None), n


def _forward(q, k, v, decay, state, lengths, scale):
    T, B, H, Dk = q.shape
    Hk, Dv = v.shape[-2:]
    dev = q.device
    out = torch.empty((T, B, H, Dv), dtype=q.dtype, device=dev)
    final = torch.empty((B, H, Dk, Dv), dtype=torch.float32, device=dev)
    sizes = (T, B, H, Hk, Dk, Dv)
    ws, n = _workspace(q, sizes, 0)
    with _device_of(q):
        _lib.call("myelin_decay_attention_fwd", q.data_ptr(), k.data_ptr(), v.data_ptr(), _lib.DT[q.dtype],
                  _strides(q, k, v), decay.data_ptr(), _lib.ptr(state), _lib.ptr(lengths), out.data_ptr(),
                  final.data_ptr(), *sizes, scale, _lib.ptr(ws), n, _lib.stream(dev))
    return final, out


class HipDecayAttentionFunction(torch.autograd.Function):
    """Saves its inputs, by reference, and nothing per step: the backward pass
    runs the recurrence again, and its adjoint."""

    @staticmethod
    def forward(ctx: Any, q, k, v, decay, state, lengths, scale):
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(q, k, v, decay, state, lengths)
        ctx.scale = scale
        return _forward(q, k, v, decay, state, lengths, scale)

    @staticmethod
    @autograd.differentiated_once
    def backward(ctx: Any, g_final, g_out):
        if g_final is None and g_out is None:
            return (None,) * 7
        q, k, v, decay, state, lengths = ctx.saved_tensors
        T, B, H, Dk = q.shape
        Hk, Dv = v.shape[-2:]
        dev = q.device
        if g_out is None:
            g_out = torch.zeros((T, B, H, Dv), dtype=q.dtype, device=dev)
        g_out = _rows(g_out)
        g_final = None if g_final is None else g_final.contiguous()
        gq, gk, gv = (torch.empty(t.shape, dtype=t.dtype, device=dev) for t in (q, k, v))
        want_state = ctx.needs_input_grad[4]
        g_state = torch.empty((B, H, Dk, Dv), dtype=torch.float32, device=dev) if want_state else None
        sizes = (T, B, H, Hk, Dk, Dv)
        ws, n = _workspace(q, sizes, 1)
        with _device_of(q):
            _lib.call("myelin_decay_attention_bwd", q.data_ptr(), k.data_ptr(), v.data_ptr(), g_out.data_ptr(),
                      _lib.DT[q.dtype], _strides(q, k, v, g_out), decay.data_ptr(), _lib.ptr(state),
                      _lib.ptr(lengths), _lib.ptr(g_final), gq.data_ptr(), gk.data_ptr(), gv.data_ptr(),
                      _lib.ptr(g_state), *sizes, ctx.scale, _lib.ptr(ws), n, _lib.stream(dev))
        return (*(g if need else None for g, need in zip((gq, gk, gv), ctx.needs_input_grad)), None, g_state, None,
                None)


def _check(q, k, v, decay, ndim, dims):
    for name, t in (("q", q), ("k", k), ("v", v)):
        if t.ndim != ndim:
            raise ValueError(f"{name} must be shaped {dims}; got {tuple(t.shape)}")
        _lib.require_device(t, name)
        if t.dtype not in _TYPES:
            raise ValueError(f"{name} must be float32 or bfloat16; got {t.dtype}")
        if t.dtype != q.dtype or t.device != q.device:
            raise ValueError("q, k and v must have the same dtype and device")
    if k.shape[:-1] != v.shape[:-1] or q.shape[:-2] != k.shape[:-2]:
        raise ValueError(f"k and v must have q's time and batch sizes and the same heads; got {tuple(q.shape)}, "
                         f"{tuple(k.shape)} and {tuple(v.shape)}")
    if q.shape[-1] != k.shape[-1]:
        raise ValueError(f"q and k must have the same width; got {q.shape[-1]} and {k.shape[-1]}")
    H, Hk = q.shape[-2], k.shape[-2]
    if H == 0 or Hk == 0 or H % Hk:
        raise ValueError(f"q's heads must be a multiple of k's; got {H} and {Hk}")
    for name, t in (("q", q), ("v", v)):
        if not 1 <= t.shape[-1] <= MAX_DIM:
            raise ValueError(f"{name}'s width must be in [1, {MAX_DIM}]; got {t.shape[-1]}")
    if decay.shape != (H,) or decay.dtype != torch.float32 or decay.device != q.device:
        raise ValueError(f"decay must be float32 of shape ({H},) on the device of q; got {decay.dtype}, "
                         f"{tuple(decay.shape)} on {decay.device}")
    if decay.requires_grad:
        raise ValueError("decay is a constant of the heads and has no gradient; pass it detached")


def _check_state(state, q, v, name):
    want = (*q.shape[-3:-1], q.shape[-1], v.shape[-1])
    if state.shape != want:
        raise ValueError(f"{name} must be shaped [B, H, Dk, Dv] = {want}; got {tuple(state.shape)}")
    if state.dtype != torch.float32 or state.device != q.device:
        raise ValueError(f"{name} must be float32 on the device of q")


def _scale(scale, q):
    scale = q.shape[-1] ** -0.5 if scale is None else float(scale)
    if scale == 0.0 or not math.isfinite(scale):
        raise ValueError(f"scale must be finite and not zero; got {scale}")
    return scale


def decay_attention(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    decay: torch.Tensor,
    initial_state: torch.Tensor | None = None,
    *,
    lengths: torch.Tensor | None = None,
    scale: float | None = None,
) -> tuple[torch.Tensor, torch.Tensor]:
    """``S_t = decay[h] S_{t-1} + k_t v_t^T``, ``out_t = scale * S_t^T q_t``.

    Time-major ``q [T, B, H, Dk]``, ``k [T, B, Hk, Dk]``, ``v [T, B, Hk, Dv]``,
    float32 or bfloat16, widths up to 128, any strides; ``Hk`` divides ``H`` and
    query heads ``h`` share the key/value head ``h // (H // Hk)``.  ``decay [H]``
    float32 in [0, 1], a constant.  ``initial_state [B, H, Dk, Dv]`` float32
    (zeros by default).  ``scale`` is ``Dk ** -0.5`` by default.

    ``lengths [B]`` (int32 or int64 on the device, taken into [0, T]) gives each
    sample's steps: later ones are not read, leave the state and give zeros.

    Returns ``(final state [B, H, Dk, Dv] float32, out [T, B, H, Dv])``,
    differentiable in q, k, v and the initial state.  States and sums are
    float32.

    An infinity or a NaN in a step makes the results that it is part of (of its
    own step and later ones, states, gradients) infinite or NaN, and no others.
    Which of the two is not the formula's where that has infinities: the
    bfloat16 kernel works in parts, whose infinities cancel.
    """

    _check(q, k, v, decay, 4, "[T, B, heads, width]")
    if q.shape[0] == 0:
        raise ValueError("q must have at least one timestep")
    if initial_state is not None:
        _check_state(initial_state, q, v, "initial_state")
        initial_state = initial_state.contiguous()
    if lengths is not None:
        if lengths.shape != q.shape[1:2] or lengths.device != q.device:
            raise ValueError(f"lengths must be shaped [B] on the device of q; got {tuple(lengths.shape)}")
        if lengths.dtype not in (torch.int32, torch.int64):
            raise ValueError(f"lengths must be int32 or int64; got {lengths.dtype}")
        if lengths.dtype == torch.int64:
            lengths = lengths.clamp(0, q.shape[0]).to(torch.int32)
        lengths = lengths.contiguous()
    scale = _scale(scale, q)
    q, k, v, decay = _rows(q), _rows(k), _rows(v), decay.contiguous()
    if autograd.plain(q, k, v) and (initial_state is None or autograd.plain(initial_state)):
        state, out = autograd.native().decay_attention(q, k, v, decay, initial_state, lengths, scale)
        return state, out
    return HipDecayAttentionFunction.apply(q, k, v, decay, initial_state, lengths, scale)


def decay_attention_step(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    decay: torch.Tensor,
    state: torch.Tensor,
    *,
    scale: float | None = None,
    out_state: torch.Tensor | None = None,
) -> tuple[torch.Tensor, torch.Tensor]:
    """One step of :func:`decay_attention`, without gradient: ``q [B, H, Dk]``,
    ``k [B, Hk, Dk]``, ``v [B, Hk, Dv]``, ``state [B, H, Dk, Dv]``.

    Returns ``(state, out [B, H, Dv])``.  The new state goes to ``out_state``
    (contiguous; ``state`` itself for an update in place) or to a new tensor.
    """

    _check(q, k, v, decay, 3, "[B, heads, width]")
    _check_state(state, q, v, "state")
    scale = _scale(scale, q)
    if torch.is_grad_enabled() and any(t.requires_grad for t in (q, k, v, state)):
        raise ValueError("decay_attention_step has no gradient; use decay_attention, or torch.no_grad()")
    autograd.refuse_tangents("decay_attention_step", q, k, v, decay, state)
    state = state.contiguous()
    if out_state is not None:
        _check_state(out_state, q, v, "out_state")
        if not out_state.is_contiguous():
            raise ValueError("out_state must be contiguous")
        if out_state.requires_grad:
            raise ValueError("out_state is written in place and must not require a gradient")
        a, b, size = state.data_ptr(), out_state.data_ptr(), 4 * state.numel()
        if a != b and a < b + size and b < a + size:
            raise ValueError("out_state must be state itself or not overlap it")
    new, out = autograd.native().decay_attention_step(_rows(q), _rows(k), _rows(v), decay.contiguous(), state,
                                                      out_state, scale)
    return (new if out_state is None else out_state), out


class DecayAttention(nn.Module):
    """The decays of a layer's heads, and attention with them.

    ``taus`` gives each head's time constant in steps (``decay = 1 - 1 / tau``,
    as ``LIFParams``; ``math.inf`` never forgets), kept in float32 whatever type the
    module is cast to.  ``forward`` takes whole sequences, ``step`` one step.
    """

    def __init__(self, taus: Sequence[float], scale: float | None = None) -> None:
        super().__init__()
        if len(taus) == 0 or not all(t >= 1.0 for t in taus):
            raise ValueError("taus must hold a time constant of at least 1 for each head")
        self.scale = scale
        decay = torch.tensor([1.0 - 1.0 / t for t in taus], dtype=torch.float64)
        self.register_buffer("decay", decay.to(torch.float32))

    def _apply(self, fn, recurse: bool = True):
        decay = self.decay
        super()._apply(fn, recurse)
        if self.decay.dtype != decay.dtype:  # in bfloat16 a decay of 1 - 1 / 1024 is 1
            self.decay = decay.to(self.decay.device)
        return self

    def forward(self, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, initial_state: torch.Tensor | None = None,
                lengths: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
        return decay_attention(q, k, v, self.decay, initial_state, lengths=lengths, scale=self.scale)

    def step(self, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, state: torch.Tensor,
             out_state: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
        return decay_attention_step(q, k, v, self.decay, state, scale=self.scale, out_state=out_state)
