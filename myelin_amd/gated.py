"""A linear recurrence with a gate for every step and channel
(``csrc/gated_recurrence.hip``): a leaky integrator, as a membrane is, whose time
constant is an input.

``h_t = a_t h_{t-1} + (1 - a_t) x_t`` with ``a_t = sigmoid(gate_t)``: a channel
holds what it has (``a`` near 1) or takes what comes (``a`` near 0).  Prompts and
training run over whole sequences (:func:`gated_recurrence`), generation one step
at a time (:func:`gated_recurrence_step`); both carry the same state, so either
continues the other.
"""

from __future__ import annotations

import ctypes
import math
from typing import Any, Literal

import torch
from torch import nn

from myelin_amd import _lib, autograd
from myelin_amd.modules import LinearSynapse
from myelin_amd.packing import _device_of

_TYPES = (torch.float32, torch.bfloat16)


def _strides(*tensors):
    """Host array of the strides of all but each tensor's last dimension."""

    s = [x for t in tensors for x in t.stride()[:-1]]
    return (ctypes.c_int64 * len(s))(*s)


def _rows(t: torch.Tensor) -> torch.Tensor:
    """``t`` with unit stride in its last dimension, and batch rows near enough for
    a workgroup's 32-bit offsets."""

    B, N = t.shape[-2:]
    near = B <= 1 or N == 0 or (64 // N + 1) * t.stride(-2) + N < 2**29
    return t if near and (t.stride(-1) == 1 or N == 1) else t.contiguous()


def _workspace(x, backward):
    n = _lib.load().myelin_gated_recurrence_workspace_elems(_lib.DT[x.dtype], *x.shape, backward)
    return (torch.empty(n, dtype=torch.float32, device=x.device) if n else None), n


def _forward(x, gate, state, lengths, keep):
    """(final state, out, kept states)"""

    T, B, N = x.shape
    dev = x.device
    out = torch.empty((T, B, N), dtype=x.dtype, device=dev)
    final = torch.empty((B, N), dtype=torch.float32, device=dev)
    kept = None
    if keep:
        kept = torch.empty(_lib.load().myelin_gated_recurrence_kept_elems(T, B, N), dtype=torch.float32, device=dev)
    ws, n = _workspace(x, 0)
    with _device_of(x):
        _lib.call("myelin_gated_recurrence_fwd", x.data_ptr(), gate.data_ptr(), _lib.DT[x.dtype], _strides(x, gate),
                  _lib.ptr(state), _lib.ptr(lengths), out.data_ptr(), final.data_ptr(), _lib.ptr(kept), T, B, N,
                  _lib.ptr(ws), n, _lib.stream(dev))
    return final, out, kept


class HipGatedRecurrenceFunction(torch.autograd.Function):
    """Saves its inputs, by reference, and the states before every 8th step:
    the backward pass runs the steps between them again, and the adjoint."""

    @staticmethod
    def forward(ctx: Any, x, gate, state, lengths):
        ctx.set_materialize_grads(False)
        final, out, kept = _forward(x, gate, state, lengths, any(ctx.needs_input_grad[:3]))
        ctx.save_for_backward(x, gate, lengths, kept)
        return final, out

    @staticmethod
    @autograd.differentiated_once
    def backward(ctx: Any, g_final, g_out):
        if g_final is None and g_out is None:
            return (None,) * 4
        x, gate, lengths, kept = ctx.saved_tensors
        T, B, N = x.shape
        dev = x.device
        g_out = None if g_out is None else _rows(g_out)
        g_final = None if g_final is None else g_final.contiguous()
        gx, gg = (torch.empty((T, B, N), dtype=x.dtype, device=dev) if need else None
                  for need in ctx.needs_input_grad[:2])
        gs = torch.empty((B, N), dtype=torch.float32, device=dev) if ctx.needs_input_grad[2] else None
        ws, n = _workspace(x, 1)
        with _device_of(x):
            _lib.call("myelin_gated_recurrence_bwd", x.data_ptr(), gate.data_ptr(), _lib.ptr(g_out), _lib.DT[x.dtype],
                      _strides(x, gate, x if g_out is None else g_out), _lib.ptr(lengths), kept.data_ptr(),
                      _lib.ptr(g_final), _lib.ptr(gx), _lib.ptr(gg), _lib.ptr(gs), T, B, N, _lib.ptr(ws), n,
                      _lib.stream(dev))
        return gx, gg, gs, None


def _check(x, gate, ndim, dims):
    if x.ndim != ndim:
        raise ValueError(f"x must be shaped {dims}; got {tuple(x.shape)}")
    _lib.require_device(x, "x")
    if x.dtype not in _TYPES:
        raise ValueError(f"x must be float32 or bfloat16; got {x.dtype}")
    if gate.shape != x.shape or gate.dtype != x.dtype or gate.device != x.device:
        raise ValueError(f"gate must have the shape, dtype and device of x; got {gate.dtype}, {tuple(gate.shape)} on "
                         f"{gate.device}")


def _check_state(state, x, name):
    if state.shape != x.shape[-2:]:
        raise ValueError(f"{name} must be shaped [B, N] = {tuple(x.shape[-2:])}; got {tuple(state.shape)}")
    if state.dtype != torch.float32 or state.device != x.device:
        raise ValueError(f"{name} must be float32 on the device of x")


def gated_recurrence(
    x: torch.Tensor,
    gate: torch.Tensor,
    initial_state: torch.Tensor | None = None,
    *,
    lengths: torch.Tensor | None = None,
) -> tuple[torch.Tensor, torch.Tensor]:
    """``h_t = a_t h_{t-1} + (1 - a_t) x_t``, ``a_t = sigmoid(gate_t)``.

    Time-major ``x [T, B, N]`` and ``gate [T, B, N]``, float32 or bfloat16, any
    strides (two halves of one projection are read in place).
    ``initial_state [B, N]`` float32 (zeros by default).

    ``lengths [B]`` (int32 or int64 on the device, taken into [0, T]) gives each
    sample's steps: later ones are part of no result, leave the state and give zeros
    (their memory may be read; what it holds, NaN too, does not count).

    Returns ``(final state [B, N] float32, out [T, B, N])``, differentiable in x,
    the gate and the initial state.  States and sums are float32.

    An infinity or a NaN makes the results that it is part of infinite or NaN, and no
    others: of ``x``, a gate or the initial state, the states from its step on and the
    gates' gradients from there on; of a gate (NaN) or an incoming gradient, the
    gradients of its own step and earlier ones.
    """

    _check(x, gate, 3, "[T, B, N]")
    if x.shape[0] == 0:
        raise ValueError("x must have at least one timestep")
    if initial_state is not None:
        _check_state(initial_state, x, "initial_state")
        initial_state = initial_state.contiguous()
    if lengths is not None:
        if lengths.shape != x.shape[1:2] or lengths.device != x.device:
            raise ValueError(f"lengths must be shaped [B] on the device of x; got {tuple(lengths.shape)}")
        if lengths.dtype not in (torch.int32, torch.int64):
            raise ValueError(f"lengths must be int32 or int64; got {lengths.dtype}")
        if lengths.dtype == torch.int64:
            lengths = lengths.clamp(0, x.shape[0]).to(torch.int32)
        lengths = lengths.contiguous()
    if autograd.plain(x, gate) and (initial_state is None or autograd.plain(initial_state)):
        state, out = autograd.native().gated_recurrence(x, gate, initial_state, lengths)
        return state, out
    return HipGatedRecurrenceFunction.apply(_rows(x), _rows(gate), initial_state, lengths)


def gated_recurrence_step(
    x: torch.Tensor,
    gate: torch.Tensor,
    state: torch.Tensor,
    *,
    out_state: torch.Tensor | None = None,
) -> tuple[torch.Tensor, torch.Tensor]:
    """One step of :func:`gated_recurrence`, without gradient: ``x [B, N]``,
    ``gate [B, N]``, ``state [B, N]``.

    Returns ``(state, out [B, N])``.  The new state goes to ``out_state``
    (contiguous; ``state`` itself for an update in place; no part of ``x`` or
    ``gate``) or to a new tensor.
    """

    _check(x, gate, 2, "[B, N]")
    _check_state(state, x, "state")
    if torch.is_grad_enabled() and any(t.requires_grad for t in (x, gate, state)):
        raise ValueError("gated_recurrence_step has no gradient; use gated_recurrence, or torch.no_grad()")
    autograd.refuse_tangents("gated_recurrence_step", x, gate, state)
    if out_state is not None:
        state = state.contiguous()
        _check_state(out_state, x, "out_state")
        if not out_state.is_contiguous():
            raise ValueError("out_state must be contiguous")
        if out_state.requires_grad:
            raise ValueError("out_state is written in place and must not require a gradient")
        a, b, size = state.data_ptr(), out_state.data_ptr(), 4 * state.numel()
        if a != b and a < b + size and b < a + size:
            raise ValueError("out_state must be state itself or not overlap it")
        for name, t in (("x", x), ("gate", gate)):
            a = t.data_ptr()
            end = a + t.element_size() * (1 + sum((n - 1) * s for n, s in zip(t.shape, t.stride())))
            if size and a < b + size and b < end:
                raise ValueError(f"out_state must not overlap {name}")
    new, out = autograd.native().gated_recurrence_step(x, gate, state, out_state)
    return (new if out_state is None else out_state), out


class GatedRecurrence(nn.Module):
    """Inputs and gates from one projection, and the recurrence with them.

    The gates' biases start at time constants spread evenly over the logarithm of
    ``taus`` (steps, as ``LIFParams``): ``sigmoid(log(tau - 1)) = 1 - 1 / tau``.
    ``forward`` takes whole sequences ``[T, B, in_features]``, ``step`` one step.
    """

    def __init__(self, in_features: int, features: int, taus: tuple[float, float] = (4.0, 64.0),
                 synapse_precision: Literal["fp32", "bf16"] = "fp32") -> None:
        super().__init__()
        low, high = taus
        if not 1.0 < low <= high < math.inf:
            raise ValueError(f"taus must be two time constants above 1, the shorter first; got {taus}")
        self.features = features
        self.synapse = LinearSynapse(in_features, 2 * features, synapse_precision=synapse_precision)
        tau = torch.logspace(math.log2(low), math.log2(high), features, base=2.0, dtype=torch.float64)
        with torch.no_grad():
            self.synapse.bias[features:] = torch.log(tau - 1.0).float()

    def forward(self, inputs: torch.Tensor, initial_state: torch.Tensor | None = None,
                lengths: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
        x, gate = self.synapse(inputs).split(self.features, -1)
        return gated_recurrence(x, gate, initial_state, lengths=lengths)

    def step(self, inputs: torch.Tensor, state: torch.Tensor,
             out_state: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
        x, gate = self.synapse(inputs[None])[0].split(self.features, -1)
        return gated_recurrence_step(x, gate, state, out_state=out_state)
