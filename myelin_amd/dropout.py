"""Dropout from a counter-based generator (``csrc/dropout.hip``).

The mask is a function of ``(seed, offset, element)``: the backward pass
computes it again, so a training step stores none, and the same call gives the
same mask on any layout, device or stream.  Spiking layers usually keep one
mask for all time steps of a sample (``time_shared=True``).
"""

from __future__ import annotations

from typing import Any

import torch
from torch import nn

from myelin_amd import _lib, autograd
from myelin_amd.packing import _device_of

_TYPES = (torch.float32, torch.bfloat16)


def _launch(x, residual, steps, threshold, scale, seed, offset):
    y = torch.empty_like(x)
    at = offset if isinstance(offset, torch.Tensor) else None
    with _device_of(x):
        _lib.call("myelin_counter_dropout", x.data_ptr(), _lib.DT[x.dtype], _lib.ptr(residual), y.data_ptr(), steps,
                  x.numel() // steps if steps else 0, threshold, scale, seed, 0 if at is not None else offset,
                  _lib.ptr(at), _lib.stream(x.device))
    return y


class HipCounterDropoutFunction(torch.autograd.Function):
    """``dx`` is the dropout of the gradient with the same mask, which is
    computed again; the residual's gradient is the gradient itself."""

    @staticmethod
    def forward(ctx: Any, x, residual, steps, threshold, scale, seed, offset):
        ctx.set_materialize_grads(False)
        ctx.meta = (steps, threshold, scale, seed)
        if isinstance(offset, torch.Tensor):
            ctx.save_for_backward(offset)
            ctx.offset = None
        else:
            ctx.offset = offset
        return _launch(x, residual, steps, threshold, scale, seed, offset)

    @staticmethod
    @autograd.differentiated_once
    def backward(ctx: Any, g):
        gx = None
        if g is not None and ctx.needs_input_grad[0]:
            offset = ctx.saved_tensors[0] if ctx.offset is None else ctx.offset
            gx = _launch(g.contiguous(), None, *ctx.meta, offset)
        return gx, g if ctx.needs_input_grad[1] else None, None, None, None, None, None


def counter_dropout(
    x: torch.Tensor,
    p: float,
    seed: int,
    offset: int | torch.Tensor = 0,
    *,
    residual: torch.Tensor | None = None,
    time_shared: bool = False,
) -> torch.Tensor:
    """``x / (1 - p)`` with probability ``1 - p``, else 0; plus ``residual``.

    ``x`` (and ``residual``, of its shape and type) is float32 or bfloat16; the
    sum is formed in float32 and rounded once.  Calls that must not share a
    mask differ in ``seed`` or ``offset``; ``offset`` may be an int64 device
    tensor of one element, so that a captured graph can advance it (it must
    then stay unchanged until the backward pass has run).  ``time_shared``
    takes dimension 0 as time and uses one mask for all of it.

    Mask element ``i`` (row-major) is word ``i % 4`` of Philox 4x32-10 at the
    counter ``(i // 4, offset)`` and key ``seed``; it keeps where the word is at
    least ``floor(p * 2**32)``.  Dropped NaNs and infinities are dropped.
    """

    p = float(p)
    if not 0.0 <= p <= 1.0:
        raise ValueError(f"p must be in [0, 1]; got {p}")
    if not 0 <= seed < 2**63:
        raise ValueError("seed must be in [0, 2**63)")
    _lib.require_device(x, "x")
    if x.dtype not in _TYPES:
        raise ValueError(f"x must be float32 or bfloat16; got {x.dtype}")
    if time_shared and x.ndim == 0:
        raise ValueError("time_shared needs a time dimension")
    if residual is not None:
        if residual.shape != x.shape:
            raise ValueError(f"residual must match x; got {tuple(residual.shape)} and {tuple(x.shape)}")
        if residual.device != x.device or residual.dtype != x.dtype:
            raise ValueError("residual must have the device and dtype of x")
        residual = residual.contiguous()
    if isinstance(offset, torch.Tensor):
        if offset.numel() != 1 or offset.dtype != torch.int64 or offset.device != x.device:
            raise ValueError("an offset tensor must hold one int64 on the device of x")
    elif not 0 <= offset < 2**63:
        raise ValueError("offset must be in [0, 2**63)")
    x = x.contiguous()
    steps = x.shape[0] if time_shared else 1
    threshold = int(p * 2**32)
    scale = 0.0 if p == 1.0 else 1.0 / (1.0 - p)
    if autograd.plain(x) and (residual is None or autograd.plain(residual)):
        at, number = (offset, 0) if isinstance(offset, torch.Tensor) else (None, offset)
        return autograd.native().counter_dropout(x, residual, at, steps, threshold, scale, seed, number)
    return HipCounterDropoutFunction.apply(x, residual, steps, threshold, scale, seed, offset)


class CounterDropout(nn.Module):
    """``counter_dropout`` with a new mask for each training call.

    Without a ``seed`` each call takes its offset from torch's generator of the
    input's device, as ``nn.Dropout`` takes its mask: ``torch.manual_seed``
    decides the masks, modules have masks of their own, a captured graph draws a
    new one at each replay, and ``torch.utils.checkpoint``, which puts the
    generator back, computes the forward pass again under the same mask.

    With a ``seed`` the masks are those of the calls 1, 2, ... of this seed,
    whatever else draws random numbers; modules that must not share masks have
    seeds of their own, as have the ranks of a data-parallel run.  The count of
    calls is a buffer (``offset``), saved with the module and advanced on the
    device, so that a captured training step draws a new mask at each replay.
    A forward pass that a backward pass computes again would draw the next mask
    and is refused: checkpointed layers take no seed.

    In evaluation mode the input passes, plus ``residual``.
    """

    def __init__(self, p: float, seed: int | None = None, time_shared: bool = False) -> None:
        super().__init__()
        if not 0.0 <= p <= 1.0:
            raise ValueError(f"p must be in [0, 1]; got {p}")
        self.p = p
        self.seed = seed
        self.time_shared = time_shared
        self.register_buffer("offset", torch.zeros(1, dtype=torch.int64))

    def forward(self, x: torch.Tensor, residual: torch.Tensor | None = None) -> torch.Tensor:
        if not self.training:
            return x if residual is None else x + residual
        # the offset is a tensor of this call's own: the backward pass reads it again
        if self.seed is None:
            seed, offset = 0, torch.randint(2**63 - 1, (1,), device=x.device)
        else:
            if torch._C._current_graph_task_id() != -1:
                raise RuntimeError("CounterDropout with a seed counts its calls, and this one computes a forward pass "
                                   "again within a backward pass, which would change its mask; leave the seed out, or "
                                   "call counter_dropout with the first pass's offset")
            seed, offset = self.seed, self.offset + 1
            self.offset.copy_(offset)
        return counter_dropout(x, self.p, seed, offset, residual=residual, time_shared=self.time_shared)
