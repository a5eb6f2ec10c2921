"""Gated linear recurrence on the HIP library (include/gdn2.h).

  gated_recurrence(x, g, ...)           h_t = exp(g_t) h_{t-1} + x_t for every channel: training and
                                        prompts
  gated_recurrence_step(state, x, g)    one token on a carried state

It has no counterpart in the reference.  The first form is differentiable, once and in reverse mode
(anything else is refused); gated_recurrence_forward and gated_recurrence_backward are the raw calls,
for a block that writes its backward out.  All run only on the GPU: there is no CPU fallback.
"""
from __future__ import annotations

import struct

import torch
from torch.autograd.graph import increment_version

from ._lib import check, lib
from ._once import once
from .linear_ops import (_CODES, F32, _call, _differentiates, _dtype, _has_tangent, _ptr,
                         _same_device, _wants_grad)

__all__ = ["gated_recurrence", "gated_recurrence_forward", "gated_recurrence_backward",
           "gated_recurrence_step"]

_VIEW = struct.Struct("Pii4q").pack
_SHAPE = struct.Struct("3q").pack
_SIZES: dict = {}


def _view(t):
    """A view of [B, T, W], [B, T] or [B, W]."""
    if t is None:
        return None
    st = t.stride()
    return _VIEW(t.data_ptr(), _CODES[t.dtype], 0, *st, *(0,) * (4 - len(st)))


def _mask(m, name, shape):
    if m is None:
        return None
    if m.shape != shape:
        raise ValueError(f"{name} must be [batch, time] (got {tuple(m.shape)})")
    return m if m.dtype == F32 else m.float()


def _inputs(x, g, valid, reset, state=None, state_name="initial"):
    """Checked inputs: (dtype code, shape, views of x, g, valid and reset, what they look at)."""
    code = _dtype(x, "x")
    _dtype(g, "g")
    if x.dim() != 3:
        raise ValueError("x must be [batch, time, width]")
    B, T, W = x.shape
    if g.shape != x.shape:
        raise ValueError(f"g must have x's shape {(B, T, W)} (got {tuple(g.shape)})")
    if state is not None and state.shape != (B, W):
        raise ValueError(f"{state_name} must be [batch, width] (got {tuple(state.shape)})")
    _same_device(x, "g valid reset " + state_name, g, valid, reset, state)
    valid, reset = _mask(valid, "valid", (B, T)), _mask(reset, "reset", (B, T))
    return code, (B, T, W), (_view(x), _view(g), _view(valid), _view(reset)), (valid, reset)


def _bytes(query: str, shape, *args) -> int:
    """A buffer's size, remembered by shape."""
    key = (query, shape) + args
    n = _SIZES.get(key)
    if n is None:
        n = getattr(lib(), query)(_SHAPE(*shape), *args)
        if n == 0:
            check(query, 2)
        _SIZES[key] = n
    return n


def _scratch(n: int, shape, dev):
    """Scratch of a query's n bytes.  16 where none is needed: two segments of a single value need as many,
    those of more values more."""
    if n == 16 and shape[0] * shape[2] > 1:
        return None
    return torch.empty((n,), dtype=torch.uint8, device=dev)


def gated_recurrence_forward(x, g, valid=None, reset=None, initial=None, train: bool = True):
    """Raw forward.  Returns (y, final_state, checkpoint); the checkpoint is private storage for
    gated_recurrence_backward, without train scratch alone, or None where none is needed."""
    code, shape, views, held = _inputs(x, g, valid, reset, initial)
    if initial is not None and initial.dtype != F32:
        initial = initial.float()
    dev, train = x.device, 1 if train else 0
    n = _bytes("gdn2_recurrence_checkpoint_bytes", shape, code, train)
    y = torch.empty(shape, dtype=x.dtype, device=dev)
    final = torch.empty((shape[0], shape[2]), dtype=F32, device=dev)
    ck = torch.empty((n,), dtype=torch.uint8, device=dev) if train else _scratch(n, shape, dev)
    _call("gdn2_recurrence_scan", dev, _SHAPE(*shape), *views, _view(initial), y.data_ptr(),
          final.data_ptr(), train, _ptr(ck), n)
    return y, final, ck


def gated_recurrence_backward(x, g, valid, reset, initial, checkpoint, dy, d_final_state=None,
                              wanted=(True,) * 3):
    """Raw VJP, from the forward's inputs and checkpoint.  Returns (dx, dg, d_initial), d_initial None
    without an initial state.  wanted (dx, dg, d_initial): those that are False are None."""
    code, shape, views, held = _inputs(x, g, valid, reset, initial)
    B, T, W = shape
    dev = x.device
    if dy.shape != x.shape:
        raise ValueError(f"dy must have shape {shape} (got {tuple(dy.shape)})")
    if d_final_state is not None and d_final_state.shape != (B, W):
        raise ValueError(f"d_final_state must be [batch, width] (got {tuple(d_final_state.shape)})")
    if checkpoint is None or checkpoint.dtype != torch.uint8 or not checkpoint.is_contiguous():
        raise ValueError("checkpoint must be what the forward returned")
    _same_device(x, "dy d_final_state checkpoint", dy, d_final_state, checkpoint)
    if dy.dtype != x.dtype:
        dy = dy.to(x.dtype)
    if d_final_state is not None:
        d_final_state = d_final_state.to(F32).contiguous()
    dx = torch.empty(shape, dtype=x.dtype, device=dev) if wanted[0] else None
    dg = torch.empty(shape, dtype=g.dtype, device=dev) if wanted[1] else None
    di = torch.empty((B, W), dtype=F32, device=dev) if wanted[2] and initial is not None else None
    n = _bytes("gdn2_recurrence_workspace_bytes", shape, code)
    ws = _scratch(n, shape, dev)
    _call("gdn2_recurrence_backward", dev, _SHAPE(*shape), *views, checkpoint.data_ptr(),
          checkpoint.numel(), _view(dy), _ptr(d_final_state), _ptr(dx), _ptr(dg), _ptr(di),
          _ptr(ws), n)
    return dx, dg, di


class _GatedRecurrence(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, g, valid, reset, initial):
        y, final, ck = gated_recurrence_forward(x, g, valid, reset, initial)
        ctx.set_materialize_grads(False)  # an unused output reaches backward as None
        ctx.save_for_backward(x, g, valid, reset, initial, ck)
        return y, final

    @staticmethod
    @once
    def backward(ctx, dy, d_final):
        x, g, valid, reset, initial, ck = ctx.saved_tensors
        if dy is None and d_final is None:
            return (None,) * 5
        if dy is None:
            dy = torch.zeros((), dtype=x.dtype, device=x.device).expand(x.shape)
        need = ctx.needs_input_grad
        dx, dg, di = gated_recurrence_backward(x, g, valid, reset, initial, ck, dy, d_final,
                                               (need[0], need[1], need[4]))
        return dx, dg, None, None, None if di is None else di.to(initial.dtype)


def gated_recurrence(x, g, valid=None, reset=None, initial=None):
    """Gated linear recurrence, for every channel and valid token
        h = exp(g) h + x,  y = h
    x, g [B, T, W], each float32 or bfloat16, any strides; g the log decay; valid, reset [B, T] float
    0/1 or None: padding keeps the state and gives zero, a reset on a valid token empties the state
    before it, as does a gate below -87.3 (exp(g) < 2^-126); initial [B, W] or None (zero).  Returns
    (y [B, T, W] in x's dtype, final_state [B, W] float32), differentiable in x, g and initial.
    States and sums are float32."""
    for name, m in (("valid", valid), ("reset", reset)):
        if m is not None and m.requires_grad:
            raise ValueError(f"{name} is nondifferentiable metadata")
    if not _differentiates(x, g, initial):
        return gated_recurrence_forward(x, g, valid, reset, initial, False)[:2]
    return _GatedRecurrence.apply(x, g, valid, reset, initial)


def gated_recurrence_step(state, x, g, valid=None, reset=None):
    """One token per sequence on a carried state, updated in place: state [B, W] float32 contiguous; x, g
    [B, 1, W], valid, reset [B, 1] or None.  Returns y [B, 1, W] in x's dtype.  It has no gradient: where
    one is recorded, inputs that require one are refused, and autograd is told that the state has
    changed."""
    if state.dtype != F32 or not state.is_contiguous():
        raise ValueError("state must be a contiguous float32 [B, W] tensor")
    if _wants_grad(state, x, g) or _has_tangent(state, x, g):
        raise ValueError("gated_recurrence_step has no gradient: call it under torch.no_grad(), or on "
                         "detached inputs")
    _, shape, views, held = _inputs(x, g, valid, reset, state, "state")
    y = torch.empty(shape, dtype=x.dtype, device=x.device)
    _call("gdn2_recurrence_step", x.device, _SHAPE(*shape), *views, state.data_ptr(), y.data_ptr())
    increment_version(state)
    return y
