"""Operators of a linear-attention block on the HIP library (include/gdn2.h).

  linear_attention(q, k, v, g, ...)    linear attention with a decay for each head: chunked, for
                                       training and prompts
  linear_attention_step(state, ...)    its recurrent form, one token on a carried state
  layer_norm(x, weight, bias)          layer norm over the last axis
  swiglu_q8(h)                         SwiGLU that keeps its input in 8 bits for the backward

They have no counterpart in the reference.  The first form of each is differentiable, once and in
reverse mode (anything else is refused);
*_forward and *_backward are the raw calls, for a block that writes its backward out
(delta_mixers.linear).  All run only on the GPU: there is no CPU fallback.
"""
from __future__ import annotations

import struct

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable
from torch.autograd.graph import increment_version

from . import _size, _shape
from ._lib import GDN2_BF16, GDN2_F32, check, lib, on_device

__all__ = ["linear_attention", "linear_attention_forward", "linear_attention_backward",
           "linear_attention_step", "layer_norm", "layer_norm_forward", "layer_norm_backward",
           "swiglu_q8", "swiglu_q8_forward", "swiglu_q8_backward", "q8_values"]

F32, BF16 = torch.float32, torch.bfloat16
Q8_BLOCK = 32  # columns that share an exponent


_CODES = {F32: GDN2_F32, BF16: GDN2_BF16}
# gdn2_view and the shapes as the bytes that the library reads: packed at once, a call spends a third
# of the time that structures take it.
_VIEW = struct.Struct("Pii4q").pack
_SHAPE = struct.Struct("5q").pack
_ROWS = struct.Struct("4q").pack


def _view(t):
    if t is None:
        return None
    st = t.stride()
    if len(st) == 3:
        return _VIEW(t.data_ptr(), GDN2_F32, 0, *st, 0)
    if len(st) == 2:
        return _VIEW(t.data_ptr(), GDN2_F32, 0, *st, 0, 0)
    return _VIEW(t.data_ptr(), _CODES[t.dtype], 0, *st)


def _ptr(t):
    return None if t is None else t.data_ptr()


def _call(fn: str, device, *args):
    """A library call on the device's current stream."""
    idx = device.index
    f = getattr(lib(), fn)
    if idx == torch._C._cuda_getDevice():
        rc = f(*args, torch._C._cuda_getCurrentRawStream(idx))
    else:
        with on_device(device):
            rc = f(*args, torch._C._cuda_getCurrentRawStream(idx))
    if rc:
        check(fn, rc)


def _dtype(t: torch.Tensor, name: str) -> int:
    code = _CODES.get(t.dtype)
    if code is None:
        raise TypeError(f"{name} must be float32 or bfloat16 (got {t.dtype})")
    if not t.is_cuda:
        raise ValueError(f"{name} must live on the GPU; there is no CPU fallback")
    return code


def _same_device(like: torch.Tensor, names: str, *tensors) -> None:
    idx = like.get_device()
    for i, t in enumerate(tensors):
        if t is not None and t.get_device() != idx:
            raise ValueError(f"{names.split()[i]} must live on {like.device} (got {t.device})")


def _wants_grad(*tensors) -> bool:
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


def _has_tangent(*tensors) -> bool:
    return forward_ad._current_level >= 0 and any(
        forward_ad.unpack_dual(t).tangent is not None for t in tensors)


def _differentiates(*tensors) -> bool:
    """Whether a call goes through its autograd function: for gradients, and inside forward-mode
    differentiation, which the function refuses for inputs with a tangent."""
    return forward_ad._current_level >= 0 or _wants_grad(*tensors)


# ---- linear attention ------------------------------------------------------------------


def _attention_inputs(q, k, v, g, valid, reset, state=None, state_name="initial"):
    """Checked inputs: (dtype code, sizes, views of q, k, v, g, valid, reset and what they look at)."""
    code = _dtype(q, "q")
    shape = q.shape
    if len(shape) != 4 or v.dim() != 4:
        raise ValueError("q must be [batch, time, head, key] and v [batch, time, head, value]")
    B, T, H, K = shape
    V = v.shape[3]
    if k.shape != shape or v.shape != (B, T, H, V):
        raise ValueError("q, k, v must share [batch, time, head], and q and k the key width")
    dtype = q.dtype
    if k.dtype != dtype or v.dtype != dtype:
        raise TypeError("q, k and v must have one dtype")
    gs = g.shape
    if gs != (B, T, H) and gs != (H,):
        raise ValueError(f"g must have shape {(B, T, H)} or {(H,)} (got {tuple(g.shape)})")
    if valid is not None and valid.shape != (B, T):
        raise ValueError(f"valid must be [batch, time] (got {tuple(valid.shape)})")
    if reset is not None and reset.shape != (B, T):
        raise ValueError(f"reset must be [batch, time] (got {tuple(reset.shape)})")
    if state is not None and state.shape != (B, H, K, V):
        raise ValueError(f"{state_name} must be [batch, head, key, value] (got "
                         f"{tuple(state.shape)})")
    _same_device(q, "k v g valid reset " + state_name, k, v, g, valid, reset, state)
    if g.dtype != F32:
        g = g.float()
    if valid is not None and valid.dtype != F32:
        valid = valid.float()
    if reset is not None and reset.dtype != F32:
        reset = reset.float()
    gv = _view(g) if g.dim() == 3 else _VIEW(g.data_ptr(), GDN2_F32, 0, 0, 0, g.stride(0), 0)
    views = (_view(q), _view(k), _view(v), gv, _view(valid), _view(reset))
    return code, (B, T, H, K, V), views, (g, valid, reset)


def _initial(state):
    """The initial state as the library reads it: float32, and copied where rows or columns lie further
    apart than its 32-bit offsets reach."""
    if state is None:
        return None
    if state.dtype != F32:
        state = state.float()
    st = state.stride()
    if st[2] >= 1 << 22 or st[3] >= 1 << 22:
        return state.clone(memory_format=torch.contiguous_format)
    return state


def _bytes(query: str, q, v, *args) -> int:
    """A buffer's size, remembered by shape."""
    n = _size(query, _shape(q, v), *args)
    if n == 0:
        check(query, 2)
    return n


def linear_attention_forward(q, k, v, g, valid=None, reset=None, initial=None,
                             train: bool = True):
    """Raw forward.  Returns (output, final_state, checkpoint); the checkpoint is
    private storage for linear_attention_backward, without train scratch alone."""
    code, shape, views, held = _attention_inputs(q, k, v, g, valid, reset, initial)
    initial = _initial(initial)
    B, T, H, K, V = shape
    dev = q.device
    n = _bytes("gdn2_linear_checkpoint_bytes", q, v, code, 1 if train else 0)
    out = torch.empty((B, T, H, V), dtype=q.dtype, device=dev)
    final = torch.empty((B, H, K, V), dtype=F32, device=dev)
    ck = torch.empty((n,), dtype=torch.uint8, device=dev)
    _call("gdn2_linear_scan", dev, _SHAPE(*shape), *views, _view(initial), out.data_ptr(),
          final.data_ptr(), 1 if train else 0, ck.data_ptr(), n)
    return out, final, ck


def linear_attention_backward(q, k, v, g, valid, reset, initial, checkpoint, d_output,
                              d_final_state=None, wanted=(True,) * 5):
    """Raw VJP, from the forward's inputs and checkpoint.  Returns (dq, dk, dv, dg,
    d_initial): dg in g's shape, d_initial None without an initial state.  wanted
    (dq, dk, dv, dg, d_initial): those that are False are None, and not computed."""
    code, shape, views, held = _attention_inputs(q, k, v, g, valid, reset, initial)
    initial = _initial(initial)
    B, T, H, K, V = shape
    dev = q.device
    if d_output.shape != v.shape:
        raise ValueError(f"d_output must have shape {tuple(v.shape)} (got {tuple(d_output.shape)})")
    if d_final_state is not None and d_final_state.shape != (B, H, K, V):
        raise ValueError("d_final_state must be [batch, head, key, value]")
    _same_device(q, "d_output d_final_state checkpoint", d_output, d_final_state, checkpoint)
    if d_output.dtype != q.dtype:
        d_output = d_output.to(q.dtype)
    if d_final_state is not None:
        d_final_state = d_final_state.to(F32).contiguous()
    dq, dk, dv = (torch.empty(t.shape, dtype=t.dtype, device=dev) if w else None
                  for t, w in zip((q, k, v), wanted))
    per_head = g.dim() == 1
    dg = torch.empty(g.shape, dtype=F32, device=dev) if wanted[3] else None
    di = torch.empty((B, H, K, V), dtype=F32, device=dev) \
        if wanted[4] and initial is not None else None
    n = _bytes("gdn2_linear_workspace_bytes", q, v, code)
    ws = torch.empty((n,), dtype=torch.uint8, device=dev)
    _call("gdn2_linear_backward", dev, _SHAPE(*shape), *views, _view(initial),
          checkpoint.data_ptr(), checkpoint.numel(), _view(d_output), _ptr(d_final_state),
          _ptr(dq), _ptr(dk), _ptr(dv), None if per_head else _ptr(dg),
          _ptr(dg) if per_head else None, _ptr(di), ws.data_ptr(), n)
    return dq, dk, dv, dg, di


class _LinearAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, g, valid, reset, initial):
        out, final, ck = linear_attention_forward(q, k, v, g, valid, reset, initial)
        ctx.set_materialize_grads(False)  # an unused output reaches backward as None
        ctx.save_for_backward(q, k, v, g, valid, reset, initial, ck)
        return out, final

    @staticmethod
    @once_differentiable
    def backward(ctx, d_out, d_final):
        q, k, v, g, valid, reset, initial, ck = ctx.saved_tensors
        if d_out is None and d_final is None:
            return (None,) * 7
        if d_out is None:
            d_out = torch.zeros((), dtype=q.dtype, device=q.device).expand(v.shape)
        need = ctx.needs_input_grad
        dq, dk, dv, dg, di = linear_attention_backward(q, k, v, g, valid, reset, initial, ck, d_out,
                                                       d_final, need[:4] + (need[6],))
        return (dq, dk, dv, None if dg is None else dg.to(g.dtype), None, None,
                None if di is None else di.to(initial.dtype))


def linear_attention(q, k, v, g, valid=None, reset=None, initial=None):
    """Linear attention with a decay for each head, per valid token
        S = exp(g) S + k v^T,  out = S^T q
    q, k [B, T, H, K], v [B, T, H, V] (float32 or bfloat16, one dtype, K and V up to 128); g the log
    decay, [B, T, H] or one a head [H]; valid, reset [B, T] float 0/1 or None: padding keeps the state
    and gives zero, a reset on a valid token empties the state before it; initial [B, H, K, V] or None
    (zero).  Returns (output [B, T, H, V] in q's dtype, final_state [B, H, K, V] float32),
    differentiable in q, k, v, g and initial.  Sums and states are float32."""
    for name, m in (("valid", valid), ("reset", reset)):
        if m is not None and m.requires_grad:
            raise ValueError(f"{name} is nondifferentiable metadata")
    if not _differentiates(q, k, v, g, initial):
        return linear_attention_forward(q, k, v, g, valid, reset, initial, False)[:2]
    return _LinearAttention.apply(q, k, v, g, valid, reset, initial)


def linear_attention_step(state, q, k, v, g, valid=None, reset=None):
    """One token per sequence on a carried state, updated in place: state [B, H, K, V] float32
    contiguous; q, k [B, 1, H, K], v [B, 1, H, V], g [B, 1, H] or [H], valid, reset [B, 1] or None.
    Returns the output [B, 1, H, V] in q's dtype.  It has no gradient: where one is recorded, inputs
    that require one are refused, and autograd is told that the state has changed."""
    if state.dtype != F32 or not state.is_contiguous():
        raise ValueError("state must be a contiguous float32 [B, H, K, V] tensor")
    if _wants_grad(state, q, k, v, g) or _has_tangent(state, q, k, v, g):
        raise ValueError("linear_attention_step has no gradient: call it under torch.no_grad(), or on "
                         "detached inputs")
    _, shape, views, held = _attention_inputs(q, k, v, g, valid, reset, state, "state")
    out = torch.empty(v.shape, dtype=q.dtype, device=q.device)
    _call("gdn2_linear_step", q.device, _SHAPE(*shape), *views, state.data_ptr(), out.data_ptr())
    increment_version(state)
    return out


# ---- layer norm ----------------------------------------------------------------------------


def _rows(x: torch.Tensor) -> torch.Tensor:
    """x as [B, T, H, W] without a copy where at most three row axes remain."""
    if x.dim() > 4:
        return x.reshape(1, 1, -1, x.shape[-1])
    while x.dim() < 4:
        x = x.unsqueeze(0)
    return x


def _row_views(*tensors):
    """The shape of the rows of tensors of one shape, and their views."""
    W = tensors[0].shape[-1]
    if all(t.is_contiguous() for t in tensors):
        rows = tensors[0].numel() // W
        return (1, 1, rows, W), [_VIEW(t.data_ptr(), _CODES[t.dtype], 0, 0, 0, W, 1)
                                 for t in tensors]
    held = [_rows(t) for t in tensors]
    return tuple(held[0].shape), [_view(t) for t in held], held


def _ln_inputs(x, weight, bias):
    _dtype(x, "x")
    W = x.shape[-1] if x.dim() else 0
    if W < 1:
        raise ValueError("x must be [..., W] with W >= 1")
    for t in (weight, bias):
        if t is not None and (t.dtype != F32 or t.shape != (W,)):
            raise ValueError(f"{'weight' if t is weight else 'bias'} must be float32 [{W}] (got "
                             f"{t.dtype} {tuple(t.shape)})")
    _same_device(x, "weight bias", weight, bias)
    return weight.contiguous(), None if bias is None else bias.contiguous()


def _ln_forward(x, weight, bias, epsilon, stats):
    weight, bias = _ln_inputs(x, weight, bias)
    shape, (view,), *held = _row_views(x)
    dev = x.device
    y = torch.empty(x.shape, dtype=x.dtype, device=dev)
    mean = inv = None
    if stats:
        rows = shape[0] * shape[1] * shape[2]
        mean = torch.empty((rows,), dtype=F32, device=dev)
        inv = torch.empty((rows,), dtype=F32, device=dev)
    _call("gdn2_layer_norm_forward", dev, _ROWS(*shape), epsilon, view, weight.data_ptr(),
          _ptr(bias), y.data_ptr(), _ptr(mean), _ptr(inv))
    return y, mean, inv


def layer_norm_forward(x, weight, bias=None, epsilon: float = 1e-5):
    """Raw forward.  Returns (y, mean [rows], inverse [rows])."""
    return _ln_forward(x, weight, bias, epsilon, True)


def layer_norm_backward(x, weight, mean, inverse, dy, want_bias: bool = True,
                        want_x: bool = True, want_weight: bool = True):
    """Raw VJP.  Returns (dx, dweight, dbias); those not wanted are None."""
    weight, _ = _ln_inputs(x, weight, None)
    if dy.shape != x.shape:
        raise ValueError(f"dy must have x's shape {tuple(x.shape)} (got {tuple(dy.shape)})")
    if dy.dtype != x.dtype:
        dy = dy.to(x.dtype)
    dev, W = x.device, x.shape[-1]
    shape, (xv, dyv), *held = _row_views(x, dy)
    rows = shape[0] * shape[1] * shape[2]
    for name, t in (("mean", mean), ("inverse", inverse)):
        if t.dtype != F32 or t.numel() != rows or not t.is_contiguous():
            raise ValueError(f"{name} must be contiguous float32 [{rows}]")
    _same_device(x, "mean inverse dy", mean, inverse, dy)
    dx = torch.empty(x.shape, dtype=x.dtype, device=dev) if want_x else None
    dw = torch.empty((W,), dtype=F32, device=dev) if want_weight else None
    db = torch.empty((W,), dtype=F32, device=dev) if want_bias else None
    n = lib().gdn2_layer_norm_workspace_bytes(rows, W)
    ws = torch.empty((n,), dtype=torch.uint8, device=dev)
    _call("gdn2_layer_norm_backward", dev, _ROWS(*shape), xv, weight.data_ptr(), mean.data_ptr(),
          inverse.data_ptr(), dyv, _ptr(dx), _ptr(dw), _ptr(db), ws.data_ptr(), n)
    return dx, dw, db


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, epsilon):
        y, mean, inv = _ln_forward(x, weight, bias, epsilon, True)
        ctx.save_for_backward(x, weight, mean, inv)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, weight, mean, inv = ctx.saved_tensors
        need = ctx.needs_input_grad
        dx, dw, db = layer_norm_backward(x, weight, mean, inv, dy, need[2], need[0], need[1])
        return dx, dw, db, None


def layer_norm(x, weight, bias=None, epsilon: float = 1e-5):
    """Layer norm over the last axis: weight (x - mean) / sqrt(var + epsilon) + bias, x [..., W]
    float32 or bfloat16, weight and bias [W] float32 (bias may be None).  The output has x's shape and
    dtype; statistics and sums are float32.  Differentiable in x, weight and bias."""
    if not _differentiates(x, weight, bias):
        return _ln_forward(x, weight, bias, epsilon, False)[0]
    return _LayerNorm.apply(x, weight, bias, float(epsilon))


# ---- SwiGLU with its input in 8 bits -------------------------------------------------------------


def _dense(t: torch.Tensor, name: str, dtype, shape) -> torch.Tensor:
    if t.dtype != dtype or t.shape != shape:
        raise ValueError(f"{name} must be {dtype} {tuple(shape)} (got {t.dtype} {tuple(t.shape)})")
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")
    return t


def swiglu_q8_forward(h: torch.Tensor):
    """h [rows, 2 M] = [gate | up], contiguous -> (a = silu(gate) up [rows, M], codes int8
    [rows, 2 M], exponents uint8 [rows, 2 ceil(M / 32)]).  The last two stand for h in the backward."""
    code = _dtype(h, "h")
    if h.dim() != 2 or h.shape[1] % 2 or h.shape[1] < 2:
        raise ValueError("h must be [rows, 2 M]")
    _dense(h, "h", h.dtype, h.shape)
    rows, M = h.shape[0], h.shape[1] // 2
    a = torch.empty((rows, M), dtype=h.dtype, device=h.device)
    codes = torch.empty((rows, 2 * M), dtype=torch.int8, device=h.device)
    exps = torch.empty((rows, 2 * -(-M // Q8_BLOCK)), dtype=torch.uint8, device=h.device)
    _call("gdn2_swiglu_q8_forward", h.device, rows, M, code, h.data_ptr(), a.data_ptr(),
          codes.data_ptr(), exps.data_ptr())
    return a, codes, exps


def swiglu_q8_backward(codes: torch.Tensor, exponents: torch.Tensor, da: torch.Tensor,
                       want_a: bool = True):
    """The VJP at the values that codes and exponents stand for: da [rows, M], contiguous ->
    (dh [rows, 2 M], a [rows, M] at those values or None), in da's dtype."""
    code = _dtype(da, "da")
    if da.dim() != 2 or da.shape[1] < 1:
        raise ValueError("da must be [rows, M]")
    rows, M = da.shape
    _dense(da, "da", da.dtype, da.shape)
    _dense(codes, "codes", torch.int8, (rows, 2 * M))
    _dense(exponents, "exponents", torch.uint8, (rows, 2 * -(-M // Q8_BLOCK)))
    _same_device(da, "codes exponents", codes, exponents)
    dh = torch.empty((rows, 2 * M), dtype=da.dtype, device=da.device)
    a = torch.empty((rows, M), dtype=da.dtype, device=da.device) if want_a else None
    _call("gdn2_swiglu_q8_backward", da.device, rows, M, code, codes.data_ptr(),
          exponents.data_ptr(), da.data_ptr(), dh.data_ptr(), _ptr(a))
    return dh, a


def q8_values(codes: torch.Tensor, exponents: torch.Tensor) -> torch.Tensor:
    """The float32 values [rows, 2 M] that codes and exponents stand for (for inspection: the backward
    does not form them)."""
    rows, width = codes.shape
    M = width // 2
    blocks = exponents.view(rows, 2, -(-M // Q8_BLOCK)).to(torch.int32)
    scale = (blocks << 23).view(F32)  # 2^e from its exponent bits
    scale = torch.where(blocks == 255, torch.full_like(scale, float("nan")), scale)
    scale = scale.repeat_interleave(Q8_BLOCK, 2)[:, :, :M]
    return (codes.view(rows, 2, M).to(F32) * scale).view(rows, width)


class _SwigluQ8(torch.autograd.Function):
    @staticmethod
    def forward(ctx, h):
        a, codes, exps = swiglu_q8_forward(h)
        ctx.save_for_backward(codes, exps)
        return a

    @staticmethod
    @once_differentiable
    def backward(ctx, da):
        codes, exps = ctx.saved_tensors
        return swiglu_q8_backward(codes, exps, da.contiguous(), False)[0]


def swiglu_q8(h: torch.Tensor) -> torch.Tensor:
    """silu(gate) * up for h [..., 2 M] = [gate | up], float32 or bfloat16.  Between the passes it keeps
    h in 8 bits (a power of two for every 32 columns): the gradient is taken at the kept values, which
    are off by less than 1/127 of their block's largest magnitude."""
    if h.dim() < 1 or h.shape[-1] % 2 or h.shape[-1] < 2:
        raise ValueError("h must be [..., 2 M]")
    rows = h.reshape(-1, h.shape[-1]).contiguous()
    a = _SwigluQ8.apply(rows) if _differentiates(h) else swiglu_q8_forward(rows)[0]
    return a.view(h.shape[:-1] + (h.shape[-1] // 2,))
