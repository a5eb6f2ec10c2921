"""Operators of a linear-attention block on the HIP library (include/gdn2.h).

  linear_attention(q, k, v, g, ...)    linear attention with a decay for each head: chunked, for
                                       training and prompts
  linear_attention_step(state, ...)    its recurrent form, one token on a carried state
  layer_norm(x, weight, bias)          layer norm over the last axis
  swiglu_q8(h)                         SwiGLU that keeps its input in 8 bits for the backward

They have no counterpart in the reference.  The first form of each is differentiable;
*_forward and *_backward are the raw calls, for a block that writes its backward out
(delta_mixers.linear).  All run only on the GPU: there is no CPU fallback.
"""
from __future__ import annotations

import ctypes
from typing import Optional

import torch

from ._lib import GDN2_BF16, GDN2_F32, Gdn2RowsShape, check, lib, on_device

__all__ = ["linear_attention", "linear_attention_forward", "linear_attention_backward",
           "linear_attention_step", "layer_norm", "layer_norm_forward", "layer_norm_backward",
           "swiglu_q8", "swiglu_q8_forward", "swiglu_q8_backward", "q8_values"]

F32, BF16 = torch.float32, torch.bfloat16
Q8_BLOCK = 32  # columns that share an exponent


def _helpers():
    from . import _ptr, _shape, _stream, _view  # the package's view/pointer/stream adapters
    return _view, _ptr, _stream, _shape


def _dtype(t: torch.Tensor, name: str) -> int:
    if t.dtype not in (F32, BF16):
        raise TypeError(f"{name} must be float32 or bfloat16 (got {t.dtype})")
    if not t.is_cuda:
        raise ValueError(f"{name} must live on the GPU; there is no CPU fallback")
    return GDN2_BF16 if t.dtype == BF16 else GDN2_F32


def _same_device(like: torch.Tensor, **tensors) -> None:
    for name, t in tensors.items():
        if t is not None and t.device != like.device:
            raise ValueError(f"{name} must live on {like.device} (got {t.device})")


# ---- linear attention ------------------------------------------------------------------


def _attention_inputs(q, k, v, g, valid, reset, state=None, state_name="initial"):
    """Checked inputs; g as a [B, T, H] view, masks and gates as float32."""
    _dtype(q, "q")
    if q.dim() != 4 or v.dim() != 4:
        raise ValueError("q must be [batch, time, head, key] and v [batch, time, head, value]")
    B, T, H, K = q.shape
    V = v.shape[3]
    if k.shape != q.shape or v.shape[:3] != q.shape[:3]:
        raise ValueError("q, k, v must share [batch, time, head], and q and k the key width")
    if k.dtype != q.dtype or v.dtype != q.dtype:
        raise TypeError("q, k and v must have one dtype")
    if tuple(g.shape) not in ((B, T, H), (H,)):
        raise ValueError(f"g must have shape {(B, T, H)} or {(H,)} (got {tuple(g.shape)})")
    for name, m in (("valid", valid), ("reset", reset)):
        if m is not None and tuple(m.shape) != (B, T):
            raise ValueError(f"{name} must be [batch, time] (got {tuple(m.shape)})")
    if state is not None and tuple(state.shape) != (B, H, K, V):
        raise ValueError(f"{state_name} must be [batch, head, key, value] (got "
                         f"{tuple(state.shape)})")
    _same_device(q, k=k, v=v, g=g, valid=valid, reset=reset, **{state_name: state})
    g = g if g.dtype == F32 else g.float()
    if g.dim() == 1:
        g = g.expand(B, T, H)
    valid, reset = (m if m is None or m.dtype == F32 else m.to(F32) for m in (valid, reset))
    return g, valid, reset


def _ref(view):
    return None if view is None else ctypes.byref(view)


def _views(q, k, v, g, valid, reset, initial):
    _view = _helpers()[0]
    vs = [_view(t) for t in (q, k, v, g)]
    return vs + [None if t is None else _view(t) for t in (valid, reset, initial)]


def linear_attention_forward(q, k, v, g, valid=None, reset=None, initial=None):
    """Raw forward.  Returns (output, final_state, checkpoint); the checkpoint is
    private storage for linear_attention_backward."""
    _, _ptr, _stream, _shape = _helpers()
    g, valid, reset = _attention_inputs(q, k, v, g, valid, reset, initial)
    if initial is not None and initial.dtype != F32:
        initial = initial.float()
    L = lib()
    shape = _shape(q, v)
    B, T, H, K = q.shape
    V = v.shape[3]
    dev = q.device
    code = _dtype(q, "q")
    n = L.gdn2_linear_checkpoint_bytes(ctypes.byref(shape), code)
    if n == 0:
        check("gdn2_linear_checkpoint_bytes", 2)
    out = torch.empty((B, T, H, V), dtype=q.dtype, device=dev)
    final = torch.empty((B, H, K, V), dtype=F32, device=dev)
    ck = torch.empty((n,), dtype=torch.uint8, device=dev)
    views = _views(q, k, v, g, valid, reset, initial)
    with on_device(dev):
        rc = L.gdn2_linear_scan(ctypes.byref(shape), *[_ref(x) for x in views], _ptr(out),
                                _ptr(final), _ptr(ck), n, _stream(q))
    check("gdn2_linear_scan", rc)
    return out, final, ck


def linear_attention_backward(q, k, v, g, valid, reset, initial, checkpoint, d_output,
                              d_final_state=None, wanted=(True,) * 5):
    """Raw VJP, from the forward's inputs and checkpoint.  Returns (dq, dk, dv, dg,
    d_initial): dg in g's shape, d_initial None without an initial state.  wanted
    (dq, dk, dv, dg, d_initial): those that are False are None, and not computed."""
    _view, _ptr, _stream, _shape = _helpers()
    per_head = g.dim() == 1
    g, valid, reset = _attention_inputs(q, k, v, g, valid, reset, initial)
    if initial is not None and initial.dtype != F32:
        initial = initial.float()
    L = lib()
    shape = _shape(q, v)
    B, T, H, K = q.shape
    V = v.shape[3]
    dev = q.device
    if tuple(d_output.shape) != (B, T, H, V):
        raise ValueError(f"d_output must have shape {(B, T, H, V)} (got {tuple(d_output.shape)})")
    if d_final_state is not None and tuple(d_final_state.shape) != (B, H, K, V):
        raise ValueError("d_final_state must be [batch, head, key, value]")
    _same_device(q, d_output=d_output, d_final_state=d_final_state, checkpoint=checkpoint)
    if d_output.dtype != q.dtype:
        d_output = d_output.to(q.dtype)
    if d_final_state is not None:
        d_final_state = d_final_state.to(F32).contiguous()
    dq, dk, dv = (torch.empty(t.shape, dtype=t.dtype, device=dev) if w else None
                  for t, w in zip((q, k, v), wanted))
    dg = torch.empty((H,) if per_head else (B, T, H), dtype=F32, device=dev) if wanted[3] else None
    di = torch.empty((B, H, K, V), dtype=F32, device=dev) \
        if wanted[4] and initial is not None else None
    n = L.gdn2_linear_workspace_bytes(ctypes.byref(shape), _dtype(q, "q"))
    if n == 0:
        check("gdn2_linear_workspace_bytes", 2)
    ws = torch.empty((n,), dtype=torch.uint8, device=dev)
    views = _views(q, k, v, g, valid, reset, initial)
    dov = _view(d_output)
    with on_device(dev):
        rc = L.gdn2_linear_backward(
            ctypes.byref(shape), *[_ref(x) for x in views], _ptr(checkpoint), checkpoint.numel(),
            ctypes.byref(dov), _ptr(d_final_state), _ptr(dq), _ptr(dk), _ptr(dv),
            None if per_head else _ptr(dg), _ptr(dg) if per_head else None, _ptr(di), _ptr(ws), n,
            _stream(q))
    check("gdn2_linear_backward", rc)
    return dq, dk, dv, dg, di


class _LinearAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, g, valid, reset, initial):
        out, final, ck = linear_attention_forward(q, k, v, g, valid, reset, initial)
        ctx.set_materialize_grads(False)  # an unused output reaches backward as None
        ctx.save_for_backward(q, k, v, g, valid, reset, initial, ck)
        return out, final

    @staticmethod
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
    return _LinearAttention.apply(q, k, v, g, valid, reset, initial)


def linear_attention_step(state, q, k, v, g, valid=None, reset=None):
    """One token per sequence on a carried state, updated in place: state [B, H, K, V] float32
    contiguous; q, k [B, 1, H, K], v [B, 1, H, V], g [B, 1, H] or [H], valid, reset [B, 1] or None.
    Returns the output [B, 1, H, V] in q's dtype.  Without gradients."""
    _, _ptr, _stream, _shape = _helpers()
    if state.dtype != F32 or not state.is_contiguous():
        raise ValueError("state must be a contiguous float32 [B, H, K, V] tensor")
    g, valid, reset = _attention_inputs(q, k, v, g, valid, reset, state, "state")
    shape = _shape(q, v)
    out = torch.empty(v.shape, dtype=q.dtype, device=q.device)
    views = _views(q, k, v, g, valid, reset, None)[:6]
    with on_device(q.device):
        rc = lib().gdn2_linear_step(ctypes.byref(shape), *[_ref(x) for x in views], _ptr(state),
                                    _ptr(out), _stream(q))
    check("gdn2_linear_step", rc)
    return out


# ---- layer norm ----------------------------------------------------------------------------


def _rows(x: torch.Tensor) -> torch.Tensor:
    """x as [B, T, H, W] without a copy where at most three row axes remain."""
    if x.dim() > 4 or x.is_contiguous():
        return x.reshape(1, 1, -1, x.shape[-1])
    while x.dim() < 4:
        x = x.unsqueeze(0)
    return x


def _ln_inputs(x, weight, bias):
    _dtype(x, "x")
    W = x.shape[-1] if x.dim() else 0
    if W < 1:
        raise ValueError("x must be [..., W] with W >= 1")
    for name, t in (("weight", weight), ("bias", bias)):
        if t is None and name == "bias":
            continue
        if t.dtype != F32 or tuple(t.shape) != (W,):
            raise ValueError(f"{name} must be float32 [{W}] (got {t.dtype} {tuple(t.shape)})")
    _same_device(x, weight=weight, bias=bias)
    return weight.contiguous(), None if bias is None else bias.contiguous()


def _ln_forward(x, weight, bias, epsilon, stats):
    _view, _ptr, _stream, _ = _helpers()
    weight, bias = _ln_inputs(x, weight, bias)
    x4 = _rows(x)
    rows = x4.shape[0] * x4.shape[1] * x4.shape[2]
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    mean, inv = (torch.empty((rows,), dtype=F32, device=x.device) if stats else None
                 for _ in range(2))
    shape = Gdn2RowsShape(*x4.shape)
    with on_device(x.device):
        rc = lib().gdn2_layer_norm_forward(ctypes.byref(shape), epsilon, ctypes.byref(_view(x4)),
                                           _ptr(weight), _ptr(bias), _ptr(y), _ptr(mean),
                                           _ptr(inv), _stream(x))
    check("gdn2_layer_norm_forward", rc)
    return y, mean, inv


def layer_norm_forward(x, weight, bias=None, epsilon: float = 1e-5):
    """Raw forward.  Returns (y, mean [rows], inverse [rows])."""
    return _ln_forward(x, weight, bias, epsilon, True)


def layer_norm_backward(x, weight, mean, inverse, dy, want_bias: bool = True,
                        want_x: bool = True, want_weight: bool = True):
    """Raw VJP.  Returns (dx, dweight, dbias); those not wanted are None."""
    _view, _ptr, _stream, _ = _helpers()
    weight, _ = _ln_inputs(x, weight, None)
    if dy.shape != x.shape:
        raise ValueError(f"dy must have x's shape {tuple(x.shape)} (got {tuple(dy.shape)})")
    if dy.dtype != x.dtype:
        dy = dy.to(x.dtype)
    x4, dy4 = _rows(x), _rows(dy)
    if x4.shape != dy4.shape:  # one of them is contiguous, and flattened
        x4, dy4 = (t.reshape(1, 1, -1, x.shape[-1]) for t in (x, dy))
    rows, W = x4.shape[0] * x4.shape[1] * x4.shape[2], x.shape[-1]
    for name, t in (("mean", mean), ("inverse", inverse)):
        if t.dtype != F32 or t.numel() != rows or not t.is_contiguous():
            raise ValueError(f"{name} must be contiguous float32 [{rows}]")
    _same_device(x, mean=mean, inverse=inverse, dy=dy)
    dx = torch.empty(x.shape, dtype=x.dtype, device=x.device) if want_x else None
    dw, db = (torch.empty((W,), dtype=F32, device=x.device) if w else None
              for w in (want_weight, want_bias))
    L = lib()
    n = L.gdn2_layer_norm_workspace_bytes(rows, W)
    ws = torch.empty((n,), dtype=torch.uint8, device=x.device)
    shape = Gdn2RowsShape(*x4.shape)
    with on_device(x.device):
        rc = L.gdn2_layer_norm_backward(ctypes.byref(shape), ctypes.byref(_view(x4)), _ptr(weight),
                                        _ptr(mean), _ptr(inverse), ctypes.byref(_view(dy4)),
                                        _ptr(dx), _ptr(dw), _ptr(db), _ptr(ws), n, _stream(x))
    check("gdn2_layer_norm_backward", rc)
    return dx, dw, db


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, epsilon, grad):
        y, mean, inv = _ln_forward(x, weight, bias, epsilon, grad and any(ctx.needs_input_grad))
        ctx.save_for_backward(x, weight, mean, inv)
        return y

    @staticmethod
    def backward(ctx, dy):
        x, weight, mean, inv = ctx.saved_tensors
        need = ctx.needs_input_grad
        dx, dw, db = layer_norm_backward(x, weight, mean, inv, dy, need[2], need[0], need[1])
        return dx, dw, db, None, None


def layer_norm(x, weight, bias=None, epsilon: float = 1e-5):
    """Layer norm over the last axis: weight (x - mean) / sqrt(var + epsilon) + bias, x [..., W]
    float32 or bfloat16, weight and bias [W] float32 (bias may be None).  The output has x's shape and
    dtype; statistics and sums are float32.  Differentiable in x, weight and bias."""
    return _LayerNorm.apply(x, weight, bias, float(epsilon), torch.is_grad_enabled())


# ---- SwiGLU with its input in 8 bits -------------------------------------------------------------


def _dense(t: torch.Tensor, name: str, dtype, shape) -> torch.Tensor:
    if t.dtype != dtype or tuple(t.shape) != tuple(shape):
        raise ValueError(f"{name} must be {dtype} {tuple(shape)} (got {t.dtype} {tuple(t.shape)})")
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")
    return t


def swiglu_q8_forward(h: torch.Tensor):
    """h [rows, 2 M] = [gate | up], contiguous -> (a = silu(gate) up [rows, M], codes int8
    [rows, 2 M], exponents uint8 [rows, 2 ceil(M / 32)]).  The last two stand for h in the backward."""
    _, _ptr, _stream, _ = _helpers()
    code = _dtype(h, "h")
    if h.dim() != 2 or h.shape[1] % 2 or h.shape[1] < 2:
        raise ValueError("h must be [rows, 2 M]")
    _dense(h, "h", h.dtype, h.shape)
    rows, M = h.shape[0], h.shape[1] // 2
    a = torch.empty((rows, M), dtype=h.dtype, device=h.device)
    codes = torch.empty((rows, 2 * M), dtype=torch.int8, device=h.device)
    exps = torch.empty((rows, 2 * -(-M // Q8_BLOCK)), dtype=torch.uint8, device=h.device)
    with on_device(h.device):
        rc = lib().gdn2_swiglu_q8_forward(rows, M, code, _ptr(h), _ptr(a), _ptr(codes), _ptr(exps),
                                          _stream(h))
    check("gdn2_swiglu_q8_forward", rc)
    return a, codes, exps


def swiglu_q8_backward(codes: torch.Tensor, exponents: torch.Tensor, da: torch.Tensor,
                       want_a: bool = True):
    """The VJP at the values that codes and exponents stand for: da [rows, M], contiguous ->
    (dh [rows, 2 M], a [rows, M] at those values or None), in da's dtype."""
    _, _ptr, _stream, _ = _helpers()
    code = _dtype(da, "da")
    if da.dim() != 2 or da.shape[1] < 1:
        raise ValueError("da must be [rows, M]")
    rows, M = da.shape
    _dense(da, "da", da.dtype, da.shape)
    _dense(codes, "codes", torch.int8, (rows, 2 * M))
    _dense(exponents, "exponents", torch.uint8, (rows, 2 * -(-M // Q8_BLOCK)))
    _same_device(da, codes=codes, exponents=exponents)
    dh = torch.empty((rows, 2 * M), dtype=da.dtype, device=da.device)
    a = torch.empty((rows, M), dtype=da.dtype, device=da.device) if want_a else None
    with on_device(da.device):
        rc = lib().gdn2_swiglu_q8_backward(rows, M, code, _ptr(codes), _ptr(exponents), _ptr(da),
                                           _ptr(dh), _ptr(a), _stream(da))
    check("gdn2_swiglu_q8_backward", rc)
    return dh, a


def q8_values(codes: torch.Tensor, exponents: torch.Tensor) -> torch.Tensor:
    """The float32 values [rows, 2 M] that codes and exponents stand for (for inspection: the backward
    does not form them)."""
    rows, width = codes.shape
    M = width // 2
    blocks = exponents.view(rows, 2, -1).to(torch.int32)
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
    def backward(ctx, da):
        codes, exps = ctx.saved_tensors
        return swiglu_q8_backward(codes, exps, da.contiguous(), False)[0]


def swiglu_q8(h: torch.Tensor) -> torch.Tensor:
    """silu(gate) * up for h [..., 2 M] = [gate | up], float32 or bfloat16.  Between the passes it keeps
    h in 8 bits (a power of two for every 32 columns): the gradient is taken at the kept values, which
    are off by less than 1/127 of their block's largest magnitude."""
    if h.dim() < 1 or h.shape[-1] % 2 or h.shape[-1] < 2:
        raise ValueError("h must be [..., 2 M]")
    return _SwigluQ8.apply(h.reshape(-1, h.shape[-1]).contiguous()).view(
        h.shape[:-1] + (h.shape[-1] // 2,))
