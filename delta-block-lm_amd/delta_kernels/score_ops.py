"""Scores of given tokens on the HIP library (include/gdn2.h).

  token_log_probs(logits, tokens, top, ...)   log probabilities of given tokens, the entropy of their
                                              distributions, and the top alternatives

The log probability is the negative of cross_entropy_rows; entropy and alternatives have no
counterpart in the reference.  Log probabilities and entropy are differentiable in the logits, once
and in reverse mode (anything else is refused); token_log_probs_forward and _backward are the raw
calls.  All run only on the GPU: there is no CPU fallback.
"""
from __future__ import annotations

from typing import NamedTuple, Optional

import torch

from ._lib import lib
from ._once import once
from .linear_ops import (_CODES, F32, _VIEW, _call, _differentiates, _dtype, _ptr, _same_device)

__all__ = ["TokenLogProbs", "token_log_probs", "token_log_probs_forward", "token_log_probs_backward"]

MAX_TOP = 64


class TokenLogProbs(NamedTuple):
    log_probs: torch.Tensor  # [...] float32
    entropy: torch.Tensor  # [...] float32
    top_log_probs: Optional[torch.Tensor]  # [..., top] float32, None without alternatives
    top_tokens: Optional[torch.Tensor]  # [..., top] int64


def _inputs(x, tokens, valid, temperature):
    """Checked inputs as rows: (rows, width, packed view, tokens, valid, what they look at)."""
    _dtype(x, "logits")
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError("logits must be [..., width] with width >= 1")
    lead = x.shape[:-1]
    if tokens.dtype != torch.int64:
        raise TypeError("tokens must hold int64 ids")
    for name, t in (("tokens", tokens), ("valid", valid)):
        if t is not None and t.shape != lead:
            raise ValueError(f"{name} must have shape {tuple(lead)} (got {tuple(t.shape)})")
    _same_device(x, "tokens valid", tokens, valid)
    if not 0 < temperature < float("inf"):
        raise ValueError(f"temperature must be positive and finite (got {temperature})")
    x = x if x.dim() == 2 else x.reshape(-1, x.shape[-1])
    tokens = tokens if tokens.dim() == 1 else tokens.reshape(-1)
    if valid is not None:
        valid = (valid if valid.dtype == F32 else valid.float()).reshape(-1)
    view = _VIEW(x.data_ptr(), _CODES[x.dtype], 0, *x.stride(), 0, 0)
    return x.shape[0], x.shape[1], view, tokens, valid, x


def _stride(t):
    return 0 if t is None or t.numel() < 2 else t.stride(0)


def _forward(x, tokens, top, valid, temperature, stats):
    rows, width, view, tokens, valid, held = _inputs(x, tokens, valid, temperature)
    if not 0 <= top <= min(MAX_TOP, width):
        raise ValueError(f"top must be 0 to {min(MAX_TOP, width)} (got {top})")
    dev, lead = x.device, x.shape[:-1]
    lp = torch.empty(lead, dtype=F32, device=dev)
    entropy = torch.empty(lead, dtype=F32, device=dev)
    top_lp = top_tokens = None
    if top:
        top_lp = torch.empty(lead + (top,), dtype=F32, device=dev)
        top_tokens = torch.empty(lead + (top,), dtype=torch.int64, device=dev)
    stats = torch.empty((rows, 3), dtype=F32, device=dev) if stats else None
    ws, n = None, 0
    if rows <= 64 and width >= 65536:  # few wide rows, whose parts are joined
        n = lib().gdn2_token_score_workspace_bytes(rows, width, top)
        ws = torch.empty((n,), dtype=torch.uint8, device=dev) if n else None
    _call("gdn2_token_score_forward", dev, rows, width, view, tokens.data_ptr(), _stride(tokens),
          _ptr(valid), _stride(valid), temperature, top, lp.data_ptr(), entropy.data_ptr(),
          _ptr(top_lp), _ptr(top_tokens), _ptr(stats), _ptr(ws), n)
    return TokenLogProbs(lp, entropy, top_lp, top_tokens), stats


def token_log_probs_forward(logits, tokens, top: int = 0, valid=None, temperature: float = 1.0):
    """Raw forward.  Returns (TokenLogProbs, stats [rows, 3]): the stats are what
    token_log_probs_backward reads of the forward."""
    return _forward(logits, tokens, top, valid, temperature, True)


def token_log_probs_backward(logits, tokens, valid, temperature, stats, d_log_probs=None,
                             d_entropy=None):
    """Raw VJP, from the forward's inputs and stats.  d_log_probs and d_entropy [...] float32 or None
    (zero).  Returns the logits' gradient in their shape and dtype."""
    rows, width, view, tokens, valid, held = _inputs(logits, tokens, valid, temperature)
    if stats.dtype != F32 or stats.shape != (rows, 3) or not stats.is_contiguous():
        raise ValueError(f"stats must be contiguous float32 {(rows, 3)}")
    ups = []
    for name, t in (("d_log_probs", d_log_probs), ("d_entropy", d_entropy)):
        if t is not None and t.shape != logits.shape[:-1]:
            raise ValueError(f"{name} must have shape {tuple(logits.shape[:-1])} (got {tuple(t.shape)})")
        ups.append(None if t is None else t.to(F32).reshape(-1))
    _same_device(logits, "stats d_log_probs d_entropy", stats, *ups)
    dx = torch.empty(logits.shape, dtype=logits.dtype, device=logits.device)
    _call("gdn2_token_score_backward", logits.device, rows, width, view, tokens.data_ptr(),
          _stride(tokens), _ptr(valid), _stride(valid), temperature, stats.data_ptr(), _ptr(ups[0]),
          _stride(ups[0]), _ptr(ups[1]), _stride(ups[1]), dx.data_ptr())
    return dx


class _TokenLogProbs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, tokens, top, valid, temperature):
        r, stats = _forward(x, tokens, top, valid, temperature, True)
        ctx.save_for_backward(x, tokens, valid, stats)
        ctx.temperature = temperature
        ctx.set_materialize_grads(False)  # an unused output reaches backward as None
        if top:
            ctx.mark_non_differentiable(r.top_log_probs, r.top_tokens)
        return tuple(r)

    @staticmethod
    @once
    def backward(ctx, d_lp, d_entropy, *_):
        x, tokens, valid, stats = ctx.saved_tensors
        if d_lp is None and d_entropy is None:
            return (None,) * 5
        return (token_log_probs_backward(x, tokens, valid, ctx.temperature, stats, d_lp, d_entropy),
                None, None, None, None)


def token_log_probs(logits, tokens, top: int = 0, valid=None,
                    temperature: float = 1.0) -> TokenLogProbs:
    """Log probabilities of given tokens under softmax(logits / temperature): logits [..., width] float32
    or bfloat16, tokens [...] int64, valid [...] float 0/1 or None (a row that is not valid is not read
    and gives zeros).  Returns log_probs and entropy [...] float32, differentiable in the logits, and,
    for top > 0 (64 at most), the largest logits' log probabilities and ids [..., top], largest first
    and the lower id first among equal ones, without gradients.  A token outside [0, width) gives NaN;
    a logit of -inf is probability 0."""
    if valid is not None and valid.requires_grad:
        raise ValueError("valid is nondifferentiable metadata")
    if not _differentiates(logits):
        return _forward(logits, tokens, top, valid, temperature, False)[0]
    return TokenLogProbs(*_TokenLogProbs.apply(logits, tokens, top, valid, temperature))
