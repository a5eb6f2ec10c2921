"""Orthogonalised updates on the HIP library (include/gdn2.h).

  orthogonalize(x)               Newton-Schulz products of matrices: U V^T of their singular value
                                 decomposition, nearly (singular values of 0.7 to 1.2)
  muon_update(x, g, m, lr, ...)  one Muon update of matrices of one shape, in place
  Muon                           the optimizer: one call for all parameters of a shape

They have no counterpart in the reference, whose optimizer is AdamW (train_ops.FusedAdamW); Muon is for
a model's matrices, next to that for everything else.  All run only on the GPU: there is no CPU fallback.
"""
from __future__ import annotations

import struct
from typing import Sequence, Union

import torch
from torch.autograd.graph import increment_version

from ._lib import check, lib
from .linear_ops import F32, _call, _dtype, _has_tangent, _wants_grad

__all__ = ["orthogonalize", "muon_update", "Muon"]

COEFFICIENTS = (3.4445, -4.7750, 2.0315)  # the quintic's, as published with Muon

_VIEW = struct.Struct("Pii4q").pack
_SHAPE = struct.Struct("3q").pack
_SIZES: dict = {}


def _bytes(shape) -> int:
    """The workspace's size, remembered by shape."""
    n = _SIZES.get(shape)
    if n is None:
        n = lib().gdn2_orthogonalize_workspace_bytes(_SHAPE(*shape))
        if n == 0:
            check("gdn2_orthogonalize_workspace_bytes", 2)
        _SIZES[shape] = n
    return n


def _coefficients(c) -> bytes:
    if len(c) != 3:
        raise ValueError("coefficients must be three numbers")
    return struct.pack("3d", *c)


def orthogonalize(x: torch.Tensor, steps: int = 5, coefficients: Sequence[float] = COEFFICIENTS,
                  epsilon: float = 1e-7) -> torch.Tensor:
    """Newton-Schulz products of the matrices x [..., rows, cols], float32 or bfloat16, any strides:
        X = x / (|x| + epsilon), then `steps` times X <- a X + (b A + c A A) X with A = X X^T
    (for tall matrices the same from the right).  Returns the result in x's shape and dtype; products
    keep 23 bits of their operands (and not the product of the lower halves, 2^-22 of theirs) and sum in
    float32; of a side of at most 64, all bits and sums in float64.  It works in memory of its own: for each
    matrix of a launch 16 to 24 bytes a value, the smaller side counted as 64 at least (1 x 2^24: 17 GB).  It
    has no gradient: where one is recorded, an input that requires one is refused."""
    code = _dtype(x, "x")
    if x.dim() < 2:
        raise ValueError("x must be [..., rows, cols]")
    if _wants_grad(x) or _has_tangent(x):
        raise ValueError("orthogonalize has no gradient: call it under torch.no_grad(), or on a detached "
                         "input")
    held = x.unsqueeze(0) if x.dim() == 2 else x if x.dim() == 3 else x.reshape((-1,) + x.shape[-2:])
    shape = tuple(held.shape)
    dev = x.device
    out = torch.empty(x.shape, dtype=x.dtype, device=dev)
    n = _bytes(shape)
    ws = torch.empty((n,), dtype=torch.uint8, device=dev)
    _call("gdn2_orthogonalize", dev, _SHAPE(*shape), _VIEW(held.data_ptr(), code, 0, *held.stride(), 0),
          out.data_ptr(), steps, _coefficients(coefficients), epsilon, ws.data_ptr(), n)
    return out


Tensors = Union[torch.Tensor, Sequence[torch.Tensor]]


def _list(t: Tensors):
    return [t] if isinstance(t, torch.Tensor) else list(t)


def _overlap(written, read) -> bool:
    """Whether of spans (begin, end) one that is written shares memory with another, of either kind."""
    merged = []
    for begin, end in sorted(read):  # those that are read may share it with each other
        if merged and begin < merged[-1][1]:
            merged[-1] = (merged[-1][0], max(end, merged[-1][1]))
        else:
            merged.append((begin, end))
    spans = sorted(written + merged)
    return any(a[1] > b[0] for a, b in zip(spans, spans[1:]))


def muon_update(x: Tensors, g: Tensors, m: Tensors, lr: float, beta: float = 0.95, nesterov: bool = True,
                decay: float = 0.0, steps: int = 5, coefficients: Sequence[float] = COEFFICIENTS,
                epsilon: float = 1e-7) -> None:
    """One Muon update of matrices of one shape [rows, cols], each float32 and contiguous; a tensor or a
    sequence of them each.  In place:
        m = beta m + g;  u = g + beta m (nesterov), or m
        x = (1 - lr decay) x - lr sqrt(max(1, rows / cols)) orthogonalize(u)
    x and m may not share memory with each other or with g.  It has no gradient: where one is recorded, g
    and m that require one are refused, and x that is not a leaf."""
    x, g, m = _list(x), _list(g), _list(m)
    if not len(x) == len(g) == len(m):
        raise ValueError("x, g and m must be equally many")
    if not x:
        return
    shape, dev = x[0].shape, x[0].device
    if len(shape) != 2:
        raise ValueError(f"x must be [rows, cols] (got {tuple(shape)})")
    if _wants_grad(*g, *m) or _wants_grad(*(t for t in x if not t.is_leaf)) or _has_tangent(*x, *g, *m):
        raise ValueError("muon_update has no gradient: call it under torch.no_grad(), or on detached tensors")
    for name, ts in (("x", x), ("g", g), ("m", m)):
        for t in ts:
            if t.dtype != F32 or not t.is_contiguous() or not t.is_cuda:
                raise ValueError(f"{name} must be contiguous float32 GPU tensors")
            if t.shape != shape or t.device != dev:
                raise ValueError(f"{name} must have shape {tuple(shape)} on {dev} (got {tuple(t.shape)} on "
                                 f"{t.device})")
    size = 4 * shape[0] * shape[1]
    written, read = ([(t.data_ptr(), t.data_ptr() + size) for t in ts] for ts in (x + m, g))
    if _overlap(written, read):
        raise ValueError("x and m may not share memory with each other or with g")
    full = (len(x),) + tuple(shape)
    n = _bytes(full)
    table = struct.pack(f"{3 * len(x)}P", *(t.data_ptr() for row in zip(x, g, m) for t in row))
    ws = torch.empty((n,), dtype=torch.uint8, device=dev)
    _call("gdn2_muon_update", dev, _SHAPE(*full), table, lr, beta, 1 if nesterov else 0, decay, steps,
          _coefficients(coefficients), epsilon, ws.data_ptr(), n)
    increment_version(x + m)


class Muon(torch.optim.Optimizer):
    """Muon: momentum, whose update is orthogonalised, and decay.  For parameters that are matrices
    (contiguous float32 [rows, cols]); embeddings, heads, norms and gates go to FusedAdamW.  All
    parameters of a shape that have a gradient are updated by one call."""

    def __init__(self, params, lr: float = 0.02, momentum: float = 0.95, nesterov: bool = True,
                 weight_decay: float = 0.0, steps: int = 5, coefficients: Sequence[float] = COEFFICIENTS,
                 epsilon: float = 1e-7):
        super().__init__(params, dict(lr=lr, momentum=momentum, nesterov=nesterov,
                                      weight_decay=weight_decay, steps=steps,
                                      coefficients=tuple(coefficients), epsilon=epsilon))
        for group in self.param_groups:
            for p in group["params"]:
                if p.dim() != 2 or p.dtype != F32:
                    raise ValueError(f"Muon takes float32 matrices (got {p.dtype} {tuple(p.shape)})")

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        for group in self.param_groups:
            shapes: dict = {}
            for p in group["params"]:
                if p.grad is None:
                    continue
                st = self.state[p]
                if not st:
                    st["momentum"] = torch.zeros_like(p)
                shapes.setdefault((p.shape, p.device), []).append(p)
            for ps in shapes.values():
                muon_update(ps, [p.grad.contiguous() for p in ps], [self.state[p]["momentum"] for p in ps],
                            group["lr"], group["momentum"], group["nesterov"], group["weight_decay"],
                            group["steps"], group["coefficients"], group["epsilon"])
        return loss
