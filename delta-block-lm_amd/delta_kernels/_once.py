"""Backward passes that can be taken once: a derivative of their gradients is refused.

A gradient depends on the saved inputs also where its upstream gradients need none, so it is marked
whenever a graph of the backward is recorded."""
from __future__ import annotations

import functools

import torch


class _Refuse(torch.autograd.Function):
    @staticmethod
    def forward(ctx, anchor, *grads):
        return tuple(g.view_as(g) for g in grads)

    @staticmethod
    def backward(ctx, *_):
        raise RuntimeError("this operator cannot be differentiated twice")


def once(backward):
    """Decorates the backward of a torch.autograd.Function."""
    @functools.wraps(backward)
    def run(ctx, *upstream):
        if not torch.is_grad_enabled():
            return backward(ctx, *upstream)
        with torch.no_grad():
            out = backward(ctx, *upstream)
        out = out if isinstance(out, tuple) else (out,)
        there = [g for g in out if g is not None]
        if not there:
            return out
        marked = iter(_Refuse.apply(torch.zeros((), requires_grad=True), *there))
        return tuple(None if g is None else next(marked) for g in out)
    return run
