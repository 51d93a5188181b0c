"""What the operators' autograd functions share."""
from __future__ import annotations

import torch
from torch.autograd import forward_ad


def no_tangents(what: str, *tensors) -> None:
    """RuntimeError where a tensor (None: skipped) carries a forward-mode tangent,
    which kernels called past autograd would drop without a word."""
    for t in tensors:
        if t is not None and forward_ad.unpack_dual(t).tangent is not None:
            raise RuntimeError(f"{what} has no forward-mode derivative")


class _NoSecond(torch.autograd.Function):
    """Its outputs are the inputs behind `anchor`; differentiating them raises."""

    @staticmethod
    def forward(ctx, anchor, what, *grads):
        ctx.what = what
        return tuple(g.view_as(g) for g in grads)

    @staticmethod
    def backward(ctx, *_):
        raise RuntimeError(f"{ctx.what} can be differentiated once, not twice")


def once(what: str):
    """Decorator of a Function's backward that has no derivative of its own: runs
    it without recording; under create_graph its results raise when they are
    differentiated, whatever they depend on, instead of passing for constants."""
    def decorate(backward):
        def run(ctx, *grads):
            if not torch.is_grad_enabled():
                return backward(ctx, *grads)
            with torch.no_grad():
                out = backward(ctx, *grads)
            some = [t for t in out if t is not None]
            if not some:
                return out
            anchor = torch.zeros((), device=some[0].device, requires_grad=True)
            kept = iter(_NoSecond.apply(anchor, what, *some))
            return tuple(None if t is None else next(kept) for t in out)
        return run
    return decorate
