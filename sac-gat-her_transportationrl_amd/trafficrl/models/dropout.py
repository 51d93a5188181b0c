"""Dropout from a counter-based generator with the residual add behind it
(csrc/dropout_add.hip): the mask is drawn again in the backward pass, never
stored."""
from __future__ import annotations

import math
from typing import Optional

import torch

from .. import _lib
from ..autograd import no_tangents, once


def _aligned(t: torch.Tensor) -> torch.Tensor:
    t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


def _launch(x, residual, rng, rest, save: bool):
    border, site, code = rest
    y = torch.empty_like(x)
    used = torch.empty_like(rng) if save else None
    _lib.check(_lib.load().trx_dropout_add_forward(x.numel(), code, x.data_ptr(),
                                                   None if residual is None else residual.data_ptr(), rng.data_ptr(),
                                                   border, site, y.data_ptr(), None if used is None else used.data_ptr(),
                                                   _lib.raw_stream(x.device)), "trx_dropout_add_forward")
    return y, used


def _launch_backward(grad_y, used, rest):
    border, site, code = rest
    g = _aligned(grad_y)
    grad_x = torch.empty_like(g)
    _lib.check(_lib.load().trx_dropout_add_backward(g.numel(), code, g.data_ptr(), used.data_ptr(), border, site,
                                                    grad_x.data_ptr(), _lib.raw_stream(g.device)),
               "trx_dropout_add_backward")
    return grad_x


class _DropoutAdd(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, rng, rest):
        y, used = _lib.on_device(x.device, _launch, x, residual, rng, rest, True)
        ctx.save_for_backward(used)
        ctx.rest = rest
        return y

    @staticmethod
    @once("dropout_add")
    def backward(ctx, grad_y):
        wants_x, wants_residual = ctx.needs_input_grad[:2]
        grad_x = None
        if wants_x:
            grad_x = _lib.on_device(grad_y.device, _launch_backward, grad_y, ctx.saved_tensors[0], ctx.rest)
        return grad_x, grad_y if wants_residual else None, None, None


def dropout_add(x: torch.Tensor, rng: torch.Tensor, p: float, *, residual: Optional[torch.Tensor] = None,
                site: int = 0) -> torch.Tensor:
    """residual + keep * x / (1 - p), each element of x kept with probability
    1 - p (p in steps of 2^-16, the factor exactly the kept share's inverse).

    x: float32, bfloat16 or float16 of any shape; residual: of the same shape and
    type, or None.  rng: int64 [2] on the device, (seed, step): the same pair and
    site give the same mask.  A program raises rng[1] by one a step (inside a
    captured graph too, so that every replay draws anew) and gives each place
    that drops out a `site` of its own (0 .. 2^32 - 1).  step counts modulo 2^32.
    Element e (row-major) is kept where its 16 bits of Philox4x32-10 reach
    round(65536 p); a dropped element adds nothing, whatever it holds.

    Differentiable once in x and residual (a forward-mode tangent is refused);
    the pair in use is kept with the graph, so rng may move on before the backward pass.  Computed in float32,
    rounded once.  Asynchronous on the current stream and capturable; before a
    backward pass is captured, drop the eager graphs of the same leaves."""
    what = "dropout_add"
    code = _lib.float_code(x, f"{what}: x")
    border = int(math.floor(float(p) * 65536.0 + 0.5)) if math.isfinite(p) else -1
    if p < 0.0 or not 0 <= border <= 65535:
        raise ValueError(f"{what}: p must be at least 0 and below 1 (at most {65535.5 / 65536.0}), got {p}")
    if rng.dtype != torch.int64 or rng.shape != (2,):
        raise ValueError(f"{what}: rng must be int64 [2]: (seed, step)")
    if residual is not None and (residual.shape != x.shape or residual.dtype != x.dtype):
        raise ValueError(f"{what}: residual {tuple(residual.shape)} {residual.dtype} for x {tuple(x.shape)} {x.dtype}")
    if not 0 <= int(site) < 2 ** 32:
        raise ValueError(f"{what}: site must be 0 .. 2^32 - 1, got {site}")
    no_tangents(what, x, residual)
    _lib.same_device(what, x, rng, residual)
    x, rng, rest = _aligned(x), rng.contiguous(), (border, int(site), code)
    if residual is not None:
        residual = _aligned(residual)
    if torch.is_grad_enabled() and (x.requires_grad or (residual is not None and residual.requires_grad)):
        return _DropoutAdd.apply(x, residual, rng, rest)
    return _lib.on_device(x.device, _launch, x, residual, rng, rest, False)[0]
