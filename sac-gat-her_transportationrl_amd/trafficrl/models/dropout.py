"""Dropout from a counter-based generator with the residual add behind it
(csrc/dropout_add.hip): the mask is drawn again in the backward pass, never
stored."""
from __future__ import annotations

import math
from typing import Optional

import torch
from torch.autograd.function import once_differentiable

from .. import _lib


def _aligned(t: torch.Tensor) -> torch.Tensor:
    t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


def _forward(x, residual, rng, border, site, code):
    y = torch.empty(x.shape, device=x.device, dtype=x.dtype)
    used = torch.empty(2, device=x.device, dtype=torch.int64)
    _lib.check(_lib.load().trx_dropout_add_forward(x.numel(), code, _lib.ptr(x), _lib.ptr(residual), _lib.ptr(rng),
                                                   border, site, _lib.ptr(y), _lib.ptr(used),
                                                   _lib.stream_ptr(x.device)), "trx_dropout_add_forward")
    return y, used


class _DropoutAdd(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, rng, border, site, code):
        with torch.cuda.device(x.device):
            y, used = _forward(x, residual, rng, border, site, code)
        ctx.save_for_backward(used)
        ctx.rest = border, site, code
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_y):
        used, = ctx.saved_tensors
        border, site, code = ctx.rest
        grad_x = None
        if ctx.needs_input_grad[0]:
            with torch.cuda.device(grad_y.device):
                g = _aligned(grad_y)
                grad_x = torch.empty(g.shape, device=g.device, dtype=g.dtype)
                _lib.check(_lib.load().trx_dropout_add_backward(g.numel(), code, _lib.ptr(g), _lib.ptr(used), border,
                                                                site, _lib.ptr(grad_x), _lib.stream_ptr(g.device)),
                           "trx_dropout_add_backward")
        return grad_x, grad_y if ctx.needs_input_grad[1] else None, None, None, None, None


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

    Differentiable once in x and residual; the pair in use is kept with the
    graph, so rng may move on before the backward pass.  Computed in float32,
    rounded once."""
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
    with _lib.on_device(what, x, rng, residual):
        x, rng, residual = _aligned(x), rng.contiguous(), None if residual is None else _aligned(residual)
        if torch.is_grad_enabled() and (x.requires_grad or (residual is not None and residual.requires_grad)):
            return _DropoutAdd.apply(x, residual, rng, border, int(site), code)
        return _forward(x, residual, rng, border, int(site), code)[0]
