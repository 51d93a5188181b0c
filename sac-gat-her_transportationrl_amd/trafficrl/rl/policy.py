"""The masked categorical policy over links as one differentiable operator
(csrc/action_log_probs.hip): log probability of given actions, entropy and the
best alternatives, next to DiscreteSAC's masked softmax (src/rl/sac.py:44-46)."""
from __future__ import annotations

from typing import NamedTuple, Optional

import torch

from .. import _lib
from ..autograd import no_tangents, once


_MASK_TYPES = (torch.float32, torch.bool, torch.uint8)


class ActionLogProbs(NamedTuple):
    log_prob: torch.Tensor                  # float32 [rows]
    entropy: torch.Tensor                   # float32 [rows]
    top_log_prob: Optional[torch.Tensor]    # float32 [rows, top_k]
    top_action: Optional[torch.Tensor]      # int64 [rows, top_k]


def _args(logits, mask, row_ptr, action, rest, outs, grads=(0, 0, 0, 0)):
    max_row, top_k, code = rest
    if row_ptr is None:
        shape = (logits.shape[0], logits.shape[1], logits.stride(0), 0, 0, 0 if mask is None else mask.stride(0))
    else:
        shape = (row_ptr.numel() - 1, 0, 0, logits.numel(), max_row, 0)
    return _lib.TrxActionLogProbsArgs(
        *shape, code, 0 if mask is None or mask.dtype == torch.float32 else 1, top_k, 0, logits.data_ptr(),
        0 if mask is None else mask.data_ptr(), 0 if row_ptr is None else row_ptr.data_ptr(), action.data_ptr(),
        *(0 if t is None else t.data_ptr() for t in outs), *grads)


def _launch(logits, mask, row_ptr, action, rest):
    L, top_k, dev = _lib.load(), rest[1], logits.device
    n = action.shape[0]
    floats = lambda *shape: torch.empty(shape, device=dev, dtype=torch.float32)  # noqa: E731
    log_prob, entropy, stats = floats(n), floats(n), floats(n, 4)
    top_log_prob = floats(n, top_k) if top_k else None
    top_action = torch.empty(n, top_k, device=dev, dtype=torch.int64) if top_k else None
    a = _args(logits, mask, row_ptr, action, rest, (log_prob, entropy, stats, top_log_prob, top_action))
    need = L.trx_action_log_probs_workspace_bytes(a)
    ws = None
    if need > 0:
        ws = torch.empty(need, device=dev, dtype=torch.uint8)
        a.workspace, a.workspace_bytes = ws.data_ptr(), need
    _lib.check(L.trx_action_log_probs_forward(a, _lib.raw_stream(dev)), "trx_action_log_probs_forward")
    return log_prob, entropy, top_log_prob, top_action, stats


def _launch_backward(logits, mask, row_ptr, action, stats, top_action, rest, grads):
    grads = [None if t is None else t.contiguous() for t in grads]   # float32, like the outputs
    grad = torch.empty(logits.shape, device=logits.device, dtype=logits.dtype)
    a = _args(logits, mask, row_ptr, action, rest, (None, None, stats, None, top_action),
              (*(0 if t is None else t.data_ptr() for t in grads), grad.data_ptr()))
    _lib.check(_lib.load().trx_action_log_probs_backward(a, _lib.raw_stream(logits.device)),
               "trx_action_log_probs_backward")
    return grad


class _ActionLogProbs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, mask, row_ptr, action, rest):
        *outs, stats = _lib.on_device(logits.device, _launch, logits, mask, row_ptr, action, rest)
        ctx.save_for_backward(logits, mask, row_ptr, action, stats, outs[3])
        ctx.rest = rest
        ctx.set_materialize_grads(False)
        if outs[3] is not None:
            ctx.mark_non_differentiable(outs[3])
        return tuple(outs)

    @staticmethod
    @once("action_log_probs")
    def backward(ctx, *grads):
        logits = ctx.saved_tensors[0]
        return _lib.on_device(logits.device, _launch_backward, *ctx.saved_tensors, ctx.rest,
                              grads[:3]), None, None, None, None


def action_log_probs(logits: torch.Tensor, action: torch.Tensor, *, mask: Optional[torch.Tensor] = None,
                     row_ptr: Optional[torch.Tensor] = None, max_row: Optional[int] = None,
                     top_k: int = 0) -> ActionLogProbs:
    """log softmax of each row of logits over the links that may be chosen, at
    `action`; the row's entropy; its top_k highest log probabilities with their
    links, highest first (ties: the lower link first).

    logits: float32, bfloat16 or float16, [rows, links], or [total] with row_ptr
    (int64 [rows + 1], each row's first link) for rows of different lengths (at
    most 2^30 links in a row).  action: int64 [rows], row-local.  mask: shaped like
    logits; a link may be chosen where it is > 0 (the env's action_mask; bool
    works too).  A logit of -inf is a link that may not be chosen; large negative
    fills are ordinary logits.  max_row: the longest row of a packed batch, a
    hint that makes many short rows faster.
    top_k: 0 (top_* are None) .. 16.

    An action that may not be chosen, or lies outside its row, has log probability
    -inf and passes no gradient; an empty row has entropy 0; where fewer than
    top_k links may be chosen the rest is -inf and -1.  A row with a logit of NaN
    or +inf that may be chosen has NaN for its values.

    Differentiable once in logits through log_prob, entropy and top_log_prob (a
    forward-mode tangent is refused).  Computed in float32 (the gradient rounded once to the logits' type).
    Asynchronous on the current stream and capturable; before a backward pass is
    captured, drop the eager graphs of the same leaves."""
    what = "action_log_probs"
    code = _lib.float_code(logits, f"{what}: logits")
    if row_ptr is None:
        if logits.dim() != 2:
            raise ValueError(f"{what}: logits must be [rows, links] (or packed with row_ptr), got {tuple(logits.shape)}")
        rows = logits.shape[0]
    else:
        if logits.dim() != 1:
            raise ValueError(f"{what}: packed logits must be [total], got {tuple(logits.shape)}")
        if row_ptr.dtype != torch.int64 or row_ptr.dim() != 1 or row_ptr.numel() < 1:
            raise ValueError(f"{what}: row_ptr must be int64 [rows + 1]")
        rows = row_ptr.numel() - 1
    if action.dtype not in (torch.int64, torch.int32) or action.shape != (rows,):
        raise ValueError(f"{what}: action must be int64 [{rows}], got {action.dtype} {tuple(action.shape)}")
    if mask is not None and mask.shape != logits.shape:
        raise ValueError(f"{what}: mask {tuple(mask.shape)} for logits {tuple(logits.shape)}")
    if not 0 <= int(top_k) <= _lib.TOP_MAX:
        raise ValueError(f"{what}: top_k must be 0..{_lib.TOP_MAX}, got {top_k}")
    max_row = logits.numel() if max_row is None else int(max_row)
    if max_row < 0:
        raise ValueError(f"{what}: max_row must be >= 0")
    max_row = min(max_row, 2 ** 30)
    no_tangents(what, logits, mask)
    _lib.same_device(what, logits, action, mask, row_ptr)
    if logits.stride(-1) != 1 and logits.numel():
        logits = logits.contiguous()
    if action.dtype != torch.int64:
        action = action.long()
    action = action.contiguous()
    if mask is not None:
        if mask.dtype not in _MASK_TYPES:
            mask = mask > 0
        if mask.stride(-1) != 1 and mask.numel():
            mask = mask.contiguous()
    if row_ptr is not None:
        row_ptr = row_ptr.contiguous()
    rest = max_row, int(top_k), code
    if torch.is_grad_enabled() and logits.requires_grad:
        return ActionLogProbs(*_ActionLogProbs.apply(logits, mask, row_ptr, action, rest))
    return ActionLogProbs(*_lib.on_device(logits.device, _launch, logits, mask, row_ptr, action, rest)[:4])
