"""Distillation from a teacher's likeliest tokens.

A teacher's distribution over a large vocabulary is kept as its likeliest words
and their log-probabilities (``token_logprobs(..., top_k=k)``); the student is
trained towards it row by row.  ``distill_loss`` is differentiable;
``distill_loss_and_grad`` gives the losses and the gradient of their weighted
sum in one pass that reads the logits once.
"""

from __future__ import annotations

from typing import Optional, Tuple

import torch
from torch import Tensor
from torch.autograd.function import once_differentiable

from . import _call, _lib
from .scoring import check_rows, check_temperature, empty_rows, no_gradient, point_rows

__all__ = ["distill_loss", "distill_loss_and_grad"]

_PLANS = _call.Plans()


def _starts(x: Tensor):
    """Where the rows of ``x`` start, in bytes, in order."""
    at = torch.zeros((), dtype=torch.int64)
    for n, st in zip(x.shape[:-1], x.stride()[:-1]):
        at = at[..., None] + torch.arange(n) * st
    return at.flatten().mul_(x.element_size()).add_(x.data_ptr()).sort()[0]


def _span(x: Tensor) -> int:
    return (sum((n - 1) * st for n, st in zip(x.shape, x.stride())) + 1) * x.element_size()


def check_out(out: Tensor, logits: Tensor) -> None:
    """Raises where rows of ``out`` overlap one another, or rows of ``logits`` other
    than as the same memory in the same places."""
    row = out.shape[-1] * out.element_size()
    inner, least = out.shape[-1], True
    for st, n in sorted((st, n) for n, st in zip(out.shape[:-1], out.stride()) if n > 1):
        least &= st >= inner  # (each dimension steps past all that lies within it: rows one after the other)
        inner = st * (n - 1) + inner
    if not least:
        at = _starts(out)
        if at.numel() > 1 and int(at.diff().min()) < row:
            raise ValueError("the rows of out must not share memory")
    a, b = out.data_ptr(), logits.data_ptr()
    if a + _span(out) <= b or b + _span(logits) <= a:
        return
    if a == b and all(n == 1 or x == y for n, x, y in zip(out.shape, out.stride(), logits.stride())):
        return
    mine, other = _starts(out), _starts(logits)
    after = torch.searchsorted(mine, other)  # (mine[after - 1] < other <= mine[after])
    before = other - mine[(after - 1).clamp_min(0)]
    behind = mine[after.clamp_max(len(mine) - 1)] - other
    if bool((((after > 0) & (before < row)) | ((after < len(mine)) & (behind < row))).any()):
        raise ValueError("out overlaps student_logits: it may be the same rows or apart from them")


def _plan(logits, ids, logprobs, weights, temperature, tail):
    """Checks the arguments; returns the tensors the kernel reads and the
    argument struct without pointers."""
    a = _lib.AiDistillArgs()
    logits, rows, index = check_rows(a, "student_logits", logits)
    if logits.shape[-1] * logits.element_size() > _lib.MAX_ROW_BYTES:
        raise ValueError(f"a row of student_logits may have {_lib.MAX_ROW_BYTES} bytes at most, got {tuple(logits.shape)} of {logits.dtype}")
    if tail not in _lib.TAILS:
        raise ValueError(f"tail must be one of {', '.join(map(repr, _lib.TAILS))}, got {tail!r}")
    a.tail = _lib.TAILS[tail]
    if ids.dtype is not torch.int64:
        raise TypeError(f"teacher_tokens must be int64, got {ids.dtype}")
    k = ids.shape[-1] if ids.dim() else 0
    if ids.shape[:-1] != rows or not 1 <= k <= _lib.MAX_TOP:
        raise ValueError(f"teacher_tokens must have shape {tuple(rows)} + (1 to {_lib.MAX_TOP},), got {tuple(ids.shape)}")
    _call.on_device("teacher_tokens", ids, index)
    a.n_top = k
    logprobs = _call.floats("teacher_logprobs", logprobs, ids.shape, index)
    if weights is not None:
        weights = _call.floats("weights", weights, rows, index)
    temperature = check_temperature(temperature, rows[0], index)
    a.status = _call.status_ptr(index)
    return (logits, ids.contiguous(), logprobs, weights, temperature), a


def _planned(logits, ids, logprobs, weights, temperature, tail):
    tensors = (logits, ids, logprobs, weights, temperature)
    at = (*_call.sigs(tensors), tail)
    plan = _PLANS.get(at)
    if plan is None:
        given = tensors
        tensors, plan = _plan(*given, tail)
        _PLANS.keep(at, given, tensors, plan)
    return tensors, plan


def _run(a, tensors, losses: Optional[Tensor], grad: Optional[Tensor]) -> None:
    logits, ids, logprobs, weights, temperature = tensors
    point_rows(a, logits)
    a.top_tokens, a.top_logprobs = ids.data_ptr(), logprobs.data_ptr()
    if weights is not None:
        a.weights = weights.data_ptr()
    if temperature is not None:
        a.temperature = temperature.data_ptr()
    if losses is not None:
        a.losses = losses.data_ptr()
    if grad is not None:
        sd = grad.stride()
        a.dlogits, a.dstride_b, a.dstride_t = grad.data_ptr(), sd[0], sd[1] if len(sd) == 3 else 0
    _call.launch(_lib.lib().ai_distill, a, logits.get_device(), "ai_distill")


def _losses(logits: Tensor) -> Tensor:
    return logits.new_empty(logits.shape[:-1], dtype=torch.float32)


class DistillFn(torch.autograd.Function):
    """Autograd wrapper: saves the inputs and eight numbers a row; backward is
    ``ai_distill_bwd``."""

    @staticmethod
    def forward(ctx, logits, ids, logprobs, temperature, plan):
        a, losses = _call.copy(plan), _losses(logits)
        stats = losses.new_empty((losses.numel(), 8))
        a.row_stats = stats.data_ptr()
        _run(a, (logits, ids, logprobs, None, temperature), losses, None)
        ctx.save_for_backward(logits, ids, logprobs, temperature, stats)
        ctx.plan = plan
        return losses

    @staticmethod
    @once_differentiable
    def backward(ctx, g):
        # (hooks on saved tensors may have brought back copies of other strides)
        logits, ids, logprobs, temperature, stats = ctx.saved_tensors
        logits, ids, logprobs, stats, g = _call.dense_d(logits), ids.contiguous(), logprobs.contiguous(), stats.contiguous(), g.contiguous()
        a = _lib.AiDistillBwdArgs()
        a.fwd = ctx.plan
        point_rows(a.fwd, logits)
        a.fwd.top_tokens, a.fwd.top_logprobs, a.fwd.row_stats = ids.data_ptr(), logprobs.data_ptr(), stats.data_ptr()
        if temperature is not None:
            temperature = temperature.contiguous()
            a.fwd.temperature = temperature.data_ptr()
        grad = empty_rows(logits)
        sd = grad.stride()
        a.g_losses, a.dlogits, a.dstride_b, a.dstride_t = g.data_ptr(), grad.data_ptr(), sd[0], sd[1] if len(sd) == 3 else 0
        _call.launch(_lib.lib().ai_distill_bwd, a, logits.get_device(), "ai_distill_bwd")
        return grad, None, None, None, None


def distill_loss(student_logits: Tensor, teacher_tokens: Tensor, teacher_logprobs: Tensor,
                 temperature: Optional[Tensor] = None, tail: str = "bucket") -> Tensor:
    """Kullback-Leibler divergence of each row of ``softmax(student_logits /
    temperature)`` from the teacher's, of which the likeliest words are known.

    ``student_logits`` ``(B, T, V)`` or ``(N, V)``; ``teacher_tokens`` int64
    ``(..., K)`` (K up to 128) and ``teacher_logprobs`` float32 as
    ``token_logprobs`` gives them (taken at the same temperature); entries with
    a negative token or ``-inf`` are left out, so lists may be shorter than K.
    ``tail="bucket"``: the teacher's remaining probability is compared with the
    student's on all other words together (a remainder of 2^-23 + 2^-24 sum p_k |ln p_k| or less, which the rounding of
    ``teacher_logprobs`` may leave, counts as none); ``"renormalize"``: the teacher's
    words are all there is (any logits will do for ``teacher_logprobs``).
    ``temperature`` as in ``token_logprobs``.

    Returns the float32 losses of the rows' shape (0 for a row without an
    entry, which is not read; ``inf`` where a listed word is masked).  A token
    outside the vocabulary, or one that an earlier entry of its row has, is left
    out and sets the status word.  Types, strides and masked logits as in
    ``token_logprobs``; rows of up to 3,145,728 bytes.  Differentiable in the student's logits (reverse mode,
    once; rounded once to their type)."""
    tensors, plan = _planned(student_logits, teacher_tokens, teacher_logprobs, None, temperature, tail)
    logits, ids, logprobs, _, temperature = tensors
    if _call.tracked(logits, teacher_logprobs, temperature):
        no_gradient("distill_loss", teacher_logprobs=teacher_logprobs, temperature=temperature)
        return DistillFn.apply(logits, ids, logprobs, temperature, plan)
    losses = _losses(logits)
    _run(_call.copy(plan), tensors, losses, None)
    return losses


def distill_loss_and_grad(student_logits: Tensor, teacher_tokens: Tensor, teacher_logprobs: Tensor,
                          weights: Optional[Tensor] = None, temperature: Optional[Tensor] = None, tail: str = "bucket",
                          out: Optional[Tensor] = None) -> Tuple[Tensor, Tensor]:
    """``distill_loss`` and the gradient of ``(weights * losses).sum()`` with
    respect to the logits, in one pass over them.

    ``weights`` float32 of the rows' shape (``None``: 1; a mean's factor and a
    loss scale belong here): a row of weight 0 is not read, its loss and
    gradient are 0.  Returns ``(losses, gradient)``, the losses without the
    weights; the gradient, of the logits' shape and type, goes on by
    ``student_logits.backward(gradient)``.  ``out`` receives it (same shape and
    type; ``student_logits`` itself is allowed, which needs no memory for it; rows
    that overlap one another, or those of ``student_logits`` in part, are refused).
    A backward through the losses raises."""
    tensors, plan = _planned(student_logits, teacher_tokens, teacher_logprobs, weights, temperature, tail)
    logits = tensors[0]
    if out is None:
        grad = empty_rows(logits)
    else:
        grad = out.detach()
        if grad.shape != logits.shape or grad.dtype is not logits.dtype:
            raise ValueError(f"out must be {logits.dtype} of shape {tuple(logits.shape)}, got {out.dtype} {tuple(out.shape)}")
        if grad.stride(-1) != 1:
            raise ValueError("out must have a contiguous last dimension")
        _call.on_device("out", grad, logits.get_device())
        check_out(grad, logits)
    losses = _losses(logits)

    def run():
        _run(_call.copy(plan), tensors, losses, grad)
        if out is not None:
            torch.autograd.graph.increment_version(out)
        return losses

    if _call.tracked(student_logits, teacher_logprobs, weights, temperature):
        return _call.no_backward("distill_loss_and_grad", run, student_logits, teacher_logprobs, weights, temperature), grad
    return run(), grad
