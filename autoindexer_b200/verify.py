"""Verification of drafted tokens against the target model's probabilities.

A drafter proposes a few tokens per sequence, the target model scores them in
one forward, and ``verify_draft`` keeps the longest prefix that leaves the
target's distribution unchanged, plus one token sampled where it stopped.
Random numbers are inputs, so a step can be repeated exactly.
"""

from __future__ import annotations

from typing import Optional, Tuple

import torch
from torch import Tensor

from . import _call, _lib

__all__ = ["verify_draft"]

MAX_DRAFT = 64
MAX_ROWS = 65535  # (sequences times 2 L + 1)


_PLANS = _call.Plans()


def _plan(target, draft_tokens, uniforms, noise, draft_logits, draft_lens, temperature):
    """Checks the arguments; returns the tensors the kernels read and the
    argument struct without pointers."""
    index = _call.cuda_index("target_logits", target)
    if target.dim() != 3 or target.numel() == 0:
        raise ValueError(f"target_logits must be (B, L + 1, V) and not empty, got {tuple(target.shape)}")
    B, rows, V = target.shape
    L = rows - 1
    if L > MAX_DRAFT:
        raise ValueError(f"at most {MAX_DRAFT} drafted tokens, got {L}")
    if B * (2 * L + 1) > MAX_ROWS:
        raise ValueError(f"B (2 L + 1) may be {MAX_ROWS} at most, got {B} sequences of {L} drafted tokens: split the batch")
    if draft_tokens.dtype is not torch.int64:
        raise TypeError(f"draft_tokens must be int64, got {draft_tokens.dtype}")
    if draft_tokens.shape != (B, L):
        raise ValueError(f"draft_tokens must have shape {(B, L)}, got {tuple(draft_tokens.shape)}")
    _call.on_device("draft_tokens", draft_tokens, index)
    draft_tokens = draft_tokens.contiguous()
    uniforms = _call.floats("uniforms", uniforms, (B, L), index)
    noise = _call.floats("noise", noise, (B, V), index)
    a = _lib.AiVerifyArgs()
    a.batch, a.n_draft, a.vocab = B, L, V
    a.dtype = _call.dtype_code(target, "target_logits")
    dtype = target.dtype
    target = _call.dense_d(target)
    a.target_stride_b, a.target_stride_t = target.stride(0), target.stride(1)
    if draft_logits is not None:
        if draft_logits.shape != (B, L, V):
            raise ValueError(f"draft_logits must have shape {(B, L, V)}, got {tuple(draft_logits.shape)}")
        if draft_logits.dtype is not dtype:
            raise TypeError(f"draft_logits is {draft_logits.dtype}, target_logits {dtype}")
        _call.on_device("draft_logits", draft_logits, index)
        draft_logits = _call.dense_d(draft_logits)
        a.draft_stride_b, a.draft_stride_t = draft_logits.stride(0), draft_logits.stride(1)
    if draft_lens is not None:
        draft_lens = _call.ints("draft_lens", draft_lens, (B,), index)
    if temperature is not None:
        temperature = _call.floats("temperature", temperature, (B,), index)
    a.status = _call.status_ptr(index)
    return (target, draft_tokens, uniforms, noise, draft_logits, draft_lens, temperature), a


def verify_draft(target_logits: Tensor, draft_tokens: Tensor, uniforms: Tensor, noise: Tensor,
                 draft_logits: Optional[Tensor] = None, draft_lens: Optional[Tensor] = None,
                 temperature: Optional[Tensor] = None) -> Tuple[Tensor, Tensor, Tensor]:
    """Accepts drafted tokens and samples the next one, per sequence.

    ``target_logits`` ``(B, L + 1, V)``: row ``i`` scores the token after the
    first ``i`` drafted ones; ``draft_tokens`` ``(B, L)`` int64;
    ``draft_logits`` ``(B, L, V)`` the logits they were sampled from (``None``:
    proposed with certainty, as by a lookup); ``draft_lens`` ``(B,)`` int32 how
    many are real; ``temperature`` ``(B,)`` float32 divides both (``None``: 1;
    0 decodes greedily; any positive value, however small, is a temperature).  ``uniforms`` ``(B, L)`` float32 in ``[0, 1)`` decide
    acceptance: ``u * q(x) < p(x)``; ``noise`` ``(B, V)`` float32 exponential
    variates (> 0) choose the next token: the largest ``r / noise`` with ``r``
    the residual ``max(p - q, 0)`` after a refusal, else ``p``; equal values
    go to the lowest index.

    Returns ``(accepted (B,) int32, tokens (B, L + 1) int64, logprobs (B, L +
    1) float32)``: the accepted tokens and the next one, then -1, and each
    one's log-probability under the target (0 past them, and in greedy rows).

    Logits are CUDA bfloat16, float16 or float32, finite or ``-inf``, with a
    contiguous vocabulary; up to 64 drafted tokens, ``B (2 L + 1)`` up to 65535.  A token outside the
    vocabulary is refused and sets the status word (so does a ``draft_lens``
    below 0 or above ``L``, taken as 0 or ``L``).  There is no gradient: a
    backward through the log-probabilities raises."""
    tensors = (target_logits, draft_tokens, uniforms, noise, draft_logits, draft_lens, temperature)
    at = tuple(map(_call.sig, tensors))
    plan = _PLANS.get(at)
    if plan is None:
        given = tensors
        tensors, plan = _plan(*given)
        _PLANS.keep(at, given, tensors, plan)
    if _call.tracked(target_logits, draft_logits, temperature):
        return _call.no_backward("verify_draft", lambda: _run(plan, tensors), target_logits, draft_logits, temperature)
    return _run(plan, tensors)


def _run(plan, tensors):
    target, draft_tokens, uniforms, noise, draft_logits, draft_lens, temperature = tensors
    B, rows, _ = target.shape
    device = target.device
    a = _call.copy(plan)
    accepted = torch.empty(B, dtype=torch.int32, device=device)
    tokens = torch.empty((B, rows), dtype=torch.int64, device=device)
    logprobs = torch.empty((B, rows), dtype=torch.float32, device=device)
    a.target, a.noise = target.data_ptr(), noise.data_ptr()
    if rows > 1:
        a.tokens, a.uniforms = draft_tokens.data_ptr(), uniforms.data_ptr()
        if draft_logits is not None:
            a.draft = draft_logits.data_ptr()
    if draft_lens is not None:
        a.draft_lens = draft_lens.data_ptr()
    if temperature is not None:
        a.temperature = temperature.data_ptr()
    a.accepted, a.out_tokens, a.logprobs = accepted.data_ptr(), tokens.data_ptr(), logprobs.data_ptr()
    lib = _lib.lib()
    ws = _call.workspace(lib.ai_verify_draft_workspace, a, device, "ai_verify_draft_workspace")
    _call.launch(lib.ai_verify_draft, a, target.get_device(), "ai_verify_draft")
    del ws
    return accepted, tokens, logprobs
