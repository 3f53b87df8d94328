"""Log-probabilities of given tokens, with the entropy and the likeliest words.

What policy training needs of a rollout (the policy's log-probability of every
sampled token and its entropy, both differentiable), what a request for
log-probabilities returns, and what a teacher hands to ``distill_loss``: one
pass over the logits forward, one backward, no softmax of the vocabulary's size
in memory.
"""

from __future__ import annotations

from typing import NamedTuple, Optional, Tuple

import torch
from torch import Tensor
from torch.autograd.function import once_differentiable

from . import _call, _lib

__all__ = ["TokenScores", "token_logprobs"]

MAX_ROWS = 0x7FFFFFFF // 16  # (rows times the most CTAs that share one)


class TokenScores(NamedTuple):
    """Results of ``token_logprobs``; ``None`` for what was not asked for."""

    logprobs: Tensor
    entropy: Optional[Tensor]
    top_logprobs: Optional[Tensor]
    top_tokens: Optional[Tensor]


def check_rows(a, name: str, logits: Tensor) -> Tuple[Tensor, Tuple[int, ...], int]:
    """Sets what ``a`` says of ``logits`` ``(B, T, V)`` or ``(N, V)``; returns
    them dense, the rows' shape and the device index."""
    index = _call.cuda_index(name, logits)
    if logits.dim() not in (2, 3) or logits.numel() == 0:
        raise ValueError(f"{name} must be (B, T, V) or (N, V) and not empty, got {tuple(logits.shape)}")
    a.dtype = _call.dtype_code(logits, name)
    rows = logits.shape[:-1]
    a.batch, a.seq_len, a.vocab = rows[0], rows[1] if len(rows) == 2 else 1, logits.shape[-1]
    if rows.numel() > MAX_ROWS:
        raise ValueError(f"at most {MAX_ROWS} rows, got {rows.numel()}")
    logits = _call.dense_d(logits)
    point_rows(a, logits)
    a.logits = None  # (a plan keeps no address)
    return logits, rows, index


def point_rows(a, logits: Tensor) -> None:
    """The strides (and the address) of dense ``logits``."""
    st = logits.stride()
    a.logits, a.stride_b, a.stride_t = logits.data_ptr(), st[0], st[1] if len(st) == 3 else 0


def check_temperature(temperature: Optional[Tensor], batch: int, index: int) -> Optional[Tensor]:
    return None if temperature is None else _call.floats("temperature", temperature, (batch,), index)


def no_gradient(what: str, **tensors: Optional[Tensor]) -> None:
    """Raises where a gradient is wanted that the operator does not give."""
    if torch.is_grad_enabled():
        for name, x in tensors.items():
            if x is not None and x.requires_grad:
                raise RuntimeError(f"{what} has no gradient for {name}: detach it")


def empty_rows(logits: Tensor) -> Tensor:
    """A tensor for the gradient of ``logits``: rows of a padded vocabulary keep
    their distance, so that both lie alike on 16-byte boundaries."""
    *rows, V = logits.shape
    pitch = logits.stride(-2)
    if not V < pitch <= V + 1024:
        return logits.new_empty(logits.shape)
    return logits.new_empty((*rows, pitch))[..., :V]


_PLANS = _call.Plans()


def _plan(logits, tokens, temperature, top_k):
    """Checks the arguments; returns the tensors the kernels read and the
    argument struct without pointers."""
    a = _lib.AiScoreArgs()
    logits, rows, index = check_rows(a, "logits", logits)
    if tokens.dtype is not torch.int64:
        raise TypeError(f"tokens must be int64, got {tokens.dtype}")
    if tokens.shape != rows:
        raise ValueError(f"tokens must have shape {tuple(rows)}, got {tuple(tokens.shape)}")
    _call.on_device("tokens", tokens, index)
    tokens = tokens.contiguous()
    temperature = check_temperature(temperature, rows[0], index)
    if not 0 <= top_k <= _lib.MAX_TOP:
        raise ValueError(f"top_k must be 0 to {_lib.MAX_TOP}, got {top_k}")
    a.top_k = top_k
    a.status = _call.status_ptr(index)
    return (logits, tokens, temperature), a


def _run(plan, tensors, entropy: bool, stats: bool):
    logits, tokens, temperature = tensors
    a = _call.copy(plan)
    a.logits, a.tokens = logits.data_ptr(), tokens.data_ptr()
    if temperature is not None:
        a.temperature = temperature.data_ptr()
    rows, k = tokens.shape, a.top_k
    logprobs = logits.new_empty(rows, dtype=torch.float32)  # (cheaper than torch.empty)
    a.logprobs = logprobs.data_ptr()
    h = top = ids = st = None
    if entropy:
        h = logprobs.new_empty(rows)
        a.entropy = h.data_ptr()
    if k:
        top, ids = logprobs.new_empty((*rows, k)), tokens.new_empty((*rows, k))
        a.top_logprobs, a.top_tokens = top.data_ptr(), ids.data_ptr()
    if stats:
        st = logprobs.new_empty((rows.numel(), 4))
        a.row_stats = st.data_ptr()
    _call.launch(_lib.lib().ai_token_logprobs, a, logits.get_device(), "ai_token_logprobs")
    return logprobs, h, top, ids, st


class TokenLogprobsFn(torch.autograd.Function):
    """Autograd wrapper: saves the logits, the tokens and four numbers a row;
    backward is ``ai_token_logprobs_bwd``."""

    @staticmethod
    def forward(ctx, logits, tokens, temperature, plan, entropy):
        logprobs, h, top, ids, st = _run(plan, (logits, tokens, temperature), entropy, True)
        ctx.save_for_backward(logits, tokens, temperature, ids, st)
        ctx.plan = plan
        ctx.set_materialize_grads(False)
        if ids is not None:
            ctx.mark_non_differentiable(ids)
        return logprobs, h, top, ids

    @staticmethod
    @once_differentiable
    def backward(ctx, g_logprobs, g_entropy, g_top, _):
        if g_logprobs is None and g_entropy is None and g_top is None:
            return None, None, None, None, None
        logits, tokens, temperature, ids, st = ctx.saved_tensors
        g = _lib.AiScoreBwdArgs()
        g.fwd = ctx.plan
        # (hooks on saved tensors may have brought back copies of other strides)
        logits, tokens, st = _call.dense_d(logits), tokens.contiguous(), st.contiguous()
        point_rows(g.fwd, logits)
        g.fwd.tokens, g.fwd.row_stats = tokens.data_ptr(), st.data_ptr()
        if temperature is not None:
            temperature = temperature.contiguous()
            g.fwd.temperature = temperature.data_ptr()
        if g_logprobs is not None:
            g_logprobs = g_logprobs.contiguous()
            g.g_logprobs = g_logprobs.data_ptr()
        if g_entropy is not None:
            g_entropy = g_entropy.contiguous()
            g.g_entropy = g_entropy.data_ptr()
        if g_top is not None:
            g_top, ids = g_top.contiguous(), ids.contiguous()
            g.g_top, g.fwd.top_tokens = g_top.data_ptr(), ids.data_ptr()
        d = empty_rows(logits)
        sd = d.stride()
        g.dlogits, g.dstride_b, g.dstride_t = d.data_ptr(), sd[0], sd[1] if len(sd) == 3 else 0
        _call.launch(_lib.lib().ai_token_logprobs_bwd, g, logits.get_device(), "ai_token_logprobs_bwd")
        return d, None, None, None, None


def token_logprobs(logits: Tensor, tokens: Tensor, temperature: Optional[Tensor] = None, top_k: int = 0,
                   entropy: bool = False) -> TokenScores:
    """Log-probability of ``tokens`` under ``softmax(logits / temperature)``.

    ``logits`` ``(B, T, V)`` or ``(N, V)``; ``tokens`` int64 of the rows' shape,
    a negative one (padding: -100) leaves its row out; ``temperature`` float32
    of the first dimension's length (``None``: 1; a value that is not above 0
    counts as 1 and sets the status word that ``read_status`` reads).

    Returns ``TokenScores(logprobs, entropy, top_logprobs, top_tokens)``:
    float32 log-probabilities of the rows' shape; with ``entropy`` each row's
    entropy (natural logarithm, else ``None``); with ``top_k`` (up to 128) the
    ``(..., top_k)`` likeliest words and their log-probabilities, best first,
    equal logits by the lowest index (else ``None``).  A row that is left out
    has 0, 0 and an empty list; lists are filled up with -1 and ``-inf``.

    Logits are CUDA bfloat16, float16 or float32 with a contiguous vocabulary
    (any row strides), finite or ``-inf`` (masked); a row of masked words alone
    has ``-inf``, entropy 0 and an empty list, one with a NaN gives NaN.  A token
    outside the vocabulary leaves its row out and sets the status word.
    Arithmetic is float32.  Differentiable in the logits through all three
    floating-point results (reverse mode, once; the gradient is rounded once to
    the logits' type), by one more read of them."""
    top_k = int(top_k)
    tensors = (logits, tokens, temperature)
    at = (*_call.sigs(tensors), top_k)
    plan = _PLANS.get(at)
    if plan is None:
        given = tensors
        tensors, plan = _plan(*given, top_k)
        _PLANS.keep(at, given, tensors, plan)
    if _call.tracked(logits, temperature):
        no_gradient("token_logprobs", temperature=temperature)
        return TokenScores(*TokenLogprobsFn.apply(*tensors, plan, bool(entropy)))
    return TokenScores(*_run(plan, tensors, entropy, False)[:4])
