"""Per-head query / key norms with the position rotation in the same pass.

``qk_norm_rope`` is what a Qwen3 attention layer does between its projections
and its attention (``q_norm`` / ``k_norm`` on every head, then the rotation),
in one launch forward and two backward, differentiable through autograd.
Without a table it is the norms alone, which is what precedes the
chain-of-edits attention (that rotates inside its kernels); without weights
it is the rotation alone.
"""

from __future__ import annotations

from typing import Optional, Tuple

import torch
from torch import Tensor
from torch.autograd.function import once_differentiable

from . import _call, _lib
from .attention import status_word

__all__ = ["qk_norm_rope"]


def _args(q, k, wq, wk, rope, positions, eps):
    """The call's arguments without its outputs, and the tensors they point to."""
    a = _lib.AiHeadNormArgs()
    a.batch, a.num_q_heads, a.seq_len, a.head_dim = q.shape
    a.dtype = _call.dtype_code(q, "query")
    a.eps = eps
    a.q = _call.t4(q)
    if k is not None:
        a.num_kv_heads = k.shape[1]
        a.k = _call.t4(k)
    w = wq if wq is not None else wk
    a.weight_dtype = a.dtype if w is None else _call.dtype_code(w, "weight")
    if wq is not None:
        a.q_weight = wq.data_ptr()
    if wk is not None:
        a.k_weight = wk.data_ptr()
    keep = _call.fill_rope(a, rope, positions, a.batch, a.seq_len, a.head_dim, q.device)
    a.status = status_word(q.device).data_ptr()
    return a, keep


def _forward(q, k, wq, wk, rope, positions, eps):
    a, keep = _args(q, k, wq, wk, rope, positions, eps)
    q_out = torch.empty_like(q)
    a.q_out = _call.t4(q_out)
    k_out = None
    if k is not None:
        k_out = torch.empty_like(k)
        a.k_out = _call.t4(k_out)
    _call.launch(_lib.lib().ai_head_norm_fwd, a, q.device, "ai_head_norm_fwd")
    del keep
    return q_out, k_out


class HeadNormFn(torch.autograd.Function):
    """Autograd wrapper: saves the inputs; backward is ``ai_head_norm_bwd``."""

    @staticmethod
    def forward(ctx, q, k, wq, wk, rope, positions, eps):
        ctx.save_for_backward(q, k, wq, wk, positions, *(rope or (None, None)))
        ctx.eps = eps
        return _forward(q, k, wq, wk, rope, positions, eps)

    @staticmethod
    @once_differentiable
    def backward(ctx, dq_out, dk_out):
        q, k, wq, wk, positions, cos, sin = ctx.saved_tensors
        g = _lib.AiHeadNormBwdArgs()
        g.fwd, keep = _args(q, k, wq, wk, None if cos is None else (cos, sin), positions, ctx.eps)
        dq_out = _call.dense_d(dq_out)
        dq = torch.empty_like(q)
        g.dq_out, g.dq = _call.t4(dq_out), _call.t4(dq)
        dk = dwq = dwk = None
        if k is not None:
            dk_out = _call.dense_d(dk_out)
            dk = torch.empty_like(k)
            g.dk_out, g.dk = _call.t4(dk_out), _call.t4(dk)
        if wq is not None:
            dwq = torch.empty_like(wq)
            g.dq_weight = dwq.data_ptr()
        if wk is not None:
            dwk = torch.empty_like(wk)
            g.dk_weight = dwk.data_ptr()
        lib = _lib.lib()
        ws = _call.workspace(lib.ai_head_norm_bwd_workspace, g, q.device, "ai_head_norm_bwd_workspace")
        _call.launch(lib.ai_head_norm_bwd, g, q.device, "ai_head_norm_bwd")
        del keep, ws
        return dq, dk, dwq, dwk, None, None, None


def qk_norm_rope(query: Tensor, key: Optional[Tensor], q_weight: Optional[Tensor] = None,
                 k_weight: Optional[Tensor] = None, rope: Optional[Tuple[Tensor, Tensor]] = None,
                 positions: Optional[Tensor] = None, eps: float = 1e-6) -> Tuple[Tensor, Optional[Tensor]]:
    """``R(pos) (w * x / sqrt(mean(x^2) + eps))`` of every head of ``query``
    ``(B, Hq, T, D)`` and ``key`` ``(B, Hkv, T, D)`` (or ``None``); returns
    both, in the inputs' memory order.

    ``q_weight`` / ``k_weight``: ``(D,)`` of the inputs' dtype or float32,
    ``None`` leaves that tensor unnormalised.  ``rope``: the ``(cos, sin)``
    table of ``rope_table`` (float32 ``(n_pos, D/2)``); ``positions``: its rows,
    ``(T,)`` or ``(B, T)``, int64 or int32 (an id outside the table takes row 0
    and sets the status word that ``read_status`` reads); without them nothing is
    rotated.  CUDA tensors, bfloat16, float16 or float32, head_dim 32, 64 or
    128, any strides with the last dimension contiguous.  Arithmetic is
    float32, rounded once.  Differentiable in query, key and the weights."""
    device = _call.cuda_device("query", query)
    if query.dim() != 4:
        raise ValueError(f"query must be (B, Hq, T, D), got {tuple(query.shape)}")
    B, _, T, D = query.shape
    if D not in (32, 64, 128):
        raise ValueError(f"head_dim must be 32, 64 or 128, got {D}")
    if key is not None:
        if key.dim() != 4 or key.shape[0] != B or key.shape[2] != T or key.shape[3] != D:
            raise ValueError(f"key must be ({B}, Hkv, {T}, {D}), got {tuple(key.shape)}")
        if key.dtype != query.dtype:
            raise TypeError(f"key is {key.dtype}, query {query.dtype}")
        _call.on_device("key", key, device)
    elif k_weight is not None:
        raise ValueError("k_weight without a key")
    wq, wk = _call.head_weight("q_weight", q_weight, query), _call.head_weight("k_weight", k_weight, query)
    if wq is not None and wk is not None and wq.dtype != wk.dtype:
        raise TypeError(f"q_weight is {wq.dtype}, k_weight {wk.dtype}")
    if query.numel() == 0 or (key is not None and key.numel() == 0):
        raise ValueError("query and key must not be empty")
    q = _call.dense_d(query)
    k = None if key is None else _call.dense_d(key)
    if torch.is_grad_enabled() and any(x is not None and x.requires_grad for x in (q, k, wq, wk)):
        return HeadNormFn.apply(q, k, wq, wk, rope, positions, float(eps))
    return _forward(q, k, wq, wk, rope, positions, float(eps))
