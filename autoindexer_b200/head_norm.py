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

__all__ = ["qk_norm_rope"]


def _args(q, k, wq, wk, rope, positions, eps, index):
    """The call's arguments without its outputs, and the (cos, sin,
    positions) tensors they point to."""
    a = _lib.AiHeadNormArgs()
    a.batch, a.num_q_heads, a.seq_len, a.head_dim = B, _, T, D = q.shape
    a.dtype = a.weight_dtype = _call.dtype_code(q, "query")
    a.eps = eps
    a.q = _call.t4(q)
    if k is not None:
        a.num_kv_heads = k.shape[1]
        a.k = _call.t4(k)
    if wq is not None:
        a.q_weight = wq.data_ptr()
        a.weight_dtype = _call.dtype_code(wq, "q_weight")
    if wk is not None:
        a.k_weight = wk.data_ptr()
        a.weight_dtype = _call.dtype_code(wk, "k_weight")
    table = _call.fill_rope(a, rope, positions, B, T, D, index)
    a.status = _call.status_ptr(index)
    return a, table


def _run(a, q, k, index):
    q_out = torch.empty_like(q)
    a.q_out = _call.t4(q_out)
    k_out = None
    if k is not None:
        k_out = torch.empty_like(k)
        a.k_out = _call.t4(k_out)
    _call.launch(_lib.lib().ai_head_norm_fwd, a, index, "ai_head_norm_fwd")
    return q_out, k_out


class HeadNormFn(torch.autograd.Function):
    """Autograd wrapper: saves the inputs; backward is ``ai_head_norm_bwd``
    with the forward's checked arguments."""

    @staticmethod
    def forward(ctx, q, k, wq, wk, table, args, index):
        ctx.save_for_backward(q, k, wq, wk, *table)
        ctx.args, ctx.index = args, index
        return _run(args, q, k, index)

    @staticmethod
    @once_differentiable
    def backward(ctx, dq_out, dk_out):
        q, k, wq, wk, cos, sin, positions = ctx.saved_tensors
        g = _lib.AiHeadNormBwdArgs()
        g.fwd = ctx.args
        f = g.fwd
        # (saved tensors may have been moved and brought back)
        f.q = _call.t4(q)
        dq_out = _call.dense_d(dq_out)
        dq = torch.empty_like(q)
        g.dq_out, g.dq = _call.t4(dq_out), _call.t4(dq)
        dk = dwq = dwk = None
        if k is not None:
            f.k = _call.t4(k)
            dk_out = _call.dense_d(dk_out)
            dk = torch.empty_like(k)
            g.dk_out, g.dk = _call.t4(dk_out), _call.t4(dk)
        if wq is not None:
            f.q_weight = wq.data_ptr()
            dwq = torch.empty_like(wq)
            g.dq_weight = dwq.data_ptr()
        if wk is not None:
            f.k_weight = wk.data_ptr()
            dwk = torch.empty_like(wk)
            g.dk_weight = dwk.data_ptr()
        if cos is not None:
            f.rope_cos, f.rope_sin, f.pos.ptr = cos.data_ptr(), sin.data_ptr(), positions.data_ptr()
        lib = _lib.lib()
        ws = _call.workspace(lib.ai_head_norm_bwd_workspace, g, q.device, "ai_head_norm_bwd_workspace")
        _call.launch(lib.ai_head_norm_bwd, g, ctx.index, "ai_head_norm_bwd")
        del ws
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
    index = _call.cuda_index("query", query)
    if query.dim() != 4:
        raise ValueError(f"query must be (B, Hq, T, D), got {tuple(query.shape)}")
    B, _, T, D = query.shape
    if D not in (32, 64, 128):
        raise ValueError(f"head_dim must be 32, 64 or 128, got {D}")
    if query.numel() == 0:
        raise ValueError("query must not be empty")
    if key is not None:
        if key.dim() != 4 or key.shape[0] != B or key.shape[2:] != query.shape[2:] or key.shape[1] == 0:
            raise ValueError(f"key must be ({B}, Hkv, {T}, {D}) and not empty, got {tuple(key.shape)}")
        if key.dtype is not query.dtype:
            raise TypeError(f"key is {key.dtype}, query {query.dtype}")
        _call.on_device("key", key, index)
        key = _call.dense_d(key)
    elif k_weight is not None:
        raise ValueError("k_weight without a key")
    query = _call.dense_d(query)
    wq = _call.head_weight("q_weight", q_weight, query, index)
    wk = _call.head_weight("k_weight", k_weight, query, index)
    if wq is not None and wk is not None and wq.dtype is not wk.dtype:
        raise TypeError(f"q_weight is {wq.dtype}, k_weight {wk.dtype}")
    args, table = _args(query, key, wq, wk, rope, positions, eps, index)
    if torch.is_grad_enabled() and (query.requires_grad or (key is not None and key.requires_grad) or
                                    (wq is not None and wq.requires_grad) or (wk is not None and wk.requires_grad)):
        return HeadNormFn.apply(query, key, wq, wk, table, args, index)
    return _run(args, query, key, index)
