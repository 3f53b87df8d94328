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


_PLANS = _call.Plans()


def _plan(query, key, q_weight, k_weight, cos, sin, positions, eps):
    """Checks the arguments; returns the tensors the kernels read (dense
    copies where those given are not) and the argument struct without
    pointers."""
    index = _call.cuda_index("query", query)
    if query.dim() != 4:
        raise ValueError(f"query must be (B, Hq, T, D), got {tuple(query.shape)}")
    B, Hq, T, D = query.shape
    if D not in (32, 64, 128):
        raise ValueError(f"head_dim must be 32, 64 or 128, got {D}")
    if query.numel() == 0:
        raise ValueError("query must not be empty")
    query = _call.dense_d(query)
    a = _lib.AiHeadNormArgs()
    a.batch, a.num_q_heads, a.seq_len, a.head_dim = B, Hq, T, D
    a.dtype = a.weight_dtype = _call.dtype_code(query, "query")
    a.eps = eps
    a.q, a.q_out = _call.strides4(query), _call.strides4(torch.empty_like(query, device="meta"))
    if key is not None:
        if key.dim() != 4 or key.shape[0] != B or key.shape[2:] != query.shape[2:] or key.shape[1] == 0:
            raise ValueError(f"key must be ({B}, Hkv, {T}, {D}) and not empty, got {tuple(key.shape)}")
        if key.dtype is not query.dtype:
            raise TypeError(f"key is {key.dtype}, query {query.dtype}")
        _call.on_device("key", key, index)
        key = _call.dense_d(key)
        a.num_kv_heads = key.shape[1]
        a.k, a.k_out = _call.strides4(key), _call.strides4(torch.empty_like(key, device="meta"))
    elif k_weight is not None:
        raise ValueError("k_weight without a key")
    q_weight = _call.head_weight("q_weight", q_weight, query, index)
    k_weight = _call.head_weight("k_weight", k_weight, query, index)
    if q_weight is not None and k_weight is not None and q_weight.dtype is not k_weight.dtype:
        raise TypeError(f"q_weight is {q_weight.dtype}, k_weight {k_weight.dtype}")
    w = q_weight if q_weight is not None else k_weight
    if w is not None:
        a.weight_dtype = _call.dtype_code(w, "weight")
    cos, sin, positions = _call.check_rope(a, None if cos is None else (cos, sin), positions, B, T, D, index)
    a.status = _call.status_ptr(index)
    return (query, key, q_weight, k_weight, cos, sin, positions), a


def _point(a, q, k, wq, wk, cos, sin, positions):
    a.q.ptr = q.data_ptr()
    if k is not None:
        a.k.ptr = k.data_ptr()
    if wq is not None:
        a.q_weight = wq.data_ptr()
    if wk is not None:
        a.k_weight = wk.data_ptr()
    _call.point_rope(a, cos, sin, positions)


def _run(plan, tensors):
    a = _call.copy(plan)
    _point(a, *tensors)
    q, k = tensors[0], tensors[1]
    q_out = torch.empty_like(q)
    a.q_out.ptr = q_out.data_ptr()
    k_out = None
    if k is not None:
        k_out = torch.empty_like(k)
        a.k_out.ptr = k_out.data_ptr()
    _call.launch(_lib.lib().ai_head_norm_fwd, a, q.get_device(), "ai_head_norm_fwd")
    return q_out, k_out


class HeadNormFn(torch.autograd.Function):
    """Autograd wrapper: saves the inputs; backward is ``ai_head_norm_bwd``
    with the forward's checked arguments."""

    @staticmethod
    def forward(ctx, q, k, wq, wk, cos, sin, positions, plan):
        tensors = (q, k, wq, wk, cos, sin, positions)
        ctx.save_for_backward(*tensors)
        ctx.plan = plan
        return _run(plan, tensors)

    @staticmethod
    @once_differentiable
    def backward(ctx, dq_out, dk_out):
        q, k, wq, wk, cos, sin, positions = ctx.saved_tensors
        g = _lib.AiHeadNormBwdArgs()
        g.fwd = ctx.plan
        # (hooks on saved tensors may have moved them and brought back copies of
        # other strides: all that the struct says of a layout is taken anew)
        q, g.fwd.q = _call.dense4(q)
        dq_out, g.dq_out = _call.dense4(dq_out)
        dq, g.dq = _call.dense4(torch.empty_like(q))
        dk = dwq = dwk = None
        if k is not None:
            k, g.fwd.k = _call.dense4(k)
            dk_out, g.dk_out = _call.dense4(dk_out)
            dk, g.dk = _call.dense4(torch.empty_like(k))
        if wq is not None:
            wq = wq.contiguous()
            dwq = torch.empty_like(wq)
            g.dq_weight = dwq.data_ptr()
        if wk is not None:
            wk = wk.contiguous()
            dwk = torch.empty_like(wk)
            g.dk_weight = dwk.data_ptr()
        if cos is not None:
            cos, sin, positions = cos.contiguous(), sin.contiguous(), _call.dense_positions(positions)
            g.fwd.pos.stride_b = _call.positions_stride(positions)
        _point(g.fwd, q, k, wq, wk, cos, sin, positions)
        lib = _lib.lib()
        ws = _call.workspace(lib.ai_head_norm_bwd_workspace, g, q.device, "ai_head_norm_bwd_workspace")
        _call.launch(lib.ai_head_norm_bwd, g, q.get_device(), "ai_head_norm_bwd")
        del ws
        return dq, dk, dwq, dwk, None, None, None, None


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
    float32, rounded once.  Differentiable in query, key and the weights (in
    reverse mode; inputs with forward-mode tangents raise)."""
    cos, sin = (None, None) if rope is None else rope
    tensors = (query, key, q_weight, k_weight, cos, sin, positions)
    eps = float(eps)
    at = (*map(_call.sig, tensors), eps)
    plan = _PLANS.get(at)
    if plan is None:
        given = tensors
        tensors, plan = _plan(*given, eps)
        _PLANS.keep(at, given, tensors, plan)
    if _call.tracked(*tensors[:4]):
        return HeadNormFn.apply(*tensors, plan)  # (which refuses tangents)
    return _run(plan, tensors)
