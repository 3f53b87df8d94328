"""The paged key / value cache: appending to it and attending over it.

Keys and values live in pools of pages ``(n_pages, Hkv, page_size, D)``; a
sequence's tokens are the slots of the pages its row of ``page_table`` lists,
and a batch may share a prefix whose pages are listed once.  All lengths and
tables are device tensors, nothing synchronises, and the calls can be captured
in a CUDA graph (the page tables' width and ``prefix_len`` fix the launch).

Keys are stored as the scores use them: ``paged_append`` normalises and
rotates them on the way in.
"""

from __future__ import annotations

from typing import Optional, Tuple

import torch
from torch import Tensor

from . import _call, _lib

__all__ = ["paged_append", "shared_prefix_attention"]

MAX_BATCH = 65535  # sequences of an attention call


def _pools(k_pages: Tensor, v_pages: Tensor, heads: int, head_dim: int, dtype, index: int) -> None:
    s = k_pages.shape
    if len(s) != 4 or s != v_pages.shape or s[1] != heads or s[3] != head_dim:
        raise ValueError(f"k_pages and v_pages must be (n_pages, {heads}, page_size, {head_dim}), got "
                         f"{tuple(k_pages.shape)} and {tuple(v_pages.shape)}")
    if s[0] == 0 or s[2] == 0:
        raise ValueError("k_pages and v_pages are empty")
    for name, p in (("k_pages", k_pages), ("v_pages", v_pages)):
        if p.dtype is not dtype:
            raise TypeError(f"{name} is {p.dtype}, the call's tensors {dtype}")
        if p.stride(3) != 1:
            raise ValueError(f"{name} must have a contiguous last dimension")
        _call.on_device(name, p, index)


def _table(page_table: Tensor, batch: int, index: int) -> Tensor:
    if page_table.dim() != 2:
        raise ValueError(f"page_table must be ({batch}, max_pages), got {tuple(page_table.shape)}")
    return _call.ints("page_table", page_table, (batch, page_table.shape[1]), index)


_APPEND_PLANS, _ATTEND_PLANS = _call.Plans(), _call.Plans()


def _append_plan(key, value, k_pages, v_pages, page_table, lens, new_lens, key_weight, cos, sin, positions, eps):
    """Checks the arguments; returns the tensors the kernel reads and the
    argument struct without pointers."""
    index = _call.cuda_index("key", key)
    if key.dim() != 4 or key.shape != value.shape:
        raise ValueError(f"key and value must be (B, Hkv, T, D), got {tuple(key.shape)} and {tuple(value.shape)}")
    B, H, T, D = key.shape
    if key.numel() == 0:
        raise ValueError("key and value must not be empty")
    if D not in (32, 64, 128):
        raise ValueError(f"head_dim must be 32, 64 or 128, got {D}")
    if value.dtype is not key.dtype:
        raise TypeError(f"value is {value.dtype}, key {key.dtype}")
    _call.on_device("value", value, index)
    _pools(k_pages, v_pages, H, D, key.dtype, index)
    page_table = _table(page_table, B, index)
    if page_table.shape[1] == 0:
        raise ValueError("page_table has no columns")
    lens = _call.ints("lens", lens, (B,), index)
    if new_lens is not None:
        new_lens = _call.ints("new_lens", new_lens, (B,), index)
    w = _call.head_weight("key_weight", key_weight, key, index)
    k, v = _call.dense_d(key), _call.dense_d(value)
    a = _lib.AiPagedAppendArgs()
    a.batch, a.num_kv_heads, a.seq_len, a.head_dim = B, H, T, D
    a.dtype = _call.dtype_code(key, "key")
    a.weight_dtype = a.dtype if w is None else _call.dtype_code(w, "key_weight")
    a.eps = eps
    a.k, a.v, a.k_pages, a.v_pages = map(_call.strides4, (k, v, k_pages, v_pages))
    a.n_pages, a.page_size = k_pages.shape[0], k_pages.shape[2]
    a.page_table_stride, a.max_pages = page_table.stride(0), page_table.shape[1]
    cos, sin, positions = _call.check_rope(a, None if cos is None else (cos, sin), positions, B, T, D, index)
    a.status = _call.status_ptr(index)
    return (k, v, k_pages, v_pages, page_table, lens, new_lens, w, cos, sin, positions), a


def paged_append(key: Tensor, value: Tensor, k_pages: Tensor, v_pages: Tensor, page_table: Tensor, lens: Tensor,
                 rope: Optional[Tuple[Tensor, Tensor]] = None, positions: Optional[Tensor] = None,
                 new_lens: Optional[Tensor] = None, key_weight: Optional[Tensor] = None, eps: float = 1e-6) -> None:
    """Writes new tokens into the cache, in place.

    ``key`` and ``value`` ``(B, Hkv, T, D)``: token ``t < new_lens[b]`` (all
    ``T`` without it) becomes sequence ``b``'s token ``lens[b] + t``, in slot
    ``n % page_size`` of page ``page_table[b, n // page_size]``.  ``lens``
    ``(B,)`` int32 counts the tokens a sequence holds already and is not
    changed.  ``key_weight`` (``(D,)``) normalises each key row as
    ``qk_norm_rope`` does, ``rope`` / ``positions`` rotate it (as there).
    ``page_table`` ``(B, max_pages)`` int32; a token whose page lies outside
    it or outside the pool is dropped and sets the status word (so does a
    ``new_lens`` below 0 or above ``T``, taken as 0 or ``T``).  CUDA tensors
    of one dtype (bfloat16, float16, float32), head_dim 32, 64 or 128, any
    page size, any strides with the last dimension contiguous.  Two tokens
    given the same slot race; no gradient flows through the cache."""
    cos, sin = (None, None) if rope is None else rope
    tensors = (key, value, k_pages, v_pages, page_table, lens, new_lens, key_weight, cos, sin, positions)
    eps = float(eps)
    at = (*map(_call.sig, tensors), eps)
    plan = _APPEND_PLANS.get(at)
    if plan is None:
        given = tensors
        tensors, plan = _append_plan(*given, eps)
        _APPEND_PLANS.keep(at, given, tensors, plan)
    k, v, k_pages, v_pages, page_table, lens, new_lens, w, cos, sin, positions = tensors
    a = _call.copy(plan)
    a.k.ptr, a.v.ptr = k.data_ptr(), v.data_ptr()
    a.k_pages.ptr, a.v_pages.ptr = k_pages.data_ptr(), v_pages.data_ptr()
    a.page_table, a.lens = page_table.data_ptr(), lens.data_ptr()
    if new_lens is not None:
        a.new_lens = new_lens.data_ptr()
    if w is not None:
        a.k_weight = w.data_ptr()
    _call.point_rope(a, cos, sin, positions)
    _call.launch(_lib.lib().ai_paged_append, a, k.get_device(), "ai_paged_append")


def _attend_plan(query, k_pages, v_pages, prefix_pages, page_table, lens, query_lens, prefix_len, scaling):
    """Checks the arguments; returns the tensors the kernels read and the
    argument struct without pointers."""
    index = _call.cuda_index("query", query)
    if query.dim() != 4 or query.numel() == 0:
        raise ValueError(f"query must be (B, Hq, T, D) and not empty, got {tuple(query.shape)}")
    B, Hq, T, D = query.shape
    if D not in (32, 64, 128):
        raise ValueError(f"head_dim must be 32, 64 or 128, got {D}")
    if B > MAX_BATCH:
        raise ValueError(f"at most {MAX_BATCH} sequences, got {B}: split the batch")
    heads = k_pages.shape[1] if k_pages.dim() == 4 else 0
    if heads == 0 or Hq % heads != 0:
        raise ValueError(f"num_q_heads {Hq} is not a multiple of num_kv_heads {heads}")
    _pools(k_pages, v_pages, heads, D, query.dtype, index)
    S = k_pages.shape[2]
    page_table = _table(page_table, B, index)
    lens = _call.ints("lens", lens, (B,), index)
    if query_lens is not None:
        query_lens = _call.ints("query_lens", query_lens, (B,), index)
    if prefix_len < 0:
        raise ValueError(f"prefix_len {prefix_len} is negative")
    if prefix_len:
        if prefix_pages is None or prefix_pages.dim() != 1 or prefix_pages.shape[0] * S < prefix_len:
            raise ValueError(f"prefix_pages must list the pages of {prefix_len} keys ({S} a page)")
        prefix_pages = _call.ints("prefix_pages", prefix_pages, (prefix_pages.shape[0],), index)
    q = _call.dense_d(query)
    st = q.stride()
    if q.data_ptr() % 16 or (st[0] | st[1] | st[2]) * q.element_size() % 16:
        q = q.clone(memory_format=torch.contiguous_format)  # the kernels read 16-byte pieces of its rows
    a = _lib.AiPrefixAttnArgs()
    a.batch, a.num_q_heads, a.seq_len, a.head_dim = B, Hq, T, D
    a.num_kv_heads = heads
    a.dtype = _call.dtype_code(query, "query")
    a.scale = scaling if scaling is not None else D ** -0.5
    a.q, a.k_pages, a.v_pages = map(_call.strides4, (q, k_pages, v_pages))
    a.out = _lib.AiTensor4(None, T * Hq * D, D, Hq * D)
    a.n_pages, a.page_size, a.prefix_len = k_pages.shape[0], S, prefix_len
    a.page_table_stride, a.max_pages = page_table.stride(0), page_table.shape[1]
    a.status = _call.status_ptr(index)
    return (q, k_pages, v_pages, prefix_pages, page_table, lens, query_lens), a


def shared_prefix_attention(query: Tensor, k_pages: Tensor, v_pages: Tensor, prefix_pages: Optional[Tensor],
                            prefix_len: int, page_table: Tensor, lens: Tensor, scaling: Optional[float] = None,
                            query_lens: Optional[Tensor] = None, return_lse: bool = False):
    """Attention of a batch over its shared prefix and each sequence's own tokens.

    ``query`` ``(B, Hq, T, D)`` (normalised and rotated): query token ``t <
    query_lens[b]`` (all ``T`` without it) sees the ``prefix_len`` keys of
    ``prefix_pages`` (int32) and the first ``lens[b] - query_lens[b] + t + 1``
    keys of the pages in row ``b`` of ``page_table``, so ``lens`` ``(B,)``
    int32 counts the new tokens, already appended.  Returns ``(B, T, Hq, D)``
    (and the float32 log-sum-exp ``(B, Hq, T)`` with ``return_lse``); a padding
    token, or one without a key, gives zeros and ``-inf``.  ``scaling``
    defaults to ``D ** -0.5``.  With ``prefix_len`` 0 it is plain paged
    decoding.

    CUDA tensors of one dtype, head_dim 32, 64 or 128, any page size, any
    strides with the last dimension contiguous, up to 65535 sequences.  The keys that some query of
    the sequence sees must hold finite values; the slots past them may hold
    anything.  A length or page out of range is clamped and sets the status
    word.  There is no gradient: a backward through the results raises."""
    prefix_len = int(prefix_len)
    if prefix_len == 0:
        prefix_pages = None
    tensors = (query, k_pages, v_pages, prefix_pages, page_table, lens, query_lens)
    scaling = None if scaling is None else float(scaling)
    at = (*map(_call.sig, tensors), prefix_len, scaling, query.data_ptr() % 16)
    plan = _ATTEND_PLANS.get(at)
    if plan is None:
        given = tensors
        tensors, plan = _attend_plan(*given, prefix_len, scaling)
        _ATTEND_PLANS.keep(at, given, tensors, plan)
    if _call.tracked(query, k_pages, v_pages):
        return _call.no_backward("shared_prefix_attention", lambda: _attend(plan, tensors, return_lse), query, k_pages, v_pages)
    return _attend(plan, tensors, return_lse)


def _attend(plan, tensors, return_lse):
    q, k_pages, v_pages, prefix_pages, page_table, lens, query_lens = tensors
    B, Hq, T, D = q.shape
    device = q.device
    out = torch.empty((B, T, Hq, D), dtype=q.dtype, device=device)
    a = _call.copy(plan)
    a.q.ptr, a.out.ptr = q.data_ptr(), out.data_ptr()
    a.k_pages.ptr, a.v_pages.ptr = k_pages.data_ptr(), v_pages.data_ptr()
    if prefix_pages is not None:
        a.prefix_pages = prefix_pages.data_ptr()
    a.page_table, a.lens = page_table.data_ptr(), lens.data_ptr()
    if query_lens is not None:
        a.query_lens = query_lens.data_ptr()
    lse = None
    if return_lse:
        lse = torch.empty((B, Hq, T), dtype=torch.float32, device=device)
        a.lse = lse.data_ptr()
    lib = _lib.lib()
    ws = _call.workspace(lib.ai_prefix_attn_workspace, a, device, "ai_prefix_attn_workspace")
    _call.launch(lib.ai_prefix_attn, a, q.get_device(), "ai_prefix_attn")
    del ws
    return (out, lse) if return_lse else out
