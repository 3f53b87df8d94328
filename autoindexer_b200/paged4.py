"""The paged key / value cache in 4 bits: appending to it, reading it back and
attending over it.

Of a head row, 32 dims share a float16 scale ``d``, minus an eighth of their
value of largest magnitude; a dim's code ``c`` in 0..15 stands for ``(c - 8)
d``.  A token takes 144 bytes per KV head at head_dim 128 (keys and values
together) where bfloat16 takes 512.  Codes live in pools ``(n_pages, Hkv,
page_size, D / 2)`` of bytes (dim ``32 c + 4 g + j``, ``g < 8``, ``j < 4``, in
byte ``g D / 16 + 2 c + j // 2``, the low half for even ``j``), scales in pools
``(n_pages, Hkv, page_size, D / 32)``.  Page tables, lengths and graph capture
are as in the 16-bit cache (``paged_append``, ``shared_prefix_attention``);
sequences that share a prompt list the same pages.
"""

from __future__ import annotations

import ctypes
import operator
from typing import Optional, Tuple

import torch
from torch import Tensor

from . import _call, _lib
from .paged import _table

__all__ = ["paged_append_4bit", "paged_read_4bit", "paged_attention_4bit"]

MAX_BATCH = 1024  # sequences of an attention call
MAX_PAGE = 16777216  # slots of a page (AI_POOL4_MAX_PAGE)
GROUP = 32


def _pool(p, k_pages, v_pages, k_scales, v_scales, page_table, batch: int, heads: int, head_dim: int, index: int) -> Tensor:
    """Sets what ``p`` says of the pools, without pointers; returns the page table."""
    s = k_pages.shape
    if len(s) != 4 or s != v_pages.shape or s[1] != heads or s[3] != head_dim // 2:
        raise ValueError(f"k_pages and v_pages must be (n_pages, {heads}, page_size, {head_dim // 2}), got "
                         f"{tuple(s)} and {tuple(v_pages.shape)}")
    if s[0] == 0 or not 16 <= s[2] <= MAX_PAGE or s[2] & (s[2] - 1):
        raise ValueError(f"page_size must be a power of two from 16 to {MAX_PAGE} and the pools not empty, got {tuple(s)}")
    size = head_dim // GROUP
    for name, x, dtype, last in (("k_pages", k_pages, torch.uint8, s[3]), ("v_pages", v_pages, torch.uint8, s[3]),
                                 ("k_scales", k_scales, torch.float16, size), ("v_scales", v_scales, torch.float16, size)):
        if x.dtype is not dtype:
            raise TypeError(f"{name} must be {dtype}, got {x.dtype}")
        if x.shape != (*s[:3], last):
            raise ValueError(f"{name} must have shape {(*s[:3], last)}, got {tuple(x.shape)}")
        st = x.stride()
        if st[2] != last or (st[3] != 1 and last > 1):
            raise ValueError(f"the slots of a page and head of {name} must follow one another")
        if (st[0] | st[1]) * x.element_size() % 16:
            raise ValueError(f"the pages and heads of {name} must start on 16-byte boundaries")
        _call.on_device(name, x, index)
    page_table = _table(page_table, batch, index)
    if page_table.shape[1] == 0:
        raise ValueError("page_table has no columns")
    p.k_codes, p.v_codes, p.k_scales, p.v_scales = map(_call.strides4, (k_pages, v_pages, k_scales, v_scales))
    p.n_pages, p.page_size = s[0], s[2]
    p.page_table_stride, p.max_pages = page_table.stride(0), page_table.shape[1]
    return page_table


def _point(p, k_pages, v_pages, k_scales, v_scales, page_table) -> None:
    k, v, ks, vs = k_pages.data_ptr(), v_pages.data_ptr(), k_scales.data_ptr(), v_scales.data_ptr()
    if (k | v | ks | vs) & 15:
        raise ValueError("the pools must start on 16-byte boundaries")
    p.k_codes.ptr, p.v_codes.ptr, p.k_scales.ptr, p.v_scales.ptr = k, v, ks, vs
    p.page_table = page_table.data_ptr()


def _head_dim(D: int) -> None:
    if D not in (32, 64, 128):
        raise ValueError(f"head_dim must be 32, 64 or 128, got {D}")


_PLANS, _READ_PLANS, _ATTEND_PLANS = _call.Plans(), _call.Plans(), _call.Plans()


def _paged_plan(key, value, k_pages, v_pages, k_scales, v_scales, page_table, lens, n, name):
    """Checks the arguments of an append (or a read, with ``key`` and ``value`` for
    its results); returns the tensors the kernel reads and the argument struct
    without pointers."""
    index = _call.cuda_index("key", key)
    if key.dim() != 4 or key.shape != value.shape:
        raise ValueError(f"key and value must be (B, Hkv, T, D), got {tuple(key.shape)} and {tuple(value.shape)}")
    B, H, T, D = key.shape
    if key.numel() == 0:
        raise ValueError("key and value must not be empty")
    _head_dim(D)
    if value.dtype is not key.dtype:
        raise TypeError(f"value is {value.dtype}, key {key.dtype}")
    _call.on_device("value", value, index)
    a = _lib.AiPaged4Args()
    a.batch, a.num_kv_heads, a.seq_len, a.head_dim = B, H, T, D
    a.dtype = _call.dtype_code(key, "key")
    page_table = _pool(a.pool, k_pages, v_pages, k_scales, v_scales, page_table, B, H, D, index)
    lens = _call.ints("lens", lens, (B,), index)
    if n is not None:
        n = _call.ints(name, n, (B,), index)
    key, value = _call.dense_d(key), _call.dense_d(value)
    a.k, a.v = _call.strides4(key), _call.strides4(value)
    a.status = _call.status_ptr(index)
    return (key, value, k_pages, v_pages, k_scales, v_scales, page_table, lens, n), a


def _paged(fn, what, plan, tensors) -> None:
    k, v, k_pages, v_pages, k_scales, v_scales, page_table, lens, n = tensors
    a = _call.copy(plan)
    a.k.ptr, a.v.ptr, a.lens = k.data_ptr(), v.data_ptr(), lens.data_ptr()
    _point(a.pool, k_pages, v_pages, k_scales, v_scales, page_table)
    if n is not None:
        a.n = n.data_ptr()
    _call.launch(fn, a, k.get_device(), what)


def paged_append_4bit(key: Tensor, value: Tensor, k_pages: Tensor, v_pages: Tensor, k_scales: Tensor, v_scales: Tensor,
                      page_table: Tensor, lens: Tensor, new_lens: Optional[Tensor] = None) -> None:
    """Writes new tokens into the cache, in place.

    ``key`` (normalised and rotated: ``qk_norm_rope`` returns them so) and
    ``value`` ``(B, Hkv, T, D)``: token ``t < new_lens[b]`` (all ``T`` without
    it) becomes sequence ``b``'s token ``lens[b] + t``, in slot ``n %
    page_size`` of page ``page_table[b, n // page_size]``; ``lens`` ``(B,)``
    int32 is not changed.  A token whose page lies outside the table or the
    pool is dropped and sets the status word (so does a ``new_lens`` below 0
    or above ``T``, taken as 0 or ``T``).  32 dims with a NaN or an infinity
    among them read back as NaN; scales are limited to 65504.  ``key`` and
    ``value`` are CUDA tensors of one dtype (bfloat16, float16, float32),
    head_dim 32, 64 or 128, any strides; page sizes are powers of two from 16
    (to 2^24), and the slots of a page and head follow one another in the pools, from a
    16-byte boundary (pages and heads may be strided).  Two tokens given the same
    slot race; no gradient flows through the cache."""
    tensors = (key, value, k_pages, v_pages, k_scales, v_scales, page_table, lens, new_lens)
    at = tuple(_call.sigs(tensors))
    plan = _PLANS.get(at)
    if plan is None:
        given = tensors
        tensors, plan = _paged_plan(*given, "new_lens")
        _PLANS.keep(at, given, tensors, plan)
    _paged(_lib.lib().ai_paged_append_4bit, "ai_paged_append_4bit", plan, tensors)


def paged_read_4bit(k_pages: Tensor, v_pages: Tensor, k_scales: Tensor, v_scales: Tensor, page_table: Tensor, lens: Tensor,
                    n_tokens: int, dtype: torch.dtype, read_lens: Optional[Tensor] = None) -> Tuple[Tensor, Tensor]:
    """What the cache holds of each sequence's tokens ``lens[b] + t``, ``t <
    n_tokens``: keys and values ``(B, Hkv, n_tokens, D)``, rounded to ``dtype``
    (0 past ``read_lens[b]``, int32, and where there is no page).  The call that
    mirrors ``paged_append_4bit``, with its arguments: what a prefill that wrote
    to the cache attends to, or a sequence on its way to another cache."""
    tensors = (k_pages, v_pages, k_scales, v_scales, page_table, lens, read_lens)
    n_tokens = operator.index(n_tokens)  # (a number: a plan kept by a tensor would outlive its value)
    at = (*_call.sigs(tensors), n_tokens, dtype)
    known = _READ_PLANS.get(at)
    if known is None:
        if page_table.dim() != 2 or k_pages.dim() != 4 or n_tokens < 1:
            raise ValueError(f"page_table must be (B, max_pages), k_pages (n_pages, Hkv, page_size, D / 2), n_tokens 1 or more, "
                             f"got {tuple(page_table.shape)}, {tuple(k_pages.shape)}, {n_tokens}")
        shape = (page_table.shape[0], k_pages.shape[1], n_tokens, 2 * k_pages.shape[3])
        given, like = tensors, torch.empty(shape, dtype=dtype, device=k_pages.device)
        (_, _, *tensors), plan = _paged_plan(like, like, *given, "read_lens")
        known = (shape, plan)
        _READ_PLANS.keep(at, given, tensors, known)
    shape, plan = known
    k = k_pages.new_empty(shape, dtype=dtype)
    v = k.new_empty(shape)
    _paged(_lib.lib().ai_paged_read_4bit, "ai_paged_read_4bit", plan, (k, v, *tensors))
    return k, v


def _attend_plan(query, k_pages, v_pages, k_scales, v_scales, page_table, lens, query_lens, scaling):
    """Checks the arguments; returns the tensors the kernels read and the
    argument struct without pointers."""
    index = _call.cuda_index("query", query)
    if query.dim() != 4 or query.numel() == 0:
        raise ValueError(f"query must be (B, Hq, T, D) and not empty, got {tuple(query.shape)}")
    B, Hq, T, D = query.shape
    _head_dim(D)
    if query.dtype not in (torch.bfloat16, torch.float16):
        raise TypeError(f"query must be bfloat16 or float16, got {query.dtype}")
    if B > MAX_BATCH:
        raise ValueError(f"at most {MAX_BATCH} sequences, got {B}: split the batch")
    heads = k_pages.shape[1] if k_pages.dim() == 4 else 0
    if heads == 0 or Hq % heads != 0:
        raise ValueError(f"num_q_heads {Hq} is not a multiple of num_kv_heads {heads}")
    a = _lib.AiPagedAttn4Args()
    a.batch, a.num_q_heads, a.num_kv_heads, a.seq_len, a.head_dim = B, Hq, heads, T, D
    a.dtype = _call.dtype_code(query, "query")
    a.scale = scaling if scaling is not None else D ** -0.5
    page_table = _pool(a.pool, k_pages, v_pages, k_scales, v_scales, page_table, B, heads, D, index)
    lens = _call.ints("lens", lens, (B,), index)
    if query_lens is not None:
        query_lens = _call.ints("query_lens", query_lens, (B,), index)
    q = _call.dense_d(query)
    a.q = _call.strides4(q)
    a.out = _lib.AiTensor4(None, T * Hq * D, D, Hq * D)
    a.status = _call.status_ptr(index)
    # (the workspace's size goes by the signature too; it is asked for with the pointers set)
    asked = _call.copy(a)
    asked.q.ptr = asked.out.ptr = q.data_ptr()
    asked.lens = lens.data_ptr()
    _point(asked.pool, k_pages, v_pages, k_scales, v_scales, page_table)
    n = ctypes.c_size_t(0)
    with torch.cuda.device(index):  # (by the device's SMs)
        _lib.check(_lib.lib().ai_paged_attn_4bit_workspace(asked, n), "ai_paged_attn_4bit_workspace")
    a.workspace_bytes = n.value
    return (q, k_pages, v_pages, k_scales, v_scales, page_table, lens, query_lens), a


def paged_attention_4bit(query: Tensor, k_pages: Tensor, v_pages: Tensor, k_scales: Tensor, v_scales: Tensor,
                         page_table: Tensor, lens: Tensor, scaling: Optional[float] = None,
                         query_lens: Optional[Tensor] = None, return_lse: bool = False):
    """Attention of each sequence's new tokens over its cache in 4 bits.

    ``query`` ``(B, Hq, T, D)`` (normalised and rotated, bfloat16 or float16):
    query token ``t < query_lens[b]`` (all ``T`` without it) sees the first
    ``lens[b] - query_lens[b] + t + 1`` keys of the pages in row ``b`` of
    ``page_table``, so ``lens`` ``(B,)`` int32 counts the new tokens, already
    appended.  Returns ``(B, T, Hq, D)`` (and the float32 log-sum-exp ``(B, Hq,
    T)`` with ``return_lse``); a padding token, or one without a key, gives
    zeros and ``-inf``.  ``scaling`` defaults to ``D ** -0.5``.

    Keys and values are taken as the cache stands for them; scores, sums and the
    softmax are float32, and the products of weights and the values' scales are
    rounded to float16 once: to 2^-11 of themselves and 2^-30 of the largest
    weight times the largest scale of their 32 dims.  Padding tokens, and slots that
    no query of the sequence sees, may hold anything.  Up to 1024 sequences, head_dim 32, 64 or 128, any strides of the
    query; the pools as ``paged_append_4bit`` takes them.  A length or page out
    of range is clamped and sets the status word.  There is no gradient: a
    backward through the results raises."""
    tensors = (query, k_pages, v_pages, k_scales, v_scales, page_table, lens, query_lens)
    scaling = None if scaling is None else float(scaling)
    at = (*_call.sigs(tensors), scaling)
    plan = _ATTEND_PLANS.get(at)
    if plan is None:
        given = tensors
        tensors, plan = _attend_plan(*given, scaling)
        _ATTEND_PLANS.keep(at, given, tensors, plan)
    if _call.tracked(query, k_scales, v_scales):
        return _call.no_backward("paged_attention_4bit", lambda: _attend(plan, tensors, return_lse), query, k_scales, v_scales)
    return _attend(plan, tensors, return_lse)


def _attend(plan, tensors, return_lse):
    q, k_pages, v_pages, k_scales, v_scales, page_table, lens, query_lens = tensors
    B, Hq, T, D = q.shape
    out = q.new_empty((B, T, Hq, D))
    a = _call.copy(plan)
    a.q.ptr, a.out.ptr, a.lens = q.data_ptr(), out.data_ptr(), lens.data_ptr()
    _point(a.pool, k_pages, v_pages, k_scales, v_scales, page_table)
    if query_lens is not None:
        a.query_lens = query_lens.data_ptr()
    lse = None
    if return_lse:
        lse = q.new_empty((B, Hq, T), dtype=torch.float32)
        a.lse = lse.data_ptr()
    ws = k_pages.new_empty(a.workspace_bytes)
    a.workspace = ws.data_ptr()
    _call.launch(_lib.lib().ai_paged_attn_4bit, a, q.get_device(), "ai_paged_attn_4bit")
    del ws
    return (out, lse) if return_lse else out
