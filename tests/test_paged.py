"""The paged cache: ``paged_append`` and ``shared_prefix_attention`` against
64-bit restatements, at the lengths, masks, page sizes and strides where they
can go wrong, and their refusals.

Tolerances.  Appended keys: as for the norms (``test_head_norm.py``); values
are copied exactly.  Attention: the probabilities may be rounded to the
tensors' type before they meet the values and the output is, each a relative
``u`` of ``sum p |v|``; a score of float32 sums is off by at most ``4 D 2^-24
A`` with A the largest ``scale * sum |q k|``, which enters twice (numerator
and sum), and the exponentials and sums by less than 2^-16."""

import ctypes

import numpy as np
import pytest
import torch

from oracle import operator_oracle as O
from test_head_norm import U, _close, _np, _table

EPS = 1e-6


def _pages(P, H, S, D, dtype, device, order="phsd", fill=float("nan")):
    shape = {"phsd": (P, H, S, D), "pshd": (P, S, H, D), "odd": (P, H, S, D + 3)}[order]
    x = torch.full(shape, fill, dtype=dtype, device=device)
    return x.transpose(1, 2) if order == "pshd" else x[..., 1:D + 1] if order == "odd" else x


APPEND = [
    # B, T, H, D, S, dtype, order, rope, weight, ragged
    (1, 1, 1, 128, 16, torch.bfloat16, "phsd", True, True, False),
    (64, 1, 8, 128, 64, torch.bfloat16, "phsd", True, True, False),
    (3, 37, 8, 128, 16, torch.float16, "pshd", True, False, True),
    (2, 65, 3, 64, 48, torch.bfloat16, "phsd", False, True, True),
    (5, 7, 2, 32, 1, torch.float32, "odd", True, True, True),
    (2, 1030, 4, 64, 128, torch.float32, "phsd", False, False, True),
]


@pytest.mark.gpu
@pytest.mark.parametrize("B,T,H,D,S,dtype,order,rot,normed,ragged", APPEND)
def test_append(B, T, H, D, S, dtype, order, rot, normed, ragged, cuda_device):
    from autoindexer_b200 import paged_append, read_status

    g = torch.Generator().manual_seed(B + T)
    k, v = (torch.randn(B, T, H, D, generator=g).to(dtype).to(cuda_device).transpose(1, 2) for _ in range(2))
    w = (1 + 0.3 * torch.randn(D, generator=g)).to(dtype).to(cuda_device) if normed else None
    lens = torch.randint(0, 3 * S, (B,), generator=g).int()
    lens[0] = 0
    M = (int(lens.max()) + T + S - 1) // S
    table = torch.randperm(B * M + 3, generator=g)[:B * M].reshape(B, M).int()
    n = torch.randint(0, T + 1, (B,), generator=g).int() if ragged else torch.full((B,), T).int()
    kp, vp = (_pages(B * M + 3, H, S, D, dtype, cuda_device, order, fill=7.0) for _ in range(2))
    rope = _table(301, D, cuda_device) if rot else None
    pos = torch.randint(0, 301, (B, T), generator=g).to(cuda_device) if rot else None
    paged_append(k, v, kp, vp, table.to(cuda_device), lens.to(cuda_device), rope, pos,
                 n.to(cuda_device) if ragged else None, w, EPS)
    assert read_status(cuda_device) == 0
    cos, sin = (None, None) if rope is None else (_np(r) for r in rope)
    want, mag = O.head_norm(_np(k), _np(w), cos, sin, None if pos is None else _np(pos).astype(int), EPS)
    gk, gv = kp.float().cpu(), vp.float().cpu()
    touched = torch.zeros(kp.shape[0], S, dtype=torch.bool)
    for b, t, page, slot in O.append_slots(lens, n, table.numpy(), S):
        _close(gk[page, :, slot], want[b, :, t], mag[b, :, t], dtype, D)
        assert torch.equal(gv[page, :, slot], v[b, :, t].float().cpu())
        touched[page, slot] = True
    assert int(touched.sum()) == int(n.sum())
    rest = ~touched[:, None, :, None].expand(gk.shape)
    assert torch.all(gk[rest] == 7) and torch.all(gv[rest] == 7)  # nothing else was written


@pytest.mark.gpu
def test_append_out_of_range_tokens_are_dropped(cuda_device):
    from autoindexer_b200 import paged_append, read_status

    k = torch.randn(3, 2, 2, 64, device=cuda_device)
    kp, vp = (_pages(4, 2, 16, 64, torch.float32, cuda_device, fill=7.0) for _ in range(2))
    table = torch.tensor([[0, 1], [4, 2], [3, -1]], dtype=torch.int32, device=cuda_device)
    lens = torch.tensor([31, 0, 16], dtype=torch.int32, device=cuda_device)
    read_status(cuda_device)
    paged_append(k, k, kp, vp, table, lens)
    assert read_status(cuda_device) == -2
    assert torch.equal(kp[1, :, 15], k[0, :, 0])  # the one token that has a place
    kp[1, :, 15] = 7
    assert torch.all(kp == 7)


def _cache(B, T, Hq, Hkv, D, S, P, lens, dtype, seed, device, order="phsd", scale=2.0):
    """A cache whose slots past the held tokens are NaN, and its queries."""
    g = torch.Generator().manual_seed(seed)
    M = max(1, -(-max(lens) // S))
    np_ = -(-P // S)
    ids = torch.randperm(np_ + B * M + 2, generator=g).int()
    table, prefix = ids[np_:np_ + B * M].reshape(B, M).contiguous(), ids[:np_].contiguous()
    kp, vp = (_pages(np_ + B * M + 2, Hkv, S, D, dtype, device, order) for _ in range(2))
    for pages in (kp, vp):
        for i in range(np_):
            m = min(S, P - i * S)
            pages[int(prefix[i]), :, :m] = torch.randn(Hkv, m, D, generator=g).to(dtype).to(device)
        for b in range(B):
            for i in range(-(-lens[b] // S)):
                m = min(S, lens[b] - i * S)
                pages[int(table[b, i]), :, :m] = torch.randn(Hkv, m, D, generator=g).to(dtype).to(device)
        # table entries past the held tokens point nowhere
    for b in range(B):
        table[b, -(-lens[b] // S):] = -5
    q = (scale * torch.randn(B, T, Hq, D, generator=g)).to(dtype).to(device).transpose(1, 2)
    return q, kp, vp, prefix.to(device), table.to(device)


def _check(q, kp, vp, prefix, P, table, lens, n, out, lse, scale, dtype):
    want, wlse, mag, most = O.prefix_attention(_np(q), _np(kp), _np(vp), prefix.cpu().numpy(), P, table.cpu().numpy(),
                                               lens, n, scale)
    D = q.shape[-1]
    eps = 2 * 4 * D * 2.0 ** -24 * most + 2.0 ** -16
    err = np.abs(_np(out) - want)
    tol = (2 * U[dtype] + eps) * mag
    assert np.all(err <= tol), float((err / np.maximum(tol, 1e-300)).max())
    if lse is not None:
        got = _np(lse)
        none = np.isinf(wlse)
        assert np.array_equal(np.isneginf(got), none)
        assert np.all(np.abs(got[~none] - wlse[~none]) <= eps * (1 + np.abs(wlse[~none])))


ATTEND = [
    # B, T, Hq, Hkv, D, S, P, own lengths, query lengths, dtype
    (1, 1, 1, 1, 128, 16, 0, [1], None, torch.bfloat16),
    (1, 1, 4, 1, 128, 64, 1, [0], None, torch.bfloat16),            # the prefix alone
    (2, 1, 8, 2, 128, 64, 0, [0, 3], None, torch.bfloat16),         # a row without any key
    (3, 1, 32, 8, 128, 16, 257, [1, 64, 65], None, torch.bfloat16),
    (4, 1, 32, 8, 128, 64, 130, [63, 64, 1, 200], None, torch.float16),
    (5, 3, 8, 2, 128, 32, 95, [3, 40, 2, 129, 65], [3, 2, 1, 3, 0], torch.bfloat16),
    (2, 5, 16, 2, 64, 128, 300, [5, 131], [5, 4], torch.float16),
    (3, 2, 6, 2, 64, 16, 64, [2, 17, 33], [1, 2, 2], torch.bfloat16),   # three query heads a KV head
    (2, 40, 16, 2, 128, 64, 190, [40, 100], [40, 37], torch.bfloat16),  # more query rows than a tile
    (9, 4, 16, 4, 128, 64, 700, [4, 5, 70, 128, 129, 64, 9, 300, 61], [4, 3, 4, 1, 2, 4, 4, 4, 1], torch.bfloat16),
    (40, 1, 8, 1, 64, 32, 513, list(range(1, 80, 2)), None, torch.float16),  # many sequences, one KV head
    (2, 3, 4, 2, 128, 64, 100, [1, 2], [3, 3], torch.bfloat16),     # fewer own keys than query tokens
    (2, 2, 4, 2, 32, 16, 40, [5, 18], None, torch.bfloat16),
    (2, 2, 4, 2, 64, 24, 50, [5, 49], [2, 1], torch.float16),       # a page size that is no power of two
    (2, 2, 4, 4, 128, 16, 33, [5, 18], None, torch.float32),
    (1, 1, 24, 8, 128, 128, 4000, [1000], None, torch.bfloat16),    # split over many CTAs
    (1, 1, 4, 1, 64, 64, 20011, [3], None, torch.float16),
]


@pytest.mark.gpu
@pytest.mark.parametrize("B,T,Hq,Hkv,D,S,P,lens,n,dtype", ATTEND)
def test_attention(B, T, Hq, Hkv, D, S, P, lens, n, dtype, cuda_device):
    from autoindexer_b200 import read_status, shared_prefix_attention

    q, kp, vp, prefix, table = _cache(B, T, Hq, Hkv, D, S, P, lens, dtype, 31, cuda_device)
    as_t = lambda x: torch.tensor(x, dtype=torch.int32, device=cuda_device)  # noqa: E731
    ql = None if n is None else as_t(n)
    read_status(cuda_device)
    out, lse = shared_prefix_attention(q, kp, vp, prefix, P, table, as_t(lens), query_lens=ql, return_lse=True)
    assert read_status(cuda_device) == 0
    assert out.shape == (B, T, Hq, D) and out.dtype == dtype
    _check(q, kp, vp, prefix, P, table, lens, n or [T] * B, out, lse, D ** -0.5, dtype)
    again = shared_prefix_attention(q, kp, vp, prefix, P, table, as_t(lens), query_lens=ql)
    assert torch.equal(again, out)


@pytest.mark.gpu
@pytest.mark.parametrize("order", ["pshd", "odd"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_attention_other_orders(order, dtype, cuda_device):
    """Pages with the slot before the head, and rows off every 16-byte boundary; queries not 16-byte aligned too."""
    from autoindexer_b200 import shared_prefix_attention

    lens = [70, 3]
    q, kp, vp, prefix, table = _cache(2, 2, 8, 2, 128, 32, 75, lens, dtype, 5, cuda_device, order)
    if order == "odd":
        wide = torch.zeros(2, 8, 2, 131, dtype=dtype, device=cuda_device)
        wide[..., 1:129] = q
        q = wide[..., 1:129]
    out, lse = shared_prefix_attention(q, kp, vp, prefix, 75, table, torch.tensor(lens, dtype=torch.int32, device=cuda_device),
                                       scaling=0.05, return_lse=True)
    _check(q, kp, vp, prefix, 75, table, lens, [2, 2], out, lse, 0.05, dtype)


@pytest.mark.gpu
def test_attention_extreme_scores(cuda_device):
    """Scores that grow along the keys by hundreds (the running maximum moves
    at every tile), and a key that takes all the weight."""
    from autoindexer_b200 import shared_prefix_attention

    P, lens = 520, [130, 7]
    q, kp, vp, prefix, table = _cache(2, 1, 8, 2, 128, 64, P, lens, torch.bfloat16, 6, cuda_device, scale=1.0)
    for i in range(-(-P // 64)):
        kp[int(prefix[i])] *= 4.0 * (i + 1)
    kp[int(table[0, 1])] *= 64.0
    out, lse = shared_prefix_attention(q, kp, vp, prefix, P, table, torch.tensor(lens, dtype=torch.int32, device=cuda_device),
                                       return_lse=True)
    _check(q, kp, vp, prefix, P, table, lens, [1, 1], out, lse, 128 ** -0.5, torch.bfloat16)


@pytest.mark.gpu
@pytest.mark.parametrize("T,P,dtype", [(1, 200, torch.bfloat16), (1, 5000, torch.bfloat16), (20, 200, torch.float16),
                                       (70, 200, torch.bfloat16), (1, 200, torch.float32), (3, 5000, torch.float32)])
def test_attention_nan_stays_with_the_rows_that_see_it(T, P, dtype, cuda_device):
    """A NaN among a sequence's keys makes its rows of that KV head NaN, and no other."""
    from autoindexer_b200 import shared_prefix_attention

    lens = [T + 70, T + 5, T + 64]
    q, kp, vp, prefix, table = _cache(3, T, 8, 2, 128, 64, P, lens, dtype, 12, cuda_device)
    held = torch.tensor(lens, dtype=torch.int32, device=cuda_device)
    want, wlse = shared_prefix_attention(q, kp, vp, prefix, P, table, held, return_lse=True)
    kp[int(table[1, 0]), 0, 2, 5] = float("nan")
    got, lse = shared_prefix_attention(q, kp, vp, prefix, P, table, held, return_lse=True)
    assert got[1, :, :4].isnan().all() and lse[1, :4].isnan().all()
    for b, heads in ((0, slice(0, 8)), (1, slice(4, 8)), (2, slice(0, 8))):
        assert torch.equal(got[b, :, heads], want[b, :, heads]) and torch.equal(lse[b, heads], wlse[b, heads])


MORE = [
    # as ATTEND: the kernels for other types and layouts, and more sequences than a scan holds
    (16, 1, 32, 8, 128, 64, 1000, list(range(3, 99, 6)), None, torch.float32),
    (3, 7, 24, 8, 128, 48, 333, [7, 130, 64], [7, 2, 0], torch.bfloat16),
    (2, 5, 8, 1, 64, 64, 4099, [500, 5], [5, 4], torch.float32),
    (1, 1, 2, 2, 32, 32, 0, [0], None, torch.float16),
    (4, 2, 4, 2, 32, 128, 129, [2, 128, 129, 400], [1, 2, 2, 2], torch.float32),
    (1030, 1, 4, 2, 64, 16, 40, [1 + i % 7 for i in range(1030)], None, torch.bfloat16),
    (30, 5, 32, 8, 128, 64, 900, [5 + 3 * i for i in range(30)], [1 + i % 5 for i in range(30)], torch.float16),
    (3, 90, 16, 4, 128, 32, 600, [90, 160, 91], [90, 17, 1], torch.bfloat16),
]


@pytest.mark.gpu
@pytest.mark.parametrize("B,T,Hq,Hkv,D,S,P,lens,n,dtype", MORE)
def test_attention_more(B, T, Hq, Hkv, D, S, P, lens, n, dtype, cuda_device):
    test_attention(B, T, Hq, Hkv, D, S, P, lens, n, dtype, cuda_device)


SIDE = [
    # as ATTEND: more than 128 rows on the prefix, own lists from none to far more work than the prefix
    (40, 1, 8, 1, 128, 64, 700, [0] * 40, None, torch.bfloat16),
    (40, 1, 8, 1, 128, 64, 5000, [0] * 39 + [700], None, torch.float16),
    (33, 2, 16, 2, 64, 16, 2900, [2 + 61 * (i % 5) for i in range(33)], [i % 3 for i in range(33)], torch.bfloat16),
    (24, 5, 32, 4, 128, 128, 2500, [5 + 37 * i for i in range(24)], [5 - i % 4 for i in range(24)], torch.bfloat16),
    (20, 1, 16, 1, 64, 64, 9000, [100] * 20, [0] * 20, torch.bfloat16),  # no query at all
]


@pytest.mark.gpu
@pytest.mark.parametrize("B,T,Hq,Hkv,D,S,P,lens,n,dtype", SIDE)
def test_attention_side_by_side(B, T, Hq, Hkv, D, S, P, lens, n, dtype, cuda_device):
    test_attention(B, T, Hq, Hkv, D, S, P, lens, n, dtype, cuda_device)


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [129, 161, 191, 193, 255, 257])
def test_attention_row_counts(rows, cuda_device):
    """Numbers of rows on one prefix that no tile, warp or half of one divides."""
    test_attention(rows, 1, 2, 2, 64, 32, 700, [1 + i % 70 for i in range(rows)], None, torch.bfloat16, cuda_device)


@pytest.mark.gpu
def test_attention_negative_scale(cuda_device):
    from autoindexer_b200 import shared_prefix_attention

    lens = [70, 3]
    q, kp, vp, prefix, table = _cache(2, 2, 8, 2, 128, 32, 75, lens, torch.bfloat16, 5, cuda_device)
    out, lse = shared_prefix_attention(q, kp, vp, prefix, 75, table, torch.tensor(lens, dtype=torch.int32, device=cuda_device),
                                       scaling=-0.05, return_lse=True)
    _check(q, kp, vp, prefix, 75, table, lens, [2, 2], out, lse, -0.05, torch.bfloat16)


@pytest.mark.gpu
def test_attention_bad_lengths_and_pages_are_reported(cuda_device):
    from autoindexer_b200 import read_status, shared_prefix_attention

    q, kp, vp, prefix, table = _cache(2, 1, 4, 2, 128, 64, 64, [64, 64], torch.bfloat16, 6, cuda_device)
    as_t = lambda x: torch.tensor(x, dtype=torch.int32, device=cuda_device)  # noqa: E731
    read_status(cuda_device)
    want = shared_prefix_attention(q, kp, vp, prefix, 64, table, as_t([64, 64]))
    assert read_status(cuda_device) == 0
    got = shared_prefix_attention(q, kp, vp, prefix, 64, table, as_t([64, 1000]))  # clamped to the table
    assert read_status(cuda_device) == -2 and torch.equal(got, want)
    got = shared_prefix_attention(q, kp, vp, prefix, 64, table, as_t([64, -3]))
    assert read_status(cuda_device) == -2 and torch.equal(got[0], want[0])
    table[1, 0] = 1 << 20
    got = shared_prefix_attention(q, kp, vp, prefix, 64, table, as_t([64, 64]))
    assert read_status(cuda_device) == -2 and torch.equal(got[0], want[0])


@pytest.mark.gpu
def test_attention_in_a_graph_and_on_another_stream(cuda_device):
    """The call captures; a replay reads the lengths as they are then."""
    from autoindexer_b200 import shared_prefix_attention

    lens = [70, 3, 128]
    q, kp, vp, prefix, table = _cache(3, 1, 8, 2, 128, 64, 200, lens, torch.bfloat16, 5, cuda_device)
    held = torch.tensor(lens, dtype=torch.int32, device=cuda_device)
    want = shared_prefix_attention(q, kp, vp, prefix, 200, table, held)
    short = torch.tensor([12, 1, 65], dtype=torch.int32, device=cuda_device)
    want_short = shared_prefix_attention(q, kp, vp, prefix, 200, table, short)
    s = torch.cuda.Stream(cuda_device)
    s.wait_stream(torch.cuda.current_stream(cuda_device))
    with torch.cuda.stream(s):
        assert torch.equal(shared_prefix_attention(q, kp, vp, prefix, 200, table, held), want)
    torch.cuda.current_stream(cuda_device).wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = shared_prefix_attention(q, kp, vp, prefix, 200, table, held)
    graph.replay()
    assert torch.equal(out, want)
    held.copy_(short)
    graph.replay()
    assert torch.equal(out, want_short)
    graph.reset()


@pytest.mark.gpu
def test_refusals(cuda_device):
    from autoindexer_b200 import paged_append, shared_prefix_attention

    q, kp, vp, prefix, table = _cache(2, 1, 4, 2, 64, 16, 20, [5, 6], torch.bfloat16, 6, cuda_device)
    lens = torch.tensor([5, 6], dtype=torch.int32, device=cuda_device)
    for error, args in [
        (ValueError, (q[:, :3], kp, vp, prefix, 20, table, lens)),
        (ValueError, (q, kp, vp[:, :1], prefix, 20, table, lens)),
        (ValueError, (q, kp, vp, prefix[:1], 20, table, lens)),
        (ValueError, (q, kp, vp, None, 20, table, lens)),
        (ValueError, (q, kp, vp, prefix, -1, table, lens)),
        (ValueError, (q, kp, vp, prefix, 20, table[:1], lens)),
        (ValueError, (q, kp, vp, prefix, 20, table, lens[:1])),
        (ValueError, (q[..., :48], kp[..., :48], vp[..., :48], prefix, 20, table, lens)),
        (TypeError, (q.half(), kp, vp, prefix, 20, table, lens)),
        (TypeError, (q, kp, vp, prefix, 20, table.long(), lens)),
        (TypeError, (q, kp, vp, prefix, 20, table, lens.long())),
        (RuntimeError, (q, kp, vp, prefix, 20, table, lens.cpu())),
        (RuntimeError, (q.cpu(), kp, vp, prefix, 20, table, lens)),
    ]:
        with pytest.raises(error):
            shared_prefix_attention(*args)
    k = torch.randn(2, 2, 1, 64, device=cuda_device, dtype=torch.bfloat16)
    rope, pos = _table(8, 64, cuda_device), torch.zeros(1, dtype=torch.int32, device=cuda_device)
    for error, args, more in [
        (ValueError, (k, k[:, :1], kp, vp, table, lens), {}),
        (ValueError, (k[:, :1], k[:, :1], kp, vp, table, lens), {}),
        (ValueError, (k, k, kp, vp, table[:, :0], lens), {}),
        (ValueError, (k, k, kp, vp, table, lens), {"rope": rope}),
        (ValueError, (k, k, kp, vp, table, lens), {"key_weight": torch.ones(32, device=cuda_device).bfloat16()}),
        (TypeError, (k, k.float(), kp, vp, table, lens), {}),
        (TypeError, (k.float(), k.float(), kp, vp, table, lens), {}),
        (TypeError, (k, k, kp, vp, table, lens), {"new_lens": lens.long()}),
        (RuntimeError, (k, k, kp, vp, table, lens), {"rope": rope, "positions": pos.cpu()}),
        (RuntimeError, (k.cpu(), k.cpu(), kp, vp, table, lens), {}),
    ]:
        with pytest.raises(error):
            paged_append(*args, **more)


def test_c_abi_refusals():
    from autoindexer_b200 import _lib

    L = _lib.lib()

    def attn(**over):
        a = _lib.AiPrefixAttnArgs()
        a.batch, a.seq_len, a.num_q_heads, a.num_kv_heads, a.head_dim = 2, 1, 4, 2, 64
        a.dtype, a.n_pages, a.page_size, a.max_pages, a.prefix_len = _lib.DTYPE_BF16, 4, 16, 2, 0
        for t in ("q", "out", "k_pages", "v_pages"):
            getattr(a, t).ptr = 256
        a.lens = a.page_table = 256
        for n, v in over.items():
            setattr(a, n, v)
        return a

    n = ctypes.c_size_t(0)
    assert L.ai_prefix_attn(None, None) == 1
    for field, value, code in (("batch", 0, 2), ("num_q_heads", 3, 2), ("page_size", 0, 2), ("prefix_len", -1, 2),
                               ("head_dim", 48, 3), ("dtype", 9, 4), ("lens", None, 1), ("prefix_len", 5, 1),
                               ("page_table", None, 1), ("page_table_stride", -1, 5)):
        assert L.ai_prefix_attn(ctypes.byref(attn(**{field: value})), None) == code, field
        assert L.ai_prefix_attn_workspace(ctypes.byref(attn(**{field: value})), ctypes.byref(n)) == code, field
    assert L.ai_prefix_attn_workspace(ctypes.byref(attn()), None) == 1

    def app(**over):
        a = _lib.AiPagedAppendArgs()
        a.batch, a.seq_len, a.num_kv_heads, a.head_dim = 2, 1, 2, 64
        a.dtype = a.weight_dtype = _lib.DTYPE_BF16
        a.n_pages, a.page_size, a.max_pages = 4, 16, 2
        for t in ("k", "v", "k_pages", "v_pages"):
            getattr(a, t).ptr = 256
        a.lens = a.page_table = 256
        for n, v in over.items():
            setattr(a, n, v)
        return a

    assert L.ai_paged_append(None, None) == 1
    for field, value, code in (("batch", 0, 2), ("max_pages", 0, 2), ("head_dim", 256, 3), ("dtype", -1, 4),
                               ("weight_dtype", 1, 4), ("lens", None, 1), ("rope_sin", 256, 1)):
        assert L.ai_paged_append(ctypes.byref(app(**{field: value})), None) == code, field
