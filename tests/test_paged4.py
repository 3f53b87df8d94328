"""The paged cache in 4 bits: ``paged_append_4bit`` and ``paged_read_4bit``
(codes, scales and values equal to the definition's), ``paged_attention_4bit``
against 64 bits on the values that the cache stands for, and refusals.

Tolerances of the attention: a score is a sum of D products in fp32, good to
2^-19 of ``scale sum |q k|`` (the matrix instructions keep 24 bits of the
largest term of 16, and the offsets they carry are at most nine times the
codes), and changes its weight by that factor; weights and scales are rounded
to fp16 for their products (2^-11 together); the output is rounded once.  So an
output is within ``(2^-19 most + 2^-10) * mag + half a step``, and the
log-sum-exp within ``2^-19 most + 1e-5 (1 + |lse|)``."""

import ctypes

import numpy as np
import pytest
import torch
from torch.autograd import forward_ad

from oracle import learning_oracle as O

DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def pools(n_pages, H, S, D, device, fill=None):
    """Empty pools whose slots hold what no one should read: NaN scales."""
    codes = [torch.full((n_pages, H, S, D // 2), 0xAB, dtype=torch.uint8, device=device) for _ in range(2)]
    scales = [torch.full((n_pages, H, S, D // 32), float("nan"), dtype=torch.float16, device=device) for _ in range(2)]
    return [*codes, *scales]


def tables(held, S, device, extra=2, seed=0, width=None):
    """A page table for sequences that hold so many tokens, in no order."""
    per = [-(-h // S) for h in held]
    g = torch.Generator().manual_seed(seed)
    order = torch.randperm(sum(per) + extra, generator=g).int()
    table = torch.full((len(held), width or max(1, max(per))), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(per):
        table[b, :n] = order[at:at + n]
        at += n
    return table.to(device), sum(per) + extra


def ints(values, device):
    return torch.tensor(values, dtype=torch.int32, device=device)


def heads(B, H, T, D, dtype, seed, device, scale=1.5):
    g = torch.Generator().manual_seed(seed)
    return (scale * torch.randn(B, T, H, D, generator=g)).to(dtype).transpose(1, 2).to(device)


def awkward(x):
    """Rows whose groups are zero, tiny, far apart, equal, or on a half."""
    flat = x.reshape(-1, 32) if x.is_contiguous() else x.contiguous().reshape(-1, 32)
    n = flat.shape[0]
    fin = torch.finfo(x.dtype)
    rows = [torch.zeros(32), torch.full((32,), -3.0), torch.full((32,), 2.5), torch.arange(32) - 15.5,
            (torch.arange(32) - 16) / 2, torch.arange(32) * 1e-7, torch.arange(32) * -1e-4, torch.where(torch.arange(32) % 2 == 0, 4.0, -4.0),
            (torch.arange(32) % 17 - 8) * 0.5 + 0.25, torch.full((32,), min(fin.max, 6e4)), torch.full((32,), -float(fin.max)),
            torch.full((32,), float(fin.tiny)), torch.cat((torch.full((1,), 8.0), torch.arange(31) / 2 - 7.5))]
    for i in range(n):
        if i % 3 == 0:
            flat[i] = rows[i // 3 % len(rows)].to(x.dtype)
    return flat.reshape(x.shape)


def check_held(k, v, cache, table, lens, new, D):
    """The slots hold the definition's codes and scales; returns them visited."""
    S = cache[0].shape[2]
    for x, codes, scales in ((k, cache[0], cache[2]), (v, cache[1], cache[3])):
        want_c, want_s = O.quantize(x.double().cpu().numpy())
        codes, scales = codes.cpu().numpy(), scales.cpu().numpy()
        for b, n in enumerate(new):
            for t in range(n):
                at = lens[b] + t
                page = int(table[b, at // S])
                assert np.array_equal(codes[page, :, at % S], want_c[b, :, t]), (b, t)
                assert np.array_equal(scales[page, :, at % S], want_s[b, :, t], equal_nan=True), (b, t)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,H,T,D,S,lens,new", [
    (1, 1, 1, 32, 16, [0], None),
    (3, 2, 1, 128, 16, [0, 15, 16], None),
    (2, 8, 37, 128, 64, [5, 60], [37, 20]),
    (4, 3, 7, 64, 32, [31, 0, 100, 2], [7, 0, 1, 6]),
    (2, 5, 130, 32, 128, [0, 127], [130, 129]),
    (3, 1, 2100, 64, 16, [0, 3, 40], [2100, 1, 77]),
])
def test_append_and_read(B, H, T, D, S, lens, new, dtype, cuda_device):
    from autoindexer_b200 import paged_append_4bit, paged_read_4bit, read_status

    k, v = (awkward(heads(B, H, T, D, dtype, s, cuda_device)) for s in (1, 2))
    n = new or [T] * B
    table, n_pages = tables([a + b for a, b in zip(lens, n)], S, cuda_device)
    cache = pools(n_pages, H, S, D, cuda_device)
    before = [x.clone() for x in cache]
    args = (*cache, table, ints(lens, cuda_device))
    paged_append_4bit(k, v, *args, new_lens=None if new is None else ints(n, cuda_device))
    assert read_status(cuda_device) == 0
    check_held(k, v, cache, table.cpu(), lens, n, D)
    # Every other slot is as it was.
    touched = torch.zeros(n_pages, S, dtype=torch.bool)
    for b in range(B):
        for t in range(n[b]):
            touched[int(table[b, (lens[b] + t) // S]), (lens[b] + t) % S] = True
    for x, y in zip(cache, before):
        same = (x.view(torch.uint8) == y.view(torch.uint8)).all(-1).all(1).cpu()
        assert bool(same[~touched].all())
    rk, rv = paged_read_4bit(*args, T, dtype, read_lens=None if new is None else ints(n, cuda_device))
    assert rk.shape == k.shape and rk.dtype == dtype
    for x, got in ((k, rk), (v, rv)):
        want = torch.tensor(O.values(*O.quantize(x.double().cpu().numpy()))).float().to(dtype)
        for b in range(B):
            assert torch.equal(got[b, :, :n[b]].cpu(), want[b, :, :n[b]])
            assert not bool(got[b, :, n[b]:].any())
    assert read_status(cuda_device) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_values_that_are_no_numbers(dtype, cuda_device):
    from autoindexer_b200 import paged_append_4bit, paged_read_4bit

    k, v = (heads(1, 2, 5, 128, dtype, s, cuda_device).contiguous() for s in (1, 2))
    k[0, 0, 1, 40], k[0, 1, 2, 0], v[0, 0, 3, 127], v[0, 1, 4] = float("nan"), float("inf"), -float("inf"), float("nan")
    table, n = tables([5], 16, cuda_device)
    cache = pools(n, 2, 16, 128, cuda_device)
    paged_append_4bit(k, v, *cache, table, ints([0], cuda_device))
    check_held(k, v, cache, table.cpu(), [0], [5], 128)
    rk, rv = paged_read_4bit(*cache, table, ints([0], cuda_device), 5, dtype)
    assert rk[0, 0, 1].isnan().sum() == 32 and rk[0, 1, 2].isnan().sum() == 32 and rk.isnan().sum() == 64
    assert rv.isnan().sum() == 32 + 128


@pytest.mark.gpu
def test_codes_are_the_nearest(cuda_device):
    """fp32 values a rounding step beside every half of a code's step."""
    from autoindexer_b200 import paged_append_4bit

    d = np.float16(0.1)  # the scale that a peak of -8 d gives
    half = ((np.arange(16) - 8 + 0.5) * np.float64(d)).astype(np.float32)
    rows = []
    for toward in (-np.inf, np.inf, None):
        r = np.zeros(32, dtype=np.float32)
        r[0] = np.float32(-8 * np.float64(d))
        r[1:17] = half if toward is None else np.nextafter(half, np.float32(toward))
        rows.append(r)
    x = torch.tensor(np.stack(rows * 2)).reshape(1, 2, 3, 32).to(cuda_device)
    table, n = tables([3], 16, cuda_device)
    cache = pools(n, 2, 16, 32, cuda_device)
    paged_append_4bit(x, -x, *cache, table, ints([0], cuda_device))
    check_held(x, -x, cache, table.cpu(), [0], [3], 32)


@pytest.mark.gpu
def test_append_out_of_range(cuda_device):
    from autoindexer_b200 import paged_append_4bit, paged_read_4bit, read_status

    B, H, T, D, S = 6, 2, 3, 64, 16
    k, v = (heads(B, H, T, D, torch.bfloat16, s, cuda_device) for s in (1, 2))
    table = torch.tensor([[0, 1], [2, 9], [-1, 3], [4, 5], [6, 7], [8, 8]], dtype=torch.int32, device=cuda_device)
    lens, new = [0, 14, 15, 31, -2, 2 ** 31 - 1], [4, 3, 3, 3, 3, -1]
    cache = pools(9, H, S, D, cuda_device)
    assert read_status(cuda_device) == 0
    paged_append_4bit(k, v, *cache, table, ints(lens, cuda_device), new_lens=ints(new, cuda_device))
    assert read_status(cuda_device) == -2
    rk, _ = paged_read_4bit(*cache, table, ints(lens, cuda_device), T, torch.bfloat16, read_lens=ints(new, cuda_device))
    assert read_status(cuda_device) == -2
    want = O.values(*O.quantize(k.double().cpu().numpy()))
    held = np.zeros((B, T), dtype=bool)
    held[0], held[1, :2], held[2, 1:], held[3, 0], held[4, 2] = True, True, True, True, True
    for b in range(B):
        for t in range(T):
            assert np.array_equal(rk[b, :, t].double().cpu().numpy(), torch.tensor(want[b, :, t]).bfloat16().double().numpy() * held[b, t])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_append_strides(dtype, cuda_device):
    """Rows off 16-byte boundaries, slices of a joint projection, expanded heads, strided pools."""
    from autoindexer_b200 import paged_append_4bit

    B, H, T, D, S = 2, 3, 5, 64, 16
    table, n = tables([T, T + 9], S, cuda_device)
    lens, new = [0, 9], [T, T]
    joint = heads(B, 2 * H, T, D, dtype, 3, cuda_device)
    odd = torch.zeros(B, H, T, D + 1, dtype=dtype, device=cuda_device)
    odd[..., 1:] = heads(B, H, T, D, dtype, 4, cuda_device)
    step = torch.zeros(B, H, T, 2 * D, dtype=dtype, device=cuda_device)
    step[..., ::2] = heads(B, H, T, D, dtype, 5, cuda_device)
    for k, v in ((joint[:, :H], joint[:, H:]), (odd[..., 1:], joint[:, H:]), (step[..., ::2], odd[..., :D]),
                 (joint[:, :1].expand(B, H, T, D), joint[:1, :H].expand(B, H, T, D))):
        wide = pools(n, 2 * H, S, D, cuda_device)
        cache = [x[:, 1:1 + H] for x in wide]
        paged_append_4bit(k, v, *cache, table, ints(lens, cuda_device), new_lens=ints(new, cuda_device))
        check_held(k, v, cache, table.cpu(), lens, new, D)
        assert bool(wide[2][:, 0].isnan().all()) and bool((wide[0][:, 1 + H:] == 0xAB).all())


# ------------------------------------------------------------------ attention
def filled(B, Hkv, D, S, lens, dtype, seed, device, spread=1.0, width=None):
    """A cache whose sequences hold so many tokens, written by the definition."""
    table, n = tables(lens, S, device, seed=seed, width=width)
    cache = pools(n, Hkv, S, D, device)
    g = torch.Generator().manual_seed(seed)
    for i in range(2):
        for b, m in enumerate(lens):
            x = (spread * torch.randn(Hkv, m, D, generator=g)).to(dtype).double().numpy()
            codes, scales = O.quantize(x)
            at = np.arange(m)
            page = table[b].cpu().numpy()[at // S]
            cache[i][page, :, at % S] = torch.tensor(codes).transpose(0, 1).to(device)
            cache[2 + i][page, :, at % S] = torch.tensor(scales).transpose(0, 1).to(device)
    return cache, table


def dense(cache, table, b, n):
    S = cache[0].shape[2]
    at = np.arange(n)
    page = table[b].cpu().numpy()[at // S]
    out = []
    for i in range(2):
        c, s = cache[i].cpu().numpy()[page, :, at % S], cache[2 + i].cpu().numpy()[page, :, at % S]
        out.append(O.values(c, s).transpose(1, 0, 2))
    return out


def check_attention(q, cache, table, lens, n, scale, out, lse):
    B, Hq, T, D = q.shape
    G = Hq // cache[0].shape[1]
    qn, got = q.double().cpu().numpy(), out.double().cpu().numpy()
    half = torch.finfo(q.dtype).eps / 2
    for b in range(B):
        m = max(0, int(lens[b]))
        k, v = dense(cache, table, b, m)
        seen = [max(0, m - n[b] + t + 1) if t < n[b] else 0 for t in range(T)]
        for h in range(Hq):
            want, wl, mag, most = O.attention(qn[b, h], k[h // G], v[h // G], seen, scale)
            tol = (2.0 ** -19 * most + 2.0 ** -10) * mag + half * np.abs(want) + 2.0 ** -24
            err = np.abs(got[b, :, h] - want)
            assert (err <= tol).all(), (b, h, err.max(), tol[err > tol][:3], want[err > tol][:3])
            if lse is not None:
                gl = lse[b, h].double().cpu().numpy()
                live = wl > -np.inf
                assert np.array_equal(gl == -np.inf, ~live)
                assert (np.abs(gl[live] - wl[live]) <= 2.0 ** -19 * most + 1e-5 * (1 + np.abs(wl[live]))).all(), (b, h)


ATTEND = [
    # B, T, Hq, Hkv, D, S, lens, query_lens
    (1, 1, 1, 1, 32, 16, [1], None),
    (1, 1, 4, 1, 128, 16, [16], None),
    (4, 1, 32, 8, 128, 64, [1, 17, 63, 300], None),
    (3, 1, 16, 2, 64, 32, [0, 33, 128], None),
    (2, 5, 8, 8, 128, 16, [5, 47], [5, 2]),
    (3, 5, 16, 2, 128, 64, [3, 64, 129], [3, 0, 5]),
    (2, 3, 24, 8, 64, 16, [100, 3], None),
    (5, 2, 4, 1, 32, 128, [2, 500, 1, 31, 32], [2, 1, 1, 2, 0]),
    (2, 1, 64, 2, 128, 16, [77, 5], None),
    (1, 70, 8, 2, 128, 32, [200], None),
    (2, 1, 40, 8, 128, 64, [3000, 1025], None),
    (1, 1, 7, 7, 64, 16, [5001], None),
    (130, 1, 4, 2, 64, 16, [(37 * i) % 90 for i in range(130)], None),
]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES[:2])
@pytest.mark.parametrize("B,T,Hq,Hkv,D,S,lens,ql", ATTEND)
def test_attention(B, T, Hq, Hkv, D, S, lens, ql, dtype, cuda_device):
    from autoindexer_b200 import paged_attention_4bit, read_status

    cache, table = filled(B, Hkv, D, S, lens, dtype, B + T, cuda_device)
    q = heads(B, Hq, T, D, dtype, 9, cuda_device)
    n = ql or [T] * B
    args = (q, *cache, table, ints(lens, cuda_device))
    more = dict(query_lens=None if ql is None else ints(ql, cuda_device), return_lse=True)
    out, lse = paged_attention_4bit(*args, **more)
    assert out.shape == (B, T, Hq, D) and out.dtype == dtype and lse.shape == (B, Hq, T)
    assert read_status(cuda_device) == 0
    check_attention(q, cache, table, lens, n, D ** -0.5, out, lse)
    again, l2 = paged_attention_4bit(*args, **more)
    assert torch.equal(out, again) and torch.equal(lse, l2)
    assert torch.equal(paged_attention_4bit(*args, query_lens=more["query_lens"]), out)
    for scaling in (0.0, -0.3, 1.7):
        got = paged_attention_4bit(*args, scaling=scaling, query_lens=more["query_lens"])
        check_attention(q, cache, table, lens, n, scaling, got, None)


@pytest.mark.gpu
def test_attention_over_a_long_list(cuda_device):
    from autoindexer_b200 import paged_attention_4bit

    lens = [40000, 1, 9000]
    cache, table = filled(3, 2, 128, 64, lens, torch.bfloat16, 3, cuda_device)
    q = heads(3, 8, 1, 128, torch.bfloat16, 4, cuda_device)
    out, lse = paged_attention_4bit(q, *cache, table, ints(lens, cuda_device), return_lse=True)
    check_attention(q, cache, table, lens, [1] * 3, 128 ** -0.5, out, lse)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES[:2])
def test_attention_of_far_values(dtype, cuda_device):
    """Queries and values whose sizes differ by many powers of two: tiny and
    large queries, values that grow along the list, a sure key among many."""
    from autoindexer_b200 import paged_attention_4bit

    B, Hkv, D, S, lens = 4, 2, 64, 16, [700, 700, 700, 700]
    cache, table = filled(B, Hkv, D, S, lens, torch.float32, 5, cuda_device)
    q = heads(B, 4, 2, D, dtype, 6, cuda_device).contiguous()
    q[0] *= 2.0 ** -12
    q[1] *= 2.0 ** 6
    q[2, :, :, ::2] *= 2.0 ** -10
    pages = table.cpu().numpy()
    for j in range(700):  # values of sequence 2 grow, those of sequence 3 shrink, by 2^30 in all
        page, slot = int(pages[2, j // S]), j % S
        cache[3][page, :, slot] *= 2.0 ** (-12 + 24 * j / 700)
        page = int(pages[3, j // S])
        cache[3][page, :, slot] *= 2.0 ** (12 - 24 * j / 700)
    out, lse = paged_attention_4bit(q, *cache, table, ints(lens, cuda_device), return_lse=True)
    check_attention(q, cache, table, lens, [2] * B, D ** -0.5, out, lse)


@pytest.mark.gpu
def test_small_weights_beside_a_large_one(cuda_device):
    """One key with weight 1 and 60,000 of 2^-13 each: their sum (7.3) is not lost."""
    from autoindexer_b200 import paged_attention_4bit

    D, S, n = 32, 64, 60001
    k, v = np.zeros((1, n, D)), np.ones((1, n, D))
    k[0, :, 0], v[0, :, 5] = -8, 3.0
    k[0, 100, 0], v[0, 100, 5] = 8.0, -3.0
    table, pages = tables([n], S, cuda_device)
    cache = pools(pages, 1, S, D, cuda_device)
    at = np.arange(n)
    page = table[0].cpu().numpy()[at // S]
    for i, x in enumerate((k, v)):
        codes, scales = O.quantize(x)
        cache[i][page, :, at % S] = torch.tensor(codes).transpose(0, 1).to(cuda_device)
        cache[2 + i][page, :, at % S] = torch.tensor(scales).transpose(0, 1).to(cuda_device)
    q = torch.zeros(1, 1, 1, D, dtype=torch.float16, device=cuda_device)
    q[..., 0] = 13 * np.log(2) / 15
    out, lse = paged_attention_4bit(q, *cache, table, ints([n], cuda_device), scaling=1.0, return_lse=True)
    check_attention(q, cache, table, [n], [1], 1.0, out, lse)


@pytest.mark.gpu
def test_attention_where_nothing_is_a_number(cuda_device):
    """A NaN that a row sees makes it NaN (of a value: in its 32 dims); one that
    it does not see changes nothing."""
    from autoindexer_b200 import paged_attention_4bit

    lens, D, S = [40, 40, 40, 40], 64, 16
    cache, table = filled(4, 2, D, S, lens, torch.bfloat16, 8, cuda_device)
    q = heads(4, 4, 2, D, torch.bfloat16, 2, cuda_device)
    args = (q, *cache, table, ints(lens, cuda_device))
    want = paged_attention_4bit(*args)
    nan, t = float("nan"), table.cpu().numpy()
    cache[2][int(t[0, 1]), 0, 3] = nan           # a key of KV head 0
    cache[3][int(t[1, 0]), 1, 5, 1] = nan        # dims 32 to 63 of a value of KV head 1
    cache[2][int(t[2, 2]), :, 7] = nan           # the last key: seen by the second token alone
    cache[3][int(t[3, 2]), :, 7] = float("inf")  # likewise a value
    got, lse = paged_attention_4bit(*args, return_lse=True)
    bad = got.isnan()
    assert bad[0, :, :2].all() and not bad[0, :, 2:].any()
    assert bad[1, :, 2:, 32:].all() and not bad[1, :, 2:, :32].any() and not bad[1, :, :2].any()
    assert bad[2, 1].all() and not bad[2, 0].any()
    assert not bad[3, 0].any() and not got[3, 1].isfinite().any()
    for b, t_, h, d in ((0, slice(0, 2), slice(2, 4), slice(0, D)), (1, slice(0, 2), slice(0, 4), slice(0, 32)),
                        (2, 0, slice(0, 4), slice(0, D)), (3, 0, slice(0, 4), slice(0, D))):
        assert torch.equal(got[b, t_, h, d], want[b, t_, h, d])
    q = q.clone()
    q[0, 2, 0, 5], q[1, 1, 1, 0] = nan, float("inf")
    cache, table = filled(4, 2, D, S, lens, torch.bfloat16, 8, cuda_device)
    got = paged_attention_4bit(q, *cache, table, ints(lens, cuda_device))
    bad = got.isnan()
    assert bad[0, 0, 2].all() and bad[1, 1, 1].all() and bad.sum() == 2 * D


@pytest.mark.gpu
def test_attention_strides_and_shared_pages(cuda_device):
    """Queries of any strides and places, pools that are part of wider ones,
    sequences that list the same pages, a page table wider than needed."""
    from autoindexer_b200 import paged_attention_4bit

    B, Hq, Hkv, T, D, S, lens = 3, 8, 2, 2, 64, 16, [50, 50, 50]
    cache, table = filled(B, Hkv, D, S, lens, torch.float16, 8, cuda_device, width=9)
    table[1] = table[0]
    table[2, :3] = table[0, :3]
    q = heads(B, Hq, T, D, torch.float16, 2, cuda_device)
    n = ints(lens, cuda_device)
    want = paged_attention_4bit(q, *cache, table, n)
    check_attention(q, cache, table, lens, [T] * B, D ** -0.5, want, None)
    odd = torch.zeros(B, Hq, T, D + 3, dtype=torch.float16, device=cuda_device)
    odd[..., 3:] = q
    step = torch.zeros(B, Hq, T, 2 * D, dtype=torch.float16, device=cuda_device)
    step[..., ::2] = q
    for other in (q.contiguous(), odd[..., 3:], step[..., ::2]):
        assert torch.equal(paged_attention_4bit(other, *cache, table, n), want)
    wide = pools(cache[0].shape[0], 5, S, D, cuda_device)
    part = [x[:, 2:4] for x in wide]
    for x, y in zip(part, cache):
        x.copy_(y)
    assert torch.equal(paged_attention_4bit(q, *part, table, n), want)
    seen = torch.zeros(B, 20, dtype=torch.int32, device=cuda_device)
    seen[:, 4:13] = table
    assert torch.equal(paged_attention_4bit(q, *cache, seen[:, 4:13], n), want)
    same = q[:1].expand(B, Hq, T, D)
    assert torch.equal(paged_attention_4bit(same, *cache, table, n)[0], paged_attention_4bit(same, *cache, table, n)[1])


@pytest.mark.gpu
def test_attention_out_of_range(cuda_device):
    """Lengths and pages out of range are clamped and reported."""
    from autoindexer_b200 import paged_attention_4bit, read_status

    lens = [40, 40, 40]
    cache, table = filled(3, 2, 64, 16, lens, torch.bfloat16, 8, cuda_device)
    q = heads(3, 4, 2, 64, torch.bfloat16, 2, cuda_device)
    for held, n, as_held, as_n in (([40, -3, 40], [2, 2, 2], [40, 0, 40], [2, 2, 2]), ([48, 40, 2 ** 31 - 1], [2] * 3, [48, 40, 48], [2] * 3),
                                   ([40, 40, 1], [3, -1, 2], [40, 40, 1], [2, 0, 2])):
        cache[2].nan_to_num_(0.25)
        cache[3].nan_to_num_(0.25)
        got = paged_attention_4bit(q, *cache, table, ints(held, cuda_device), query_lens=ints(n, cuda_device))
        assert read_status(cuda_device) == (-2 if (held, n) != (as_held, as_n) else 0)
        check_attention(q, cache, table, as_held, as_n, 64 ** -0.5, got, None)
    wrong = table.clone()
    wrong[1, 1], wrong[2, 2] = cache[0].shape[0], -1
    got = paged_attention_4bit(q, *cache, wrong, ints(lens, cuda_device))
    assert read_status(cuda_device) == -2
    wrong[1, 1], wrong[2, 2] = 0, 0
    check_attention(q, cache, wrong, lens, [2] * 3, 64 ** -0.5, got, None)


@pytest.mark.gpu
def test_offsets_past_31_bits(cuda_device):
    """Pages whose bytes lie more than 2^32 behind the pool's start."""
    from autoindexer_b200 import paged_append_4bit, paged_attention_4bit

    H, S, D, far = 2, 16, 128, 2 ** 32 + 4096
    base = [torch.empty(far + 2 ** 16, dtype=torch.uint8, device=cuda_device) for _ in range(2)]
    codes = [x.as_strided((2, H, S, D // 2), (far, S * D // 2, D // 2, 1)) for x in base]
    sbase = [x.view(torch.float16) for x in base]
    scales = [x.as_strided((2, H, S, D // 32), (far // 2, S * D // 32, D // 32, 1), 8192) for x in sbase]
    cache = [*codes, *scales]
    table = torch.tensor([[1, 0]], dtype=torch.int32, device=cuda_device)
    k, v = (heads(1, H, 20, D, torch.bfloat16, s, cuda_device) for s in (1, 2))
    paged_append_4bit(k, v, *cache, table, ints([0], cuda_device))
    check_held(k, v, cache, table.cpu(), [0], [20], D)
    q = heads(1, 4, 1, D, torch.bfloat16, 3, cuda_device)
    out, lse = paged_attention_4bit(q, *cache, table, ints([20], cuda_device), return_lse=True)
    check_attention(q, cache, table, [20], [1], D ** -0.5, out, lse)


@pytest.mark.gpu
@pytest.mark.parametrize("B,T,n0", [(2, 1, 20), (40, 3, 600)])
def test_captured_graph_and_another_stream(B, T, n0, cuda_device):
    """Append, read and attention of a step in one graph: a replay reads lengths,
    tables and values as they are then; two graphs run one after the other."""
    from autoindexer_b200 import paged_append_4bit, paged_attention_4bit, paged_read_4bit, read_status

    Hq, Hkv, D, S = 8, 2, 128, 16
    lens = [(n0 + 7 * i) % n0 for i in range(B)]
    cache, table = filled(B, Hkv, D, S, [n0 + 2 * T] * B, torch.bfloat16, 4, cuda_device)
    before, after, n = ints(lens, cuda_device), ints([x + T for x in lens], cuda_device), ints([T] * B, cuda_device)
    k, v, q = (heads(B, H, T, D, torch.bfloat16, s, cuda_device) for H, s in ((Hkv, 1), (Hkv, 2), (Hq, 3)))

    def step():
        paged_append_4bit(k, v, *cache, table, before, new_lens=n)
        out = paged_attention_4bit(q, *cache, table, after, query_lens=n, return_lse=True)
        return [*out, *paged_read_4bit(*cache, table, before, T, torch.bfloat16, read_lens=n)]

    step()
    torch.cuda.synchronize(cuda_device)
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = step()
        graphs.append((graph, got))
    for turn in range(3):
        for graph, got in graphs:
            graph.replay()
        want = step()
        side = torch.cuda.Stream(cuda_device)
        side.wait_stream(torch.cuda.current_stream(cuda_device))
        with torch.cuda.stream(side):
            third = step()
        torch.cuda.synchronize(cuda_device)
        for _, got in graphs:
            assert all(torch.equal(a, b) and torch.equal(a, c) for a, b, c in zip(got, want, third))
        before.add_(T - (turn == 0))
        after.add_(T - (turn == 0))
        q.mul_(-1)
    assert read_status(cuda_device) == 0
    for graph, _ in graphs:
        graph.reset()


@pytest.mark.gpu
def test_attention_refuses_gradients(cuda_device):
    from autoindexer_b200 import paged_attention_4bit

    cache, table = filled(2, 2, 64, 16, [9, 20], torch.bfloat16, 8, cuda_device)
    q, n = heads(2, 4, 1, 64, torch.bfloat16, 2, cuda_device), ints([9, 20], cuda_device)
    want = paged_attention_4bit(q, *cache, table, n)
    got = paged_attention_4bit(q.clone().requires_grad_(), *cache, table, n)
    assert torch.equal(got, want)
    with pytest.raises(RuntimeError, match="paged_attention_4bit has no backward"):
        got.sum().backward()
    with forward_ad.dual_level(), pytest.raises(RuntimeError, match="forward"):
        paged_attention_4bit(forward_ad.make_dual(q, torch.ones_like(q)), *cache, table, n)


@pytest.mark.gpu
def test_refusals(cuda_device):
    from autoindexer_b200 import paged_append_4bit, paged_attention_4bit, paged_read_4bit

    cache, table = filled(2, 2, 64, 16, [9, 20], torch.bfloat16, 8, cuda_device)
    kc, vc, ks, vs = cache
    q, n = heads(2, 4, 1, 64, torch.bfloat16, 2, cuda_device), ints([9, 20], cuda_device)
    k = heads(2, 2, 1, 64, torch.bfloat16, 2, cuda_device)
    base = torch.zeros(kc.numel() + 64, dtype=torch.uint8, device=cuda_device)
    off = base[8:8 + kc.numel()].view(kc.shape)
    thin = torch.zeros(*kc.shape[:3], 40, dtype=torch.uint8, device=cuda_device)[..., :32]
    pool_refusals = [
        (ValueError, (kc[0], vc, ks, vs)),
        (ValueError, (kc, vc[:1], ks, vs)),
        (ValueError, (kc[:, :, :8], vc[:, :, :8], ks[:, :, :8], vs[:, :, :8])),
        (ValueError, (*(torch.cat((x, x, x), 2) for x in cache),)),
        (ValueError, (kc, vc, ks[..., :1], vs)),
        (ValueError, (off, vc, ks, vs)),
        (ValueError, (thin, vc, ks, vs)),
        (ValueError, (kc[:0], vc[:0], ks[:0], vs[:0])),
        (TypeError, (kc.int(), vc, ks, vs)),
        (TypeError, (kc, vc, ks, vs.float())),
        (RuntimeError, (kc, vc, ks, vs.cpu())),
    ]
    for error, bad in pool_refusals:
        with pytest.raises(error):
            paged_attention_4bit(q, *bad, table, n)
        with pytest.raises(error):
            paged_append_4bit(k, k, *bad, table, n)
        with pytest.raises(error):
            paged_read_4bit(*bad, table, n, 1, torch.bfloat16)
    for error, args in [
        (ValueError, (q[0], *cache, table, n)), (ValueError, (q[:, :3], *cache, table, n)), (ValueError, (q[..., :32], *cache, table, n)),
        (ValueError, (q, *cache, table[0], n)), (ValueError, (q, *cache, table[:, :0], n)), (ValueError, (q, *cache, table, n[:1])),
        (ValueError, (q.expand(2, 4, 1, 64)[:, :, :0], *cache, table, n)), (TypeError, (q.float(), *cache, table, n)),
        (TypeError, (q, *cache, table.long(), n)), (TypeError, (q, *cache, table, n.long())), (RuntimeError, (q, *cache, table, n.cpu())),
        (ValueError, (q[:1].expand(1025, 4, 1, 64), *cache, table[:1].expand(1025, -1), n[:1].expand(1025))),
    ]:
        with pytest.raises(error):
            paged_attention_4bit(*args)
    for error, args in [
        (ValueError, (k[0], k[0], *cache, table, n)), (ValueError, (k, k[:1], *cache, table, n)), (ValueError, (k[:, :1], k[:, :1], *cache, table, n)),
        (ValueError, (k[..., :16], k[..., :16], *cache, table, n)), (TypeError, (k, k.half(), *cache, table, n)),
        (TypeError, (k.double(), k.double(), *cache, table, n)), (RuntimeError, (k, k.cpu(), *cache, table, n)),
        (ValueError, (k, k, *cache, table, n, n[:1])),
    ]:
        with pytest.raises(error):
            paged_append_4bit(*args)
    for error, args in [(ValueError, (*cache, table[0], n, 1, torch.bfloat16)), (ValueError, (*cache, table, n, 0, torch.bfloat16)),
                        (TypeError, (*cache, table, n, 1, torch.float64)), (ValueError, (*cache, table, n, 1, torch.bfloat16, n[:1]))]:
        with pytest.raises(error):
            paged_read_4bit(*args)


def test_cpu_tensors_are_refused():
    from autoindexer_b200 import paged_append_4bit, paged_attention_4bit, paged_read_4bit

    cache, table = filled(2, 2, 64, 16, [9, 20], torch.bfloat16, 8, "cpu")
    q, n = heads(2, 4, 1, 64, torch.bfloat16, 2, "cpu"), ints([9, 20], "cpu")
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        paged_attention_4bit(q, *cache, table, n)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        paged_append_4bit(q[:, :2], q[:, :2], *cache, table, n)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        paged_read_4bit(*cache, table, n, 1, torch.bfloat16)


def test_c_abi_refusals():
    from autoindexer_b200 import _lib

    L = _lib.lib()

    def fill(p, D):
        for name, unit in (("k_codes", D // 2), ("v_codes", D // 2), ("k_scales", D // 32), ("v_scales", D // 32)):
            t = getattr(p, name)
            t.ptr, t.stride_b, t.stride_h, t.stride_t = 256, 32 * unit, 16 * unit, unit
        p.n_pages, p.page_size, p.page_table, p.page_table_stride, p.max_pages = 4, 16, 256, 2, 2

    def put(a, **over):
        for n, v in over.items():
            at = a
            *path, last = n.split("__")
            for x in path:
                at = getattr(at, x)
            setattr(at, last, v)
        return ctypes.byref(a)

    def paged(**over):
        a = _lib.AiPaged4Args()
        a.batch, a.seq_len, a.num_kv_heads, a.head_dim, a.dtype = 2, 3, 2, 64, _lib.DTYPE_BF16
        a.k.ptr = a.v.ptr = a.lens = 256
        fill(a.pool, 64)
        return put(a, **over)

    def attn(**over):
        a = _lib.AiPagedAttn4Args()
        a.batch, a.seq_len, a.num_q_heads, a.num_kv_heads, a.head_dim, a.dtype, a.scale = 2, 1, 4, 2, 64, _lib.DTYPE_BF16, 0.1
        a.q.ptr = a.out.ptr = a.lens = 256
        fill(a.pool, 64)
        return put(a, **over)

    pool = (("pool__n_pages", 0, 2), ("pool__page_size", 24, 2), ("pool__page_size", 8, 2), ("pool__max_pages", 0, 2),
            ("pool__page_table", None, 1), ("pool__page_table_stride", -1, 5), ("pool__k_codes__ptr", None, 1),
            ("pool__v_codes__ptr", 264, 6), ("pool__v_scales__ptr", 258, 6), ("pool__k_codes__stride_t", 24, 5),
            ("pool__k_scales__stride_h", 3, 5), ("pool__v_codes__stride_b", -16, 5), ("lens", None, 1))
    n = ctypes.c_size_t(0)
    for fn in (L.ai_paged_append_4bit, L.ai_paged_read_4bit):
        assert fn(None, None) == 1
        for field, value, code in pool + (("batch", 0, 2), ("seq_len", 0, 2), ("num_kv_heads", 0, 2), ("head_dim", 96, 3),
                                          ("dtype", 7, 4), ("k__ptr", None, 1), ("v__stride_t", -1, 5), ("seq_len", 2 ** 31 - 1, 2)):
            assert fn(paged(**{field: value}), None) == code, field
    assert L.ai_paged_attn_4bit(None, None) == 1 and L.ai_paged_attn_4bit_workspace(None, ctypes.byref(n)) == 1
    assert L.ai_paged_attn_4bit_workspace(attn(), None) == 1
    for field, value, code in pool + (("batch", 1025, 2), ("seq_len", 0, 2), ("num_q_heads", 5, 2), ("head_dim", 16, 3),
                                      ("dtype", _lib.DTYPE_F32, 4), ("q__ptr", None, 1), ("out__stride_h", -1, 5)):
        assert L.ai_paged_attn_4bit(attn(**{field: value}), None) == code, field
        assert L.ai_paged_attn_4bit_workspace(attn(**{field: value}), ctypes.byref(n)) == code, field
    assert L.ai_paged_attn_4bit_workspace(attn(), ctypes.byref(n)) == 0


@pytest.mark.parametrize("D", [32, 64, 128])
def test_oracle_format(D):
    """The documented place of each dim, and a code's error of half a step at most."""
    rng = np.random.default_rng(0)
    x = rng.normal(size=(3, D))
    codes, scales = O.quantize(x)
    assert codes.shape == (3, D // 2) and scales.shape == (3, D // 32) and scales.dtype == np.float16
    for d in range(D):
        c, g, j = d // 32, d % 32 // 4, d % 4
        byte = int(codes[1, g * D // 16 + 2 * c + j // 2])
        assert ((byte >> (4 * (j % 2))) & 15) - 8 == np.clip(np.rint(x[1, d] / np.float64(scales[1, c])), -8, 7)
    y = O.values(codes, scales)
    step = np.abs(scales.astype(np.float64))[:, np.arange(D) // 32]
    inside = np.abs(x) <= 7.5 * step
    assert (np.abs(x - y)[inside] <= step[inside] / 2 + 1e-12).all()
