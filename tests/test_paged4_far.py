"""``paged_attention_4bit`` where parts of one call are far apart in size: what
padding rows hold, query heads and tokens, groups of value dims, a key of large
values that no one attends to.

Tolerances as in ``test_paged4``; beside them a product of a weight and a value's
scale is rounded to an fp16 number that may be subnormal: the largest weight is
held as 2^7 at least, the group's largest scale as a quarter at least, so half a step
(2^-25) is 2^-30 of the largest scale, and a code is at most 8: 2^-27 of the group's
largest scale for a key that has the weight, and for the mean over equal ones."""

import numpy as np
import pytest
import torch

from oracle import learning_oracle as O
from test_paged4 import check_attention, dense, filled, heads, ints

HALVES = [torch.bfloat16, torch.float16]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("Hq,Hkv,D,lens,ql,T", [
    (32, 8, 128, [70, 33, 200], [1, 0, 3], 5),
    (4, 4, 64, [40, 40], [1, 2], 3),
    (8, 2, 32, [90, 300], [20, 70], 70),
    (16, 1, 128, [9, 1], [1, 1], 2),
])
def test_padding_rows_may_hold_anything(Hq, Hkv, D, lens, ql, T, dtype, cuda_device):
    from autoindexer_b200 import paged_attention_4bit, read_status

    B = len(lens)
    cache, table = filled(B, Hkv, D, 16, lens, dtype, 3, cuda_device)
    q = heads(B, Hq, T, D, dtype, 4, cuda_device).contiguous()
    padding = (torch.arange(T) >= torch.tensor(ql)[:, None])[:, None, :, None].to(cuda_device)
    args = (*cache, table, ints(lens, cuda_device))
    more = dict(query_lens=ints(ql, cuda_device), return_lse=True)
    want, lse = paged_attention_4bit(q.masked_fill(padding, 0.0), *args, **more)
    check_attention(q, cache, table, lens, ql, D ** -0.5, want, lse)
    top = torch.finfo(dtype).max
    for value in (top, -top, min(top, 1e30), 4096.0, float("nan"), float("inf"), -float("inf")):
        got, l2 = paged_attention_4bit(q.masked_fill(padding, value), *args, **more)
        assert torch.equal(got, want) and torch.equal(l2, lse), value
    assert read_status(cuda_device) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,far", [(torch.bfloat16, 2.0 ** 30), (torch.bfloat16, 2.0 ** 60), (torch.float16, 2.0 ** 13)])
@pytest.mark.parametrize("T,D", [(1, 128), (3, 64), (5, 128)])
def test_heads_far_apart(T, D, dtype, far, cuda_device):
    """Large queries in some heads of a KV head leave the others' scores as they are."""
    from autoindexer_b200 import paged_attention_4bit

    lens = [65, 300]
    cache, table = filled(2, 2, D, 32, lens, torch.float32, 5, cuda_device)
    q = heads(2, 8, T, D, dtype, 6, cuda_device).contiguous()
    scaling = None
    if dtype is torch.float16:  # (2^13 times these still fit the type)
        q *= 2.0 ** -3
        scaling = 0.7
    alone = q.clone()
    q[:, [0, 3, 5]] *= far
    args = (*cache, table, ints(lens, cuda_device))
    out, lse = paged_attention_4bit(q, *args, scaling=scaling, return_lse=True)
    same, l2 = paged_attention_4bit(alone, *args, scaling=scaling, return_lse=True)
    check_attention(alone, cache, table, lens, [T] * 2, scaling or D ** -0.5, same, l2)
    for h in (1, 2, 4, 6, 7):
        assert torch.equal(out[:, :, h], same[:, :, h]) and torch.equal(lse[:, h], l2[:, h])


@pytest.mark.gpu
def test_tokens_far_apart(cuda_device):
    """A token's large query leaves the other tokens as they are."""
    from autoindexer_b200 import paged_attention_4bit

    cache, table = filled(2, 2, 128, 16, [77, 310], torch.float32, 5, cuda_device)
    q = heads(2, 8, 5, 128, torch.bfloat16, 6, cuda_device).contiguous()
    args = (*cache, table, ints([77, 310], cuda_device))
    want, lse = paged_attention_4bit(q, *args, return_lse=True)
    check_attention(q, cache, table, [77, 310], [5, 5], 128 ** -0.5, want, lse)
    q[:, :, 2] *= 2.0 ** 40
    got, l2 = paged_attention_4bit(q, *args, return_lse=True)
    for t in (0, 1, 3, 4):
        assert torch.equal(got[:, t], want[:, t]) and torch.equal(l2[:, :, t], lse[:, :, t])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,of_q,of_k,scaling", [
    (torch.bfloat16, 2.0 ** 20, 1.0, None), (torch.bfloat16, 2.0 ** 30, 1.0, None), (torch.bfloat16, 2.0 ** 60, 1.0, -0.1),
    (torch.bfloat16, 2.0 ** 100, 1.0, None), (torch.float16, 2.0 ** 12, 2.0 ** 12, 8.0), (torch.float16, 2.0 ** 10, 2.0 ** 10, 1.0)])
@pytest.mark.parametrize("T,D", [(1, 128), (3, 64), (5, 128)])
def test_large_scores(T, D, dtype, of_q, of_k, scaling, cuda_device):
    """Scores of 2^20 and more, whose steps in fp32 are many powers of e: a row is the
    value of its best key where that is best by more than a score's rounding."""
    from autoindexer_b200 import paged_attention_4bit, read_status

    lens = [65, 1300]
    cache, table = filled(2, 2, D, 32, lens, torch.float32, 5, cuda_device)
    cache[2].mul_(of_k)
    q = (heads(2, 8, T, D, dtype, 6, cuda_device) * of_q).contiguous()
    out, lse = paged_attention_4bit(q, *cache, table, ints(lens, cuda_device), scaling=scaling, return_lse=True)
    assert read_status(cuda_device) == 0
    scale = scaling or D ** -0.5
    qn, got, l = q.double().cpu().numpy(), out.double().cpu().numpy(), lse.double().cpu().numpy()
    sure = 0
    for b in range(2):
        k, v = dense(cache, table, b, lens[b])
        for h in range(8):
            for t in range(T):
                n = lens[b] - T + t + 1
                s = k[h // 4, :n] @ qn[b, h, t] * scale
                most = (np.abs(k[h // 4, :n]) @ np.abs(qn[b, h, t])).max() * abs(scale)
                best, second = np.sort(s)[::-1][:2]
                assert abs(l[b, h, t] - best) <= 2.0 ** -19 * most + 1e-5 * (1 + abs(best)) + np.log(n)
                assert (np.abs(got[b, t, h]) <= np.abs(v[h // 4, :n]).max(0) * (1 + 2.0 ** -8)).all()
                if best - second > 2.0 ** -18 * most + 40:
                    sure += 1
                    want = v[h // 4, int(np.argmax(s))]
                    tol = (2.0 ** -10 + torch.finfo(dtype).eps / 2) * np.abs(want) + 2.0 ** -24
                    assert (np.abs(got[b, t, h] - want) <= tol).all(), (b, h, t)
    assert sure >= 8 * T


def check_dims(q, cache, table, lens, out, extra):
    """``check_attention`` with, per dim, ``extra`` of the group's largest scale on top."""
    B, Hq, T, D = q.shape
    G = Hq // cache[0].shape[1]
    qn, got, half = q.double().cpu().numpy(), out.double().cpu().numpy(), torch.finfo(q.dtype).eps / 2
    for b in range(B):
        k, v = dense(cache, table, b, lens[b])
        at = np.arange(lens[b])
        S = cache[0].shape[2]
        scales = np.abs(cache[3].double().cpu().numpy()[table[b].cpu().numpy()[at // S], :, at % S])  # (n, Hkv, groups)
        most_scale = np.repeat(scales.max(0), 32, axis=-1)
        for h in range(Hq):
            want, _, mag, most = O.attention(qn[b, h], k[h // G], v[h // G], [lens[b] - T + t + 1 for t in range(T)], D ** -0.5)
            tol = (2.0 ** -19 * most + 2.0 ** -10) * mag + half * np.abs(want) + 2.0 ** -24 * (1 if q.dtype is torch.float16 else 0)
            tol = tol + extra * most_scale[h // G]
            err = np.abs(got[b, :, h] - want)
            assert (err <= tol).all(), (b, h, err.max(), tol[err > tol][:3], want[err > tol][:3])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("T,D,at,up", [(1, 128, 2, 16), (1, 64, 0, 25), (5, 128, 3, 25), (3, 64, 1, 20), (2, 128, 0, 16)])
def test_groups_of_dims_far_apart(T, D, at, up, dtype, cuda_device):
    """32 dims of large values leave the others' digits as they are."""
    from autoindexer_b200 import paged_attention_4bit

    lens = [200, 31]
    cache, table = filled(2, 2, D, 32, lens, torch.float32, 5, cuda_device, spread=2.0 ** -9)
    q = heads(2, 8, T, D, dtype, 6, cuda_device).contiguous()
    if dtype is torch.float16:
        q[..., :] *= 0.25
    cache[2].mul_(2.0 ** 9)  # (keys as usual)
    cache[3][..., at] *= 2.0 ** up
    out = paged_attention_4bit(q, *cache, table, ints(lens, cuda_device))
    if dtype is torch.float16:
        # (the large dims do not fit the output's type; the others are compared)
        keep = torch.ones(D, dtype=torch.bool)
        keep[32 * at:32 * at + 32] = out[..., 32 * at:32 * at + 32].isfinite().all().item()
        if not bool(keep.all()):
            other = cache[3].clone()
            other[..., at] = cache[3][..., at] * 2.0 ** -up
            want = paged_attention_4bit(q, *cache[:3], other, table, ints(lens, cuda_device))
            assert torch.equal(out[..., keep.to(cuda_device)], want[..., keep.to(cuda_device)])
            return
    check_dims(q, cache, table, lens, out, 2.0 ** -27)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("where", [0, 100, 299])
@pytest.mark.parametrize("T", [1, 4])
def test_a_large_value_of_no_weight(T, where, dtype, cuda_device):
    """A key whose values are 2^20 times the others', and whose weight is below
    2^-80, beside one that has almost all of the weight."""
    from autoindexer_b200 import paged_attention_4bit

    D, S, lens = 64, 16, [310]
    cache, table = filled(1, 1, D, S, lens, torch.float32, 7, cuda_device, spread=2.0 ** -5)
    pages = table[0].cpu().numpy()

    def key(j, row):
        codes, scale = O.quantize(row[None])
        cache[0][int(pages[j // S]), 0, j % S] = torch.tensor(codes[0]).to(cuda_device)
        cache[2][int(pages[j // S]), 0, j % S] = torch.tensor(scale[0]).to(cuda_device)

    q = heads(1, 4, T, D, dtype, 8, cuda_device).contiguous()
    q[..., 0] = 16.0
    key(50, np.eye(D)[0] * 20.0)
    key(where, np.eye(D)[0] * -60.0)
    cache[3][int(pages[where // S]), 0, where % S] *= 2.0 ** 20
    out = paged_attention_4bit(q, *cache, table, ints(lens, cuda_device))
    check_dims(q, cache, table, lens, out, 2.0 ** -27)
