"""``paged_attention_4bit`` where parts of one call are far apart in size: what
padding rows hold, query heads and tokens.  Tolerances as in ``test_paged4``."""

import numpy as np
import pytest
import torch

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
