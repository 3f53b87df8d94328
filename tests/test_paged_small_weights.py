"""``shared_prefix_attention`` where one key takes nearly all the weight and
very many others in the same stretch share the rest.

Tolerance of the log-sum: as in ``test_paged.py`` (exponentials are added up
in blocks first, the running sum takes one number a block)."""

import math

import pytest
import torch


def _lists(B, T, Hq, n, gap, v0, v1, dtype, device):
    """Sequences that list the same n keys, as many as there are workers, so
    that a list is one worker's: key 0 with score 0 and value ``v0(d)``, the
    others with score ``-gap`` and value ``v1(d)``.  Returns the call's
    arguments and the gap that the type holds."""
    D, S = 64, 128
    pages = n // S
    kp = torch.zeros(pages, 1, S, D, dtype=dtype, device=device)
    kp[..., 0] = -gap
    kp[0, 0, 0, 0] = 0.0
    vp = torch.empty(pages, 1, S, D)
    vp[:] = v1(torch.arange(D))
    vp[0, 0, 0] = v0(torch.arange(D))
    q = torch.zeros(B, Hq, T, D, dtype=dtype, device=device)
    q[..., 0] = 1
    table = torch.arange(pages, dtype=torch.int32, device=device).expand(B, pages).contiguous()
    lens = torch.full((B,), n, dtype=torch.int32, device=device)
    return (q, kp, vp.to(dtype).to(device), None, 0, table, lens), float(torch.tensor(gap, dtype=dtype))


SHAPES = [
    # B, T, Hq
    (888, 1, 1),    # streaming kernel, up to 8 rows a warp
    (888, 1, 16),   # streaming kernel, 16 rows
    (296, 5, 16),   # tile kernel, 80 rows
    (148, 9, 16),   # tile kernel, 144 rows
]
GAPS = [16.234375, 17.53125, 12.0]  # weights beside the largest: 2^-23.4, 2^-25.3, 2^-17.3


def _eps(D, gap):
    return 2 * 4 * D * 2.0 ** -24 * gap + 2.0 ** -16


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("gap", GAPS)
@pytest.mark.parametrize("B,T,Hq", SHAPES)
def test_log_sum_of_many_small_weights(B, T, Hq, gap, dtype, cuda_device):
    from autoindexer_b200 import read_status, shared_prefix_attention

    n = 1 << 18
    args, gap = _lists(B, T, Hq, n, gap, lambda d: torch.ones(len(d)), lambda d: torch.ones(len(d)), dtype, cuda_device)
    _, lse = shared_prefix_attention(*args, scaling=1.0, return_lse=True)
    assert read_status(cuda_device) == 0
    for t in range(T):
        want = math.log1p((n - T + t) * math.exp(-gap))
        err = float((lse[:, :, t].double() - want).abs().max())
        assert err <= _eps(64, gap) * (1 + want), err / (_eps(64, gap) * (1 + want))
