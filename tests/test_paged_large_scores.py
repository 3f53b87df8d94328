"""``shared_prefix_attention`` with scores of 2^26: the running maximum's own
rounding is then up to 4 in the exponent, a factor that every weight of a row
shares and that has to fit beside the weights in the tensors' type.

Scores are exact (multiples of 8 below 2^27).  Within a stretch of keys the
weights are those of the scores' differences; the stretches' log-sums are
float32 numbers of 2^26, rounded by up to 4, so two stretches' weights may stand
in a ratio that is wrong by 2^8.  The values are 1 in one of two dimensions:
what a row gathers is 1 in all, within the rounding of each dimension.
"""

import math

import pytest
import torch

from test_head_norm import U


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("B,T,Hq", [(888, 1, 1), (888, 1, 16), (296, 5, 16), (148, 9, 16)])
def test_scores_of_two_to_the_26(B, T, Hq, dtype, cuda_device):
    from autoindexer_b200 import shared_prefix_attention

    D, S, n = 64, 128, 1024
    kp = torch.zeros(n // S, 1, S, D, dtype=dtype, device=cuda_device)
    kp[..., 0] = 8192
    late = 700  # one key a little above the others, in a later tile
    kp[late // S, 0, late % S, 1] = 8
    vp = torch.zeros_like(kp)
    vp[..., 0] = 1
    vp[late // S, 0, late % S, 0], vp[late // S, 0, late % S, 1] = 0, 1
    q = torch.zeros(B, Hq, T, D, dtype=dtype, device=cuda_device)
    q[..., 0], q[..., 1] = 8192, 1
    table = torch.arange(n // S, dtype=torch.int32, device=cuda_device).expand(B, n // S).contiguous()
    lens = torch.full((B,), n, dtype=torch.int32, device=cuda_device)
    for i in range(40):
        scale = 0.66 + 0.001 * i  # (a row maximum of up to 2^26.01 in powers of two)
        out = shared_prefix_attention(q, kp, vp, None, 0, table, lens, scaling=scale).double().cpu()
        total = out[..., 0] + out[..., 1]
        assert float((total - 1).abs().max()) <= 2 * U[dtype] + 2.0 ** -16, scale
        for t in range(T):
            want = math.exp(8 * scale) / (n - T + t)
            got = out[:, t, :, 1] / out[:, t, :, 0]
            assert float(got.min()) >= want / 257 and float(got.max()) <= want * 257, (scale, t)
