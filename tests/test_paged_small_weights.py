"""``shared_prefix_attention`` where one key takes nearly all the weight and
very many others in the same stretch share the rest.

Tolerance of the log-sum: as in ``test_paged.py`` (exponentials are added up
in blocks first, the running sum takes one number a block).  Of the output:
as there, and with n keys in one stretch

* ``n 2^-25 sum p |v|``: the matrix instructions align a step's products with
  the accumulator and cut each of them 25 bits below it;
* in float16 ``n 2^-32 max |v|``: a weight is held to 2^-25 (half of the
  smallest number), and weights are scaled by 2^7 for it."""

import math

import numpy as np
import pytest
import torch

from test_head_norm import U


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


VALUES = {
    "even": (lambda d: torch.where(d % 3 == 0, 1.0, 0.25), lambda d: torch.where(d % 2 == 0, 1.0, -0.75)),
    "nothing from the large one": (lambda d: torch.zeros(len(d)), lambda d: torch.where(d % 2 == 0, 1.0, -0.75)),
}


@pytest.mark.gpu
@pytest.mark.parametrize("values", list(VALUES))
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("gap", GAPS)
@pytest.mark.parametrize("B,T,Hq", SHAPES)
def test_output_of_many_small_weights(B, T, Hq, gap, dtype, values, cuda_device):
    from autoindexer_b200 import read_status, shared_prefix_attention

    n, (f0, f1) = 1 << 18, VALUES[values]
    args, gap = _lists(B, T, Hq, n, gap, f0, f1, dtype, cuda_device)
    out = shared_prefix_attention(*args, scaling=1.0)
    assert read_status(cuda_device) == 0
    v0, v1 = (f(torch.arange(64)).double().numpy() for f in (f0, f1))
    for t in range(T):
        rest = (n - T + t) * math.exp(-gap)
        want, mag = (v0 + rest * v1) / (1 + rest), (np.abs(v0) + rest * np.abs(v1)) / (1 + rest)
        tol = (2 * U[dtype] + _eps(64, gap) + n * 2.0 ** -25) * mag
        if dtype == torch.float16:
            tol = tol + n * 2.0 ** -32 * max(np.abs(v0).max(), np.abs(v1).max()) / (1 + rest)
        err = np.abs(out[:, t].double().cpu().numpy() - want)
        assert np.all(err <= tol), float((err / tol).max())
