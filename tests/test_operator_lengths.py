"""Lengths out of range are clamped and set the status word, in all operators."""

import pytest
import torch

from test_verify import _case, _verify


@pytest.mark.gpu
@pytest.mark.parametrize("bad", [-1, 4, 2 ** 31 - 1, -2 ** 31])
def test_append_new_lens(bad, cuda_device):
    from autoindexer_b200 import paged_append, read_status

    k = torch.randn(3, 2, 3, 64, device=cuda_device)
    table = torch.arange(3, dtype=torch.int32, device=cuda_device)[:, None]
    lens = torch.zeros(3, dtype=torch.int32, device=cuda_device)

    def run(n):
        kp, vp = (torch.zeros(3, 2, 16, 64, device=cuda_device) for _ in range(2))
        paged_append(k, k, kp, vp, table, lens, new_lens=torch.tensor(n, dtype=torch.int32, device=cuda_device))
        return kp, vp

    read_status(cuda_device)
    want = run([3, min(max(bad, 0), 3), 0])
    assert read_status(cuda_device) == 0
    got = run([3, bad, 0])
    assert read_status(cuda_device) == -2
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.gpu
@pytest.mark.parametrize("bad", [-1, 4, 2 ** 31 - 1, -2 ** 31])
def test_verify_draft_lens(bad, cuda_device):
    from autoindexer_b200 import read_status, verify_draft

    t, x, u, e, d, n, tau = _case(3, 3, 700, torch.bfloat16, True, 4, cuda_device)
    n[1] = min(max(bad, 0), 3)
    read_status(cuda_device)
    want = verify_draft(t, x, u, e, d, n, tau)
    assert read_status(cuda_device) == 0
    wrong = n.clone()
    wrong[1] = bad
    got = verify_draft(t, x, u, e, d, wrong, tau)
    assert read_status(cuda_device) == -2
    assert all(torch.equal(p, q) for p, q in zip(got, want))
    _verify(t, x, u, e, d, n, tau, got)
