"""The norm (forward and backward), the append and the verification in a
captured graph: a replay reads lengths, ids and tables as they are then."""

import pytest
import torch

from test_head_norm import _inputs, _table
from test_verify import _case


def _captured(fn, device):
    fn()  # (workspaces and the status word exist before the capture)
    torch.cuda.synchronize(device)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = fn()
    return graph, out


@pytest.mark.gpu
@pytest.mark.parametrize("T", [1, 300])
def test_norm_forward_and_backward(T, cuda_device):
    from autoindexer_b200 import qk_norm_rope, read_status

    ins = [x.requires_grad_() for x in _inputs(3, T, 8, 2, 128, torch.bfloat16, 3, cuda_device)]
    rope = _table(400, 128, cuda_device)
    pos = torch.arange(T, device=cuda_device).repeat(3, 1)
    gs = [torch.randn_like(x) for x in ins[:2]]

    def step():
        out = qk_norm_rope(*ins, rope, pos)
        return [*out, *torch.autograd.grad(out, ins, gs)]

    graph, got = _captured(step, cuda_device)
    for shift in (0, 57):
        pos.copy_(torch.arange(T, device=cuda_device) + shift)
        graph.replay()
        want = step()
        torch.cuda.synchronize(cuda_device)
        assert all(torch.equal(x, y) for x, y in zip(got, want))
    assert read_status(cuda_device) == 0
    del got
    graph.reset()


@pytest.mark.gpu
def test_append(cuda_device):
    from autoindexer_b200 import paged_append, read_status

    B, T, H, D, S = 3, 2, 2, 64, 16
    g = torch.Generator().manual_seed(1)
    k, v = (torch.randn(B, H, T, D, generator=g).to(cuda_device) for _ in range(2))
    table = torch.arange(2 * B, dtype=torch.int32, device=cuda_device).reshape(B, 2)
    lens, n = (torch.zeros(B, dtype=torch.int32, device=cuda_device) for _ in range(2))
    rope, pos = _table(64, D, cuda_device), torch.zeros(B, T, dtype=torch.long, device=cuda_device)
    pools = [torch.zeros(2 * B, H, S, D, device=cuda_device) for _ in range(4)]

    def step(kp, vp):
        paged_append(k, v, kp, vp, table, lens, rope, pos, n)

    graph, _ = _captured(lambda: step(*pools[:2]), cuda_device)
    for held, new in (([0, 5, 15], [2, 1, 2]), ([14, 30, 2], [2, 2, 0])):
        for x, y in ((lens, held), (n, new)):
            x.copy_(torch.tensor(y, dtype=torch.int32))
        pos.copy_(lens[:, None] + torch.arange(T, device=cuda_device))
        graph.replay()
        step(*pools[2:])
        torch.cuda.synchronize(cuda_device)
        assert torch.equal(pools[0], pools[2]) and torch.equal(pools[1], pools[3])
        assert bool(pools[0].any())
    assert read_status(cuda_device) == 0
    graph.reset()


@pytest.mark.gpu
@pytest.mark.parametrize("B,L,V", [(1, 3, 50001), (6, 2, 999)])
def test_verification(B, L, V, cuda_device):
    from autoindexer_b200 import read_status, verify_draft

    args = _case(B, L, V, torch.bfloat16, True, 8, cuda_device)
    other = _case(B, L, V, torch.bfloat16, True, 9, cuda_device)
    graph, got = _captured(lambda: verify_draft(*args), cuda_device)
    for values in (None, other):
        if values is not None:
            for x, y in zip(args, values):
                x.copy_(y)
        for _ in range(3):
            graph.replay()
        want = verify_draft(*args)
        torch.cuda.synchronize(cuda_device)
        assert all(torch.equal(x, y) for x, y in zip(got, want))
    assert read_status(cuda_device) == 0
    del got
    graph.reset()
