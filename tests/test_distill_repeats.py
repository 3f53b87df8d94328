"""Words that a teacher's list has twice, wherever the two entries stand: the later
one is left out and reported, none else."""

import pytest
import torch


@pytest.mark.gpu
@pytest.mark.parametrize("tail", ["bucket", "renormalize"])
@pytest.mark.parametrize("K,V,n", [(64, 900, 64), (128, 900, 128), (97, 70001, 200), (128, 200003, 40)])
def test_any_two_places(K, V, n, tail, cuda_device):
    from autoindexer_b200 import distill_loss, distill_loss_and_grad, read_status

    g = torch.Generator().manual_seed(K)
    x = 2 * torch.randn(n, V, generator=g)
    ids = torch.stack([torch.randperm(V, generator=g)[:K] for _ in range(n)])
    t = torch.log_softmax(torch.randn(n, K, generator=g), -1) - 0.1
    args = [y.to(cuda_device) for y in (x, ids, t)]
    assert read_status(cuda_device) == 0
    distill_loss_and_grad(*args, tail=tail)
    distill_loss(*args, tail=tail)
    assert read_status(cuda_device) == 0
    # Row i: the entry at `first` again at `later` (each set of 32 with each), and the same list without it.
    twice, once = ids.clone(), ids.clone()
    for i in range(n):
        first, later = sorted((int(torch.randint(0, K, (1,), generator=g)), i % K))
        if first == later:
            first, later = (later - 1, later) if later else (0, K - 1)
        twice[i, later], once[i, later] = ids[i, first], -1
    twice, once = twice.to(cuda_device), once.to(cuda_device)
    got = distill_loss_and_grad(args[0], twice, args[2], tail=tail)
    assert read_status(cuda_device) == -2
    want = distill_loss_and_grad(args[0], once, args[2], tail=tail)
    assert read_status(cuda_device) == 0
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    leaf = args[0].clone().requires_grad_()
    loss = distill_loss(leaf, twice, args[2], tail=tail)
    assert read_status(cuda_device) == -2
    d = torch.autograd.grad(loss.sum(), leaf)[0]
    other = distill_loss(leaf, once, args[2], tail=tail)
    assert torch.equal(loss, other) and torch.equal(d, torch.autograd.grad(other.sum(), leaf)[0])
