"""An infinite temperature: every word that is not masked has the same probability,
a masked one none.  Tolerances as in ``test_scoring``."""

import math

import pytest
import torch

from test_scoring import INF, REL


@pytest.mark.gpu
@pytest.mark.parametrize("V", [50, 20001, 150001])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_scores(V, dtype, cuda_device):
    from autoindexer_b200 import read_status, token_logprobs

    g = torch.Generator().manual_seed(V)
    x = (3 * torch.randn(5, V, generator=g)).to(dtype)
    x[:, ::3] = -INF
    x[4] = -INF
    tokens = torch.tensor([3, 4, 0, V - 1 - (V - 1) % 3, 2])  # masked, not, masked, masked, no word at all
    tau = torch.full((5,), INF)
    x, tokens, tau = (y.to(cuda_device) for y in (x, tokens, tau))
    leaf = x.clone().requires_grad_()
    got = token_logprobs(leaf, tokens, tau, top_k=4, entropy=True)
    n = V - (V + 2) // 3
    for i, seen in enumerate((False, True, False, False, False)):
        if seen:
            assert abs(got.logprobs[i].item() + math.log(n)) <= REL * (1 + math.log(n))
        else:
            assert got.logprobs[i].item() == -INF
    want = torch.tensor([math.log(n)] * 4 + [0.0])
    assert bool(((got.entropy.cpu() - want).abs() <= 4 * REL * (1 + want)).all())
    assert bool((got.top_logprobs[:4].cpu() + math.log(n)).abs().le(REL * (1 + math.log(n))).all())
    assert bool(got.top_logprobs[4].eq(-INF).all()) and bool(got.top_tokens[4].eq(-1).all())
    d = torch.autograd.grad([got.entropy.sum() + got.top_logprobs[:4].sum()], leaf)[0]
    assert not bool(d.any())
    assert read_status(cuda_device) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("tail", ["bucket", "renormalize"])
@pytest.mark.parametrize("V", [50, 20001, 150001])
def test_distillation(V, tail, cuda_device):
    """A masked listed word makes the loss infinite, as at any temperature."""
    from autoindexer_b200 import distill_loss, distill_loss_and_grad

    g = torch.Generator().manual_seed(V)
    x = 3 * torch.randn(4, V, generator=g)
    x[0, 7], x[1, 20:], x[3, 20:] = -INF, -INF, -INF
    ids = torch.tensor([[7, 8, 9], [1, 2, 3], [1, 2, 3], [30, 31, 32]])
    t = torch.log(torch.tensor([0.5, 0.3, 0.1])).repeat(4, 1)
    args = [y.to(cuda_device) for y in (x, ids, t)]
    tau = torch.full((4,), INF, device=cuda_device)
    losses, grad = distill_loss_and_grad(*args, temperature=tau, tail=tail)
    alone = distill_loss(args[0].repeat(200, 1), *(y.repeat(200, 1) for y in args[1:]), tau.repeat(200), tail)
    p = t[0].double().exp()
    for i, n in ((1, 20), (2, V)):
        q = p / p.sum() if tail == "renormalize" else p
        want = float((q * (q.log() + math.log(n))).sum())
        if tail == "bucket":
            left = float(1 - p.sum())
            want += left * (math.log(left) - math.log((n - 3) / n))
        assert abs(losses[i].item() - want) <= REL * (1 + 10 * math.log(n))
    assert losses[0].item() == INF and losses[3].item() == INF
    assert not bool(grad.any())
    assert torch.equal(alone.view(200, 4), losses.expand(200, 4))


@pytest.mark.gpu
@pytest.mark.parametrize("tail", ["bucket", "renormalize"])
def test_the_smallest_temperature(tail, cuda_device):
    """1 / tau is as large as fp32 goes: a student that is sure of the teacher's word."""
    from autoindexer_b200 import distill_loss_and_grad

    x = torch.zeros(2, 100)
    x[:, 5] = 1.0
    ids = torch.tensor([[5], [5]])
    t = torch.tensor([[0.0], [2.0 ** -20]])  # (the second sums to more than 1)
    losses, grad = distill_loss_and_grad(*(y.to(cuda_device) for y in (x, ids, t)), tail=tail,
                                         temperature=torch.full((2,), 1e-45, device=cuda_device))
    assert bool((losses.abs() <= 2.0 ** -19).all())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("tau", [1e-45, 1e-38, 1e-36, 1e-30])
def test_gradients_at_small_temperatures(tau, dtype, cuda_device):
    """Upstream gradients over tau may pass fp32's range; a row that is sure of its
    word has the gradient 0 all the same."""
    from autoindexer_b200 import distill_loss, distill_loss_and_grad, token_logprobs

    V = 1003
    x = torch.randn(3, V, generator=torch.Generator().manual_seed(1)).clamp(-2, 2)
    x[0, 5], x[1, V - 1], x[2, 40] = 9.0, 8.0, 7.0
    best = torch.tensor([5, V - 1, 40])
    x, best = x.to(dtype).to(cuda_device), best.to(cuda_device)
    t = torch.full((3,), tau, device=cuda_device)
    for up in (1.0, -3.0, 1e6):
        leaf = x.clone().requires_grad_()
        got = token_logprobs(leaf, best, t, top_k=1, entropy=True)
        d = torch.autograd.grad([got.logprobs, got.entropy, got.top_logprobs], leaf,
                                [torch.full((3,), up, device=cuda_device), torch.full((3,), up, device=cuda_device),
                                 torch.full((3, 1), up, device=cuda_device)])[0]
        assert not bool(d.any()), (tau, up)
        ids, lp = best[:, None], torch.zeros(3, 1, device=cuda_device)
        w = torch.full((3,), up, device=cuda_device)
        losses, grad = distill_loss_and_grad(x, ids, lp, w, t)
        loss = distill_loss(leaf, ids, lp, t)
        through = torch.autograd.grad(loss, leaf, w)[0]
        assert not bool(grad.any()) and not bool(through.any()) and not bool(losses.any()) and torch.equal(loss, losses)
