"""Distillation with a bucket where the teacher's list leaves little: p_r = 1 - sum
p_k keeps its digits.

Tolerances as in ``test_distill`` with p_r as good as fp32 holds it: the gradient of
a word that is not listed is ``share (q_r - p_r)``, each part good to 4 REL."""

import math

import numpy as np
import pytest
import torch

from test_scoring import FLUSH, REL

V = 700


def lists(left, K, seed):
    """fp32 log-probabilities of K words that leave about ``left``, and what they leave."""
    g = np.random.default_rng(seed)
    p = np.sort(g.random(K) ** 3 + 1e-3)[::-1]
    p = p / p.sum() * (1 - left)
    t = np.log(p).astype(np.float32)
    return t, 1 - math.fsum(math.exp(float(x)) for x in t)


def expected(x, ids, t, left):
    """Loss and gradient of one row from its definition, and the magnitudes."""
    p = np.exp(t.astype(np.float64))
    other = np.ones(V, dtype=bool)
    other[ids] = False
    z = x - x.max()
    total = math.fsum(np.exp(z))
    ln_q = z - math.log(total)
    m = x[other].max()
    share = np.exp(x[other] - m) / math.fsum(np.exp(x[other] - m))
    ln_r = m - x.max() - math.log(total) + math.log(math.fsum(np.exp(x[other] - m)))
    loss = math.fsum(p * (t - ln_q[ids])) + left * (math.log(left) - ln_r)
    big = math.fsum(p * (np.abs(t) + np.abs(ln_q[ids]))) + left * (abs(math.log(left)) + abs(ln_r))
    d, mag = np.zeros(V), np.zeros(V)
    d[ids], mag[ids] = np.exp(ln_q[ids]) - p, np.exp(ln_q[ids]) + p
    d[other], mag[other] = share * (math.exp(ln_r) - left), share * (math.exp(ln_r) + left)
    return loss, big, d, mag


@pytest.mark.gpu
@pytest.mark.parametrize("K", [1, 2, 17, 32, 33, 128])
@pytest.mark.parametrize("left", [1e-2, 1e-4, 1e-5, 2e-6, 9e-7])
@pytest.mark.parametrize("lift", [3.0, 12.0, 60.0])
def test_small_remainders(left, K, lift, cuda_device):
    """A student whose other words have e^-lift of its probability or so."""
    from autoindexer_b200 import distill_loss, distill_loss_and_grad, read_status

    rows = 3
    g = np.random.default_rng(K)
    x, ids, t, lefts = np.zeros((rows, V), np.float32), np.zeros((rows, K), np.int64), np.zeros((rows, K), np.float32), []
    for i in range(rows):
        ids[i] = g.permutation(V)[:K]
        t[i], rest = lists(left, K, 100 * i + K)
        lefts.append(rest)
        x[i] = g.normal(size=V)
        x[i, ids[i]] = lift + t[i]
    args = [torch.tensor(y).to(cuda_device) for y in (x, ids, t)]
    losses, grad = distill_loss_and_grad(*args)
    leaf = args[0].clone().requires_grad_()
    alone = distill_loss(leaf, *args[1:])
    through = torch.autograd.grad(alone.sum(), leaf)[0]
    assert read_status(cuda_device) == 0
    for i in range(rows):
        loss, big, d, mag = expected(x[i].astype(np.float64), ids[i], t[i], lefts[i])
        for got in (losses, alone.detach()):
            assert abs(got[i].item() - loss) <= REL * (5e-2 + big), (got[i].item(), loss)
        for got in (grad, through):
            err = np.abs(got[i].double().cpu().numpy() - d)
            tol = 4 * REL * mag + 2.0 ** -24 * np.abs(d) + FLUSH
            assert (err <= tol).all(), (i, (err / np.maximum(mag, 1e-300)).max())


@pytest.mark.gpu
@pytest.mark.parametrize("K", [1, 5, 128])
def test_what_rounding_leaves_counts_as_none(K, cuda_device):
    """Lists that hold all of the teacher's probability, but for fp32's rounding of
    them, beside other words that the student has masked with the type's lowest value."""
    from autoindexer_b200 import distill_loss_and_grad

    rows = 64
    g = torch.Generator().manual_seed(K)
    x = torch.full((rows, V), torch.finfo(torch.float32).min)
    ids = torch.stack([torch.randperm(V, generator=g)[:K] for _ in range(rows)])
    z = 2 * torch.randn(rows, K, generator=g)
    x.scatter_(-1, ids, z + torch.randn(rows, K, generator=g))
    t = torch.log_softmax(z.double(), -1).float()
    losses, grad = distill_loss_and_grad(*(y.to(cuda_device) for y in (x, ids, t)))
    y = x.gather(-1, ids).double()
    lq, tt = torch.log_softmax(y, -1), t.double()
    want = (tt.exp() * (tt - lq)).sum(-1)
    assert bool(((losses.double().cpu() - want).abs() <= REL * (1 + want.abs())).all())
    assert bool(((grad.cpu().gather(-1, ids).double() - (lq.exp() - tt.exp())).abs() <= 8 * REL).all())
