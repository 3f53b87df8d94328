"""Distillation from a teacher's likeliest tokens (``distill_loss``,
``distill_loss_and_grad``) against the definition in 64 bits, and refusals.

Tolerances as in ``test_scoring``: sums of weights are good to 2^-18, so ln q_k
and ln q_r to REL (1 + |value|), REL = 1e-5, and a loss to REL times the
magnitude of the terms it sums, and p_r = 1 - sum p_k to 2^-21; an entry of the gradient to 4 REL times the
magnitude of its terms and half a step of its type, and 0 for what the exponential
flushes (below 2^-126)."""

import ctypes

import numpy as np
import pytest
import torch
from torch.autograd import forward_ad

from oracle import learning_oracle as O
from test_scoring import FLUSH, INF, REL, close, odd_rows

TAILS = ["bucket", "renormalize"]


def make(shape, V, K, dtype, seed, ragged=True):
    g = torch.Generator().manual_seed(seed)
    x = 2 * torch.randn(*shape, V, generator=g)
    n = int(np.prod(shape))
    ids = torch.stack([torch.randperm(V, generator=g)[:K] for _ in range(n)])
    if ids.shape[1] < K:  # a vocabulary smaller than the list
        ids = torch.cat((ids, torch.full((n, K - ids.shape[1]), -1)), 1)
    ids = ids.reshape(*shape, K)
    t = torch.log_softmax(torch.sort(2 * torch.randn(*shape, K, generator=g), -1, descending=True)[0], -1)
    t = t + torch.log(0.5 + 0.45 * torch.rand(*shape, 1, generator=g))
    x.scatter_add_(-1, ids.clamp_min(0), 4 + t)
    if ragged and n > 2:
        ids.view(n, K)[1] = -1                      # no list
        ids.view(n, K)[2, K // 2:] = -1             # a shorter one
        t.view(n, K)[2, K // 2:] = -INF
    w = 0.5 + torch.rand(shape, generator=g)
    w.view(-1)[-1] = 0.0 if n > 1 else 1.0
    tau = 0.5 + torch.rand(shape[0], generator=g)
    return x.to(dtype), ids, t.float(), w, tau


def check(x, ids, t, w, tau, tail, losses, grad):
    dtype, V, K = x.dtype, x.shape[-1], ids.shape[-1]
    flat = x.detach().double().cpu().reshape(-1, V).numpy()
    ids, t = ids.cpu().reshape(-1, K).numpy(), t.double().cpu().reshape(-1, K).numpy()
    per = len(flat) // x.shape[0]
    for i, row in enumerate(flat):
        weight = 1.0 if w is None else w.reshape(-1)[i].double().item()
        loss, d, mag, big = O.distill_row(row, ids[i], t[i], 1.0 if tau is None else float(tau[i // per]), tail, weight)
        if losses is not None:
            if loss > torch.finfo(torch.float32).max:  # rounds to inf: logits at the type's lowest value, divided by tau < 1
                loss = INF
            close(losses.reshape(-1)[i].item(), loss, REL * (1 + big), f"loss of row {i}")
        if grad is not None:
            fin = torch.finfo(dtype)
            tol = 4 * REL * mag + fin.eps / 2 * np.abs(d) + fin.smallest_normal * fin.eps + FLUSH
            close(grad.reshape(-1, V)[i].double().cpu().numpy(), d, tol, f"gradient of row {i}")


CASES = [
    ((1, 1), 1, 1, torch.float32),
    ((3,), 2, 3, torch.bfloat16),
    ((2, 3), 37, 5, torch.float16),
    ((4, 5), 1001, 20, torch.bfloat16),
    ((7,), 8191, 128, torch.float32),
    ((3, 3), 32003, 64, torch.float16),
    ((1, 3), 151936, 33, torch.bfloat16),
    ((5, 33), 4099, 1, torch.float32),
    ((2, 2), 140001, 40, torch.float32),
    ((650,), 3000, 8, torch.bfloat16),
    ((3,), 786431, 16, torch.float32),
]


@pytest.mark.gpu
@pytest.mark.parametrize("tail", TAILS)
@pytest.mark.parametrize("shape,V,K,dtype", CASES)
def test_against_definition(shape, V, K, dtype, tail, cuda_device):
    from autoindexer_b200 import distill_loss, distill_loss_and_grad, read_status

    x, ids, t, w, tau = (y.to(cuda_device) for y in make(shape, V, K, dtype, V + K))
    for temp in (None, tau):
        losses, grad = distill_loss_and_grad(x, ids, t, w, temperature=temp, tail=tail)
        assert losses.shape == shape and losses.dtype == torch.float32 and grad.shape == x.shape and grad.dtype == dtype
        check(x, ids, t, w, temp, tail, losses, grad)
        again = distill_loss_and_grad(x, ids, t, w, temperature=temp, tail=tail)
        assert torch.equal(losses, again[0]) and torch.equal(grad, again[1])
        y = x.clone().requires_grad_()
        loss = distill_loss(y, ids, t, temperature=temp, tail=tail)
        check(x, ids, t, None, temp, tail, loss.detach(), None)
        check(x, ids, t, w, temp, tail, None, torch.autograd.grad(loss, y, w)[0])
        assert torch.equal(distill_loss(x, ids, t, temperature=temp, tail=tail), loss.detach())
    check(x, ids, t, None, None, tail, *distill_loss_and_grad(x, ids, t, tail=tail))
    assert read_status(cuda_device) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("tail", TAILS)
def test_gradient_against_differences(tail, cuda_device):
    from autoindexer_b200 import distill_loss_and_grad

    x, ids, t, w, tau = make((2, 3), 301, 9, torch.float32, 5)
    grad = distill_loss_and_grad(*(y.to(cuda_device) for y in (x, ids, t, w, tau)), tail=tail)[1].double().cpu()
    step, g = 1e-5, torch.Generator().manual_seed(1)

    def f(y):
        return sum(w.view(-1)[i].double().item() * O.distill_row(y.reshape(-1, 301)[i].numpy(), ids.view(-1, 9)[i].numpy(),
                                                                 t.view(-1, 9)[i].double().numpy(), float(tau[i // 3]), tail)[0]
                   for i in range(6))

    for _ in range(5):
        way = torch.randn(x.shape, generator=g, dtype=torch.float64)
        slope = (f(x.double() + step * way) - f(x.double() - step * way)) / (2 * step)
        assert abs(slope - float((grad * way).sum())) < 1e-4 * (1 + abs(slope))


@pytest.mark.gpu
@pytest.mark.parametrize("tail", TAILS)
@pytest.mark.parametrize("V", [40, 9001, 140003])
def test_awkward_rows(V, tail, cuda_device):
    """Masked rows, ties and far values; lists whose words are masked, cover the
    whole row, or leave nothing for the bucket."""
    from autoindexer_b200 import distill_loss_and_grad, read_status

    rows = odd_rows(V)
    x = torch.stack(list(rows.values()))
    n, K = len(rows), 4
    ids = torch.tensor([V // 2, 3, 1, V - 1]).repeat(n, 1)
    t = torch.log(torch.tensor([0.4, 0.3, 0.2, 0.05])).repeat(n, 1)
    x, ids, t = (y.to(cuda_device) for y in (x, ids, t))
    check(x, ids, t, None, None, tail, *distill_loss_and_grad(x, ids, t, tail=tail))
    # The teacher is sure (sum p rounds to 1 or beyond), or knows nothing at all.
    t[:] = torch.log(torch.tensor([0.7, 0.3, 1e-9, 1e-12]))
    ids[1::2] = torch.tensor([-1, -5, V // 3, -1], device=cuda_device)
    check(x, ids, t, None, None, tail, *distill_loss_and_grad(x, ids, t, tail=tail))
    t[:, 2] = -INF
    check(x, ids, t, None, None, tail, *distill_loss_and_grad(x, ids, t, tail=tail))
    assert read_status(cuda_device) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("tail", TAILS)
@pytest.mark.parametrize("V,K,dtype,n", [(7, 3, torch.bfloat16, 50), (1003, 40, torch.float16, 50), (3077, 128, torch.bfloat16, 50),
                                         (9001, 64, torch.float32, 50), (30011, 100, torch.bfloat16, 50), (65541, 128, torch.float16, 7),
                                         (32800, 33, torch.float32, 13), (70003, 5, torch.bfloat16, 40)])
def test_many_rows(V, K, dtype, n, tail, cuda_device):
    """More rows than run at once, awkward ones among them: copies of a row come out alike,
    in place too, and through autograd."""
    from autoindexer_b200 import distill_loss, distill_loss_and_grad, read_status

    x, ids, t, w, tau = make((24,), V, K, dtype, K)
    for i, row in enumerate(list(odd_rows(V).values())[:12] if V > 20 else []):
        x[3 + i] = row.to(dtype)
    ids[20, 0], ids[20, -1] = 0, V - 1
    few = [x, ids, t, w, tau]
    many = [y.to(cuda_device).repeat(n, *[1] * (y.dim() - 1)) for y in few]
    losses, grad = distill_loss_and_grad(*many, tail=tail)
    check(*few[:3], w, tau, tail, losses[:24].cpu(), grad[:24].cpu())
    leaf = many[0].clone().requires_grad_()
    alone = distill_loss(leaf, *many[1:3], many[4], tail=tail)
    through = torch.autograd.grad(alone, leaf, many[3])[0]
    live = w != 0
    check(x[live], ids[live], t[live], w[live], tau[live], tail, alone.detach()[:24][live.to(cuda_device)].cpu(),
          through[:24][live.to(cuda_device)].cpu())
    for y in (losses, grad, alone.detach(), through):
        assert all(torch.equal(y[24 * i:24 * i + 24].nan_to_num(9), y[:24].nan_to_num(9)) for i in range(n))
    here = distill_loss_and_grad(*many, tail=tail, out=many[0])
    assert torch.equal(here[1].nan_to_num(9), grad.nan_to_num(9))
    read_status(cuda_device)  # (word 0 is also word V - 1 where a list has one twice)


@pytest.mark.gpu
@pytest.mark.parametrize("tail", TAILS)
def test_a_sure_student_keeps_its_tail(tail, cuda_device):
    """The other words' probability of 1e-9 and 1e-40 is not lost beside the listed ones'."""
    from autoindexer_b200 import distill_loss_and_grad

    V, K = 5000, 3
    x = torch.zeros(4, V)
    for i, up in enumerate((30.0, 100.0, 300.0, 3000.0)):
        x[i, :K] = up
    ids = torch.arange(K).repeat(4, 1)
    t = torch.log(torch.tensor([0.5, 0.2, 0.1])).repeat(4, 1)
    x, ids, t = (y.to(cuda_device) for y in (x, ids, t))
    check(x, ids, t, None, None, tail, *distill_loss_and_grad(x, ids, t, tail=tail))


@pytest.mark.gpu
@pytest.mark.parametrize("tail", TAILS)
def test_words_out_of_range_and_twice(tail, cuda_device):
    from autoindexer_b200 import distill_loss_and_grad, read_status

    x, ids, t, w, tau = (y.to(cuda_device) for y in make((5,), 700, 6, torch.float32, 2, ragged=False))
    ids[0, 2], ids[1, 0], ids[2, 5] = 700, 2 ** 32 + 3, -7
    assert read_status(cuda_device) == 0
    got = distill_loss_and_grad(x, ids, t, w, tau, tail)
    assert read_status(cuda_device) == -2
    check(x, ids, t, w, tau, tail, *got)
    ids[0, 2], ids[1, 0] = -1, -1
    distill_loss_and_grad(x, ids, t, w, tau, tail)
    assert read_status(cuda_device) == 0
    ids[3, 4] = ids[3, 1]
    got = distill_loss_and_grad(x, ids, t, w, tau, tail)
    assert read_status(cuda_device) == -2
    check(x, ids, t, w, tau, tail, *got)


@pytest.mark.gpu
@pytest.mark.parametrize("tail", TAILS)
@pytest.mark.parametrize("V", [33, 20001])
def test_nan_and_infinity(V, tail, cuda_device):
    from autoindexer_b200 import distill_loss_and_grad

    x, ids, t, w, tau = make((8,), V, 5, torch.float32, 3)
    nan = float("nan")
    x[0, V - 1], x[3, int(ids[3, 2])], x[4, 0] = nan, nan, INF
    t[5, 1] = nan
    x[1], x[7] = nan, nan  # no list; weight 0: not read
    args = [y.to(cuda_device) for y in (x, ids, t, w, tau)]
    losses, grad = distill_loss_and_grad(*args, tail=tail)
    check(x, ids, t, w, tau, tail, losses, grad)
    assert losses[[1, 7]].eq(0).all() and not bool(grad[[1, 7]].any())
    assert bool(losses[[0, 3, 4, 5]].isnan().all()) and bool(grad[[0, 3, 4, 5]].isnan().all())


@pytest.mark.gpu
@pytest.mark.parametrize("lay", ["padded", "off", "transposed", "stepped", "place", "into"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_strides_and_places(lay, dtype, cuda_device):
    """Rows of other strides, and the gradient written to ``out``, over the logits too."""
    from autoindexer_b200 import distill_loss, distill_loss_and_grad

    x, ids, t, w, tau = (y.to(cuda_device) for y in make((3, 4), 1003, 7, dtype, 12))
    want = distill_loss_and_grad(x, ids, t, w, tau)
    check(x, ids, t, w, tau, "bucket", *want)
    guard = 77.0
    if lay in ("padded", "off"):
        at = 0 if lay == "padded" else 5
        base = torch.full((3, 4, 1016), guard, dtype=dtype, device=cuda_device)
        base[..., at:at + 1003] = x
        view = base[..., at:at + 1003]
        got = distill_loss_and_grad(view, ids, t, w, tau)
        if lay == "off":
            here = distill_loss_and_grad(view, ids, t, w, tau, out=view)
            assert torch.equal(here[1], got[1])
            assert base[..., :5].eq(guard).all() and base[..., 1008:].eq(guard).all()
    elif lay == "transposed":
        got = distill_loss_and_grad(x.transpose(0, 1).contiguous().transpose(0, 1), ids, t, w, tau)
    elif lay == "stepped":
        base = torch.zeros(3, 4, 2006, dtype=dtype, device=cuda_device)
        base[..., ::2] = x
        got = distill_loss_and_grad(base[..., ::2], ids.transpose(0, 1).contiguous().transpose(0, 1), t, w, tau)
    elif lay == "place":
        y = x.clone().requires_grad_()
        got = distill_loss_and_grad(y, ids, t, w, tau, out=y)
        assert got[1].data_ptr() == y.data_ptr()
        y = x.clone().requires_grad_()
        loss = distill_loss(y, ids, t, tau)
        distill_loss_and_grad(y, ids, t, w, tau, out=y)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            loss.sum().backward()
    else:
        out = torch.full((3, 4, 1010), guard, dtype=dtype, device=cuda_device)
        got = distill_loss_and_grad(x, ids, t, w, tau, out=out[..., 3:1006])
        assert out[..., :3].eq(guard).all() and out[..., 1006:].eq(guard).all()
    check(x, ids, t, w, tau, "bucket", *got)


@pytest.mark.gpu
def test_offsets_past_31_bits(cuda_device):
    from autoindexer_b200 import distill_loss_and_grad

    far, V = 2 ** 31 + 5, 1000
    base = torch.empty(far + V, dtype=torch.bfloat16, device=cuda_device)
    x = base.as_strided((2, 1, V), (far, V, 1))
    src, ids, t, w, tau = (y.to(cuda_device) for y in make((2, 1), V, 6, torch.bfloat16, 4))
    x.copy_(src)
    check(src, ids, t, None, tau, "bucket", *distill_loss_and_grad(x, ids, t, None, tau, out=x))


@pytest.mark.gpu
@pytest.mark.parametrize("shape,V", [((2,), 50001), ((40, 20), 700)])
def test_captured_graph_and_another_stream(shape, V, cuda_device):
    from autoindexer_b200 import distill_loss, distill_loss_and_grad

    args = [y.to(cuda_device) for y in make(shape, V, 9, torch.bfloat16, 8)]
    other = make(shape, V, 9, torch.bfloat16, 9)
    x = args[0].requires_grad_()

    def step():
        loss, grad = distill_loss_and_grad(x.detach(), *args[1:])
        soft = distill_loss(x, *args[1:3], args[4])
        return [loss, grad, soft.detach(), *torch.autograd.grad(soft, x, args[3])]

    step()
    torch.cuda.synchronize(cuda_device)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for values in (None, other):
        if values is not None:
            for a, b in zip(args, values):
                a.data.copy_(b)
        graph.replay()
        want = step()
        side = torch.cuda.Stream(cuda_device)
        side.wait_stream(torch.cuda.current_stream(cuda_device))
        with torch.cuda.stream(side):
            third = step()
        torch.cuda.synchronize(cuda_device)
        assert all(torch.equal(a, b) and torch.equal(a, c) for a, b, c in zip(got, want, third))
    del got
    graph.reset()


@pytest.mark.gpu
@pytest.mark.parametrize("tail", TAILS)
@pytest.mark.parametrize("shape,V,dtype", [((5,), 7, torch.float32), ((3, 2), 1003, torch.float16), ((2,), 150001, torch.bfloat16),
                                           ((700,), 515, torch.float32)])
def test_backward_of_its_own(shape, V, dtype, tail, cuda_device):
    """Upstream gradients of either sign, zero and NaN; saved tensors that hooks bring
    back with other strides; lists with a word twice and words that are masked."""
    from autoindexer_b200 import distill_loss, distill_loss_and_grad, read_status

    x, ids, t, w, tau = (y.to(cuda_device) for y in make(shape, V, 5, dtype, 21))
    ids.view(-1, 5)[0, 3] = ids.view(-1, 5)[0, 1]
    x.view(-1, V)[-2, int(ids.view(-1, 5)[-2, 0].clamp_min(0))] = -INF
    x.view(-1, V)[0, V // 2:] = -INF
    w.view(-1)[0] *= -1
    check(x, ids, t, w, tau, tail, *distill_loss_and_grad(x, ids, t, w, tau, tail))
    y = x.clone().requires_grad_()
    plain = distill_loss(y, ids, t, tau, tail)
    want = torch.autograd.grad(plain, y, w)[0]
    check(x, ids, t, w, tau, tail, None, want)
    wide = lambda z: torch.stack((z, z), -1)[..., 0]  # noqa: E731
    with torch.autograd.graph.saved_tensors_hooks(lambda z: z, wide):
        loss = distill_loss(y, ids, t, tau, tail)
    assert torch.equal(torch.autograd.grad(loss, y, wide(w), retain_graph=True)[0], want)
    base = torch.zeros(*shape, 2 * V, dtype=dtype, device=cuda_device)
    base[..., ::2] = x
    base.requires_grad_()
    d = torch.autograd.grad(distill_loss(base[..., ::2], ids, t, tau, tail), base, w)[0]
    assert torch.equal(d[..., ::2], want) and not bool(d[..., 1::2].any())
    read_status(cuda_device)  # (the word twice)
    nan = torch.full(shape, float("nan"), device=cuda_device)
    d = torch.autograd.grad(loss, y, nan)[0].reshape(-1, V)
    live = (ids.view(-1, 5) >= 0).any(1)
    assert bool(d[live].isnan().any(1).all()) and not bool(d[~live].any())


@pytest.mark.gpu
def test_gradients_that_do_not_exist(cuda_device):
    from autoindexer_b200 import distill_loss, distill_loss_and_grad

    x, ids, t, w, tau = (y.to(cuda_device) for y in make((3,), 50, 4, torch.float32, 3))
    for bad in ((x, ids, t.clone().requires_grad_()), (x, ids, t, tau.clone().requires_grad_())):
        with pytest.raises(RuntimeError, match="no gradient for"):
            distill_loss(*bad)
    y = x.clone().requires_grad_()
    losses, grad = distill_loss_and_grad(y, ids, t, w, tau)
    assert not grad.requires_grad
    with pytest.raises(RuntimeError, match="distill_loss_and_grad has no backward"):
        losses.sum().backward()
    y.backward(grad)
    assert torch.equal(y.grad, grad)
    for fn in (distill_loss, distill_loss_and_grad):
        with forward_ad.dual_level(), pytest.raises(RuntimeError, match="forward"):
            fn(forward_ad.make_dual(x, torch.ones_like(x)), ids, t)


@pytest.mark.gpu
def test_refusals(cuda_device):
    from autoindexer_b200 import distill_loss, distill_loss_and_grad

    x, ids, t, w, tau = (y.to(cuda_device) for y in make((2, 3), 200, 4, torch.bfloat16, 0))
    many = torch.zeros(2, 3, 129, dtype=torch.int64, device=cuda_device)
    for error, args in [
        (ValueError, (x[0, 0], ids, t)),
        (ValueError, (x[:, :0], ids[:, :0], t[:, :0])),
        (ValueError, (x, ids[:, :2], t)),
        (ValueError, (x, ids[..., :0], t[..., :0])),
        (ValueError, (x, many, many.float())),
        (ValueError, (x, ids, t[..., :3])),
        (ValueError, (x, ids, t, tau[:1])),
        (ValueError, (x, ids, t, None, "drop")),
        (ValueError, (x[:, :1].expand(2, 3, 200)[..., :1].expand(2, 3, 2 ** 21), ids, t)),
        (TypeError, (x, ids.int(), t)),
        (TypeError, (x, ids, t.double())),
        (TypeError, (x.double(), ids, t)),
        (RuntimeError, (x, ids.cpu(), t)),
        (RuntimeError, (x.cpu(), ids, t)),
    ]:
        with pytest.raises(error):
            distill_loss(*args)
    for error, more in [(ValueError, dict(weights=w[:, :1])), (TypeError, dict(weights=w.double())),
                        (ValueError, dict(out=x[:1])), (ValueError, dict(out=x.float())), (RuntimeError, dict(out=x.cpu())),
                        (ValueError, dict(out=x[:, :1].expand(2, 3, 200))),
                        (ValueError, dict(out=torch.empty(2, 200, 3, dtype=x.dtype, device=cuda_device).transpose(1, 2)))]:
        with pytest.raises(error):
            distill_loss_and_grad(x, ids, t, **more)


def test_cpu_tensors_are_refused():
    from autoindexer_b200 import distill_loss, distill_loss_and_grad

    x, ids, t, _, _ = make((2, 3), 50, 4, torch.bfloat16, 0)
    for fn in (distill_loss, distill_loss_and_grad):
        with pytest.raises(RuntimeError, match="CUDA tensors only"):
            fn(x, ids, t)


def test_c_abi_refusals():
    from autoindexer_b200 import _lib

    L = _lib.lib()

    def args(**over):
        a = _lib.AiDistillArgs()
        a.batch, a.seq_len, a.vocab, a.dtype, a.n_top = 2, 3, 100, _lib.DTYPE_BF16, 4
        a.logits = a.top_tokens = a.top_logprobs = a.losses = 256
        for n, v in over.items():
            setattr(a, n, v)
        return ctypes.byref(a)

    assert L.ai_distill(None, None) == 1
    for field, value, code in (("batch", 0, 2), ("vocab", 0, 2), ("n_top", 0, 2), ("n_top", 129, 2), ("tail", 2, 2), ("dtype", 5, 4),
                               ("batch", 2 ** 30, 2), ("vocab", 2 ** 21, 2), ("logits", None, 1), ("top_tokens", None, 1), ("top_logprobs", None, 1),
                               ("losses", None, 1), ("stride_b", -1, 5), ("dstride_t", -1, 5), ("logits", 257, 6), ("dlogits", 255, 6)):
        assert L.ai_distill(args(**{field: value}), None) == code, field


def test_c_abi_refusals_of_the_backward():
    from autoindexer_b200 import _lib

    L = _lib.lib()
    assert L.ai_distill_bwd(None, None) == 1

    def args(**over):
        g = _lib.AiDistillBwdArgs()
        a = g.fwd
        a.batch, a.seq_len, a.vocab, a.dtype, a.n_top = 2, 3, 100, _lib.DTYPE_BF16, 4
        a.logits = a.top_tokens = a.top_logprobs = a.row_stats = g.g_losses = g.dlogits = 256
        for n, v in over.items():
            setattr(a if n in ("vocab", "row_stats", "top_tokens") else g, n, v)
        return ctypes.byref(g)

    for field, value, code in (("vocab", 0, 2), ("row_stats", None, 1), ("row_stats", 264, 6), ("top_tokens", None, 1), ("g_losses", None, 1),
                               ("dlogits", None, 1), ("dlogits", 255, 6), ("dstride_b", -1, 5), ("dstride_t", -1, 5)):
        assert L.ai_distill_bwd(args(**{field: value}), None) == code, field


@pytest.mark.parametrize("tail", TAILS)
def test_oracle_gradient_follows_its_values(tail):
    rng = np.random.default_rng(0)
    x, ids, step = rng.normal(size=40), np.array([3, 9, -1, 30]), 1e-6
    t = np.log([0.4, 0.2, 0.5, 0.1])
    _, d, _, _ = O.distill_row(x, ids, t, 0.7, tail, 1.3)
    for v in (0, 3, 30):
        e = np.eye(40)[v] * step
        slope = 1.3 * (O.distill_row(x + e, ids, t, 0.7, tail)[0] - O.distill_row(x - e, ids, t, 0.7, tail)[0]) / (2 * step)
        assert abs(slope - d[v]) < 1e-7
    assert O.distill_row(np.log([0.25, 0.75]), np.array([0, 1]), np.log([0.25, 0.75]), 1.0, tail)[0] < 1e-12
