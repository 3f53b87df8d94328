"""Token log-probabilities, entropy, likeliest words and their gradient
(``token_logprobs``) against the definition in 64 bits, and refusals.

Tolerances.  A weight's exponent y = (x - m) c has two roundings (2^-23 |y|
together, of which weights that matter have |y| < 30) and its exponential one
of 2^-22; a thread's sum has a few dozen additions in a row (2^-24 each, all of
one sign).  So sums are good to 2^-18, log-probabilities to REL (1 + |value|) with
REL = 1e-5 > 2^-17, entropies (a difference of two such numbers, of at most
log2 V + 30) to 4 REL (1 + H), and an entry of the gradient to 4 REL times the
magnitude of its terms and half a step of its type; the exponential flushes
weights below 2^-126 to 0, which meet upstream gradients of less than 2^7."""

import ctypes

import numpy as np
import pytest
import torch
from torch.autograd import forward_ad

from oracle import learning_oracle as O

REL = 1e-5
FLUSH = 2.0 ** -119
INF = float("inf")


def make(shape, V, dtype, seed, spread=3.0):
    g = torch.Generator().manual_seed(seed)
    x = (spread * torch.randn(*shape, V, generator=g)).to(dtype)
    tokens = torch.randint(0, V, shape, generator=g)
    if len(shape) == 2 and shape[1] > 1:
        tokens[:, -1] = -100
    tau = 0.4 + 1.5 * torch.rand(shape[0], generator=g)
    return x, tokens, tau


def rows_of(x, tokens, tau):
    """(row, token, temperature) of each row, 64 bits."""
    V = x.shape[-1]
    flat, t = x.detach().double().cpu().reshape(-1, V).numpy(), tokens.cpu().reshape(-1).numpy()
    per = len(t) // x.shape[0]
    for i in range(len(t)):
        yield flat[i], int(t[i]), 1.0 if tau is None else float(tau[i // per])


def close(got, want, tol, what):
    got, want = np.asarray(got, dtype=np.float64), np.asarray(want, dtype=np.float64)
    with np.errstate(invalid="ignore"):
        ok = (got == want) | (np.isnan(got) & np.isnan(want)) | (np.abs(got - want) <= tol)
    assert ok.all(), f"{what}: {got[~ok][:4]} expected {want[~ok][:4]}, at {np.argwhere(~ok)[:4].tolist()}"


def check(x, tokens, tau, k, got):
    for i, (row, token, t) in enumerate(rows_of(x, tokens, tau)):
        lp, h, ids, top = O.score_row(row, token, t, k)
        close(got.logprobs.reshape(-1)[i].item(), lp, REL * (1 + abs(lp)), f"logprob of row {i}")
        if got.entropy is not None:
            close(got.entropy.reshape(-1)[i].item(), h, 4 * REL * (1 + abs(h)), f"entropy of row {i}")
        if k:
            assert got.top_tokens.reshape(-1, k)[i].tolist() == ids.tolist(), f"row {i}"
            close(got.top_logprobs.detach().reshape(-1, k)[i].cpu().numpy(), top, REL * (1 + np.abs(top)), f"list of row {i}")


def check_grad(x, tokens, tau, ids, ups, d, dtype):
    k = 0 if ids is None else ids.shape[-1]
    for i, (row, token, t) in enumerate(rows_of(x, tokens, tau)):
        up = [0.0 if u is None else u.reshape(-1)[i].double().item() for u in ups[:2]]
        top = np.zeros(k) if ups[2] is None else ups[2].reshape(-1, k)[i].double().cpu().numpy()
        at = np.full(k, -1) if ids is None else ids.reshape(-1, k)[i].cpu().numpy()
        want, mag = O.score_row_grad(row, token, t, at, *up, top)
        got = d.reshape(-1, d.shape[-1])[i].double().cpu().numpy()
        tol = 4 * REL * mag + torch.finfo(dtype).eps / 2 * np.abs(want) + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps + FLUSH
        close(got, want, tol, f"gradient of row {i}")


@pytest.mark.gpu
@pytest.mark.parametrize("shape,V,dtype,k,tau", [
    ((1, 1), 1, torch.float32, 1, False),
    ((3,), 2, torch.bfloat16, 3, True),
    ((2, 3), 37, torch.float16, 5, True),
    ((4, 5), 1001, torch.bfloat16, 20, False),
    ((7,), 8191, torch.float32, 128, True),
    ((3, 3), 32003, torch.float16, 64, True),
    ((1, 2), 151936, torch.bfloat16, 8, True),
    ((5, 40), 4099, torch.float32, 0, True),
    ((2, 3), 70001, torch.float32, 33, False),
    ((600,), 5000, torch.bfloat16, 2, True),
])
def test_against_definition(shape, V, dtype, k, tau, cuda_device):
    from autoindexer_b200 import read_status, token_logprobs

    x, tokens, temp = (t.to(cuda_device) for t in make(shape, V, dtype, V + len(shape)))
    temp = temp if tau else None
    got = token_logprobs(x, tokens, temp, top_k=k, entropy=True)
    assert got.logprobs.shape == tokens.shape and got.logprobs.dtype == torch.float32
    assert read_status(cuda_device) == 0
    check(x, tokens, temp, k, got)
    again = token_logprobs(x, tokens, temp, top_k=k, entropy=True)
    assert all(a is b is None or torch.equal(a, b) for a, b in zip(got, again))
    alone = token_logprobs(x, tokens, temp)
    assert torch.equal(alone.logprobs, got.logprobs) and alone[1:] == (None, None, None)


@pytest.mark.gpu
@pytest.mark.parametrize("ups", ["all", "logprob", "entropy", "top", "none"])
@pytest.mark.parametrize("shape,V,dtype,k", [
    ((3,), 5, torch.float32, 7),
    ((2, 3), 1003, torch.bfloat16, 9),
    ((2, 2), 33001, torch.float16, 128),
    ((1, 5), 151936, torch.float32, 1),
    ((300, 3), 513, torch.bfloat16, 3),
])
def test_gradient(shape, V, dtype, k, ups, cuda_device):
    from autoindexer_b200 import token_logprobs

    x, tokens, tau = (t.to(cuda_device) for t in make(shape, V, dtype, 7 * V))
    x.requires_grad_()
    out = token_logprobs(x, tokens, tau, top_k=k, entropy=True)
    g = torch.Generator().manual_seed(3)
    gl, gh, gt = (torch.randn(s, generator=g).to(cuda_device) for s in (shape, shape, (*shape, k)))
    gl.view(-1)[0] = gh.view(-1)[0] = 0
    gt.view(-1, k)[0] = 0  # a row without any upstream gradient
    use = {"all": (gl, gh, gt), "logprob": (gl, None, None), "entropy": (None, gh, None), "top": (None, None, gt),
           "none": (None, None, None)}[ups]
    outs = (out.logprobs, out.entropy, out.top_logprobs)
    assert not out.top_tokens.requires_grad
    if ups == "none":
        d = torch.autograd.grad([out.logprobs], x, [torch.zeros_like(gl)])[0]
        assert not bool(d.any())
        return
    d = torch.autograd.grad([o for o, u in zip(outs, use) if u is not None], x, [u for u in use if u is not None])[0]
    assert d.dtype == dtype and d.shape == x.shape
    check_grad(x, tokens, tau, out.top_tokens, use, d, dtype)


@pytest.mark.gpu
def test_gradient_against_differences(cuda_device):
    """Central differences of the definition in 64 bits along random directions."""
    from autoindexer_b200 import token_logprobs

    x, tokens, tau = make((2, 3), 301, torch.float32, 5)
    k, step = 6, 1e-5
    g = torch.Generator().manual_seed(1)
    ups = [torch.randn(2, 3, generator=g), torch.randn(2, 3, generator=g), torch.randn(2, 3, k, generator=g)]
    xd = x.to(cuda_device).requires_grad_()
    out = token_logprobs(xd, tokens.to(cuda_device), tau.to(cuda_device), top_k=k, entropy=True)
    d = torch.autograd.grad([out.logprobs, out.entropy, out.top_logprobs], xd, [u.to(cuda_device) for u in ups])[0].double().cpu()

    def f(y):
        total = 0.0
        for i, (row, token, t) in enumerate(rows_of(y, tokens, tau)):
            lp, h, _, top = O.score_row(row, token, t, k)
            if token >= 0:
                total += lp * ups[0].view(-1)[i].item() + h * ups[1].view(-1)[i].item() + float(top @ ups[2].view(-1, k)[i].double().numpy())
        return total

    for _ in range(5):
        way = torch.randn(x.shape, generator=g, dtype=torch.float64)
        slope = (f(x.double() + step * way) - f(x.double() - step * way)) / (2 * step)
        # (the difference's own error: step^2 times a third derivative below 1e2, and 1e-15 / step of rounding)
        assert abs(slope - float((d * way).sum())) < 1e-4 * (1 + abs(slope))


def odd_rows(V):
    """Rows that masks, ties and order make awkward, and how they are called."""
    n = torch.arange(V, dtype=torch.float32)
    low = torch.finfo(torch.float32).min
    rows = {
        "all masked": torch.full((V,), -INF),
        "one word": torch.full((V,), -INF).index_fill_(0, torch.tensor([V // 2]), -7.0),
        "few words": torch.where(n % (V // 3 + 1) == 1, n / V, -INF),
        "lowest values": torch.full((V,), low),
        "lowest and one": torch.full((V,), low).index_fill_(0, torch.tensor([3]), 0.5),
        "largest apart": torch.where(n < 2, 1e38 * (1 - n), -1e38),
        "constant": torch.zeros(V),
        "signed zeros": torch.where(n % 2 == 0, -0.0, 0.0),
        "rising": n / 64,
        "falling": -n / 64,
        "two values": torch.where(n % 3 == 0, 1.0, 0.0),
        "peaked": torch.where(n == V - 1, 80.0, -20.0),
    }
    return rows


@pytest.mark.gpu
@pytest.mark.parametrize("V", [40, 9001, 140003])
def test_awkward_rows(V, cuda_device):
    from autoindexer_b200 import read_status, token_logprobs

    rows = odd_rows(V)
    x = torch.stack(list(rows.values())).to(cuda_device).requires_grad_()
    tokens = torch.full((len(rows),), V // 2, device=cuda_device)
    k = 40
    out = token_logprobs(x, tokens, top_k=k, entropy=True)
    check(x, tokens, None, k, out)
    ups = [torch.ones_like(out.logprobs), torch.ones_like(out.logprobs), torch.ones_like(out.top_logprobs)]
    d = torch.autograd.grad(out[:3], x, ups)[0]
    check_grad(x, tokens, None, out.top_tokens, ups, d, torch.float32)
    assert read_status(cuda_device) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V", [33, 20001])
def test_nan_and_infinity(V, dtype, cuda_device):
    """A row with a NaN or a +inf is NaN, its neighbours are not; padding rows
    may hold anything."""
    from autoindexer_b200 import token_logprobs

    x, tokens, _ = make((6,), V, dtype, 1)
    x[1, V - 1], x[2, 0], x[3], x[5] = float("nan"), INF, float("nan"), float("nan")
    tokens[5] = -100
    x, tokens = x.to(cuda_device).requires_grad_(), tokens.to(cuda_device)
    out = token_logprobs(x, tokens, top_k=4, entropy=True)
    check(x, tokens, None, 4, out)
    ups = [torch.ones_like(out.logprobs), torch.ones_like(out.logprobs), torch.ones_like(out.top_logprobs)]
    d = torch.autograd.grad(out[:3], x, ups)[0]
    check_grad(x, tokens, None, out.top_tokens, ups, d, dtype)
    assert not bool(d[5].any())


@pytest.mark.gpu
def test_tokens_and_temperatures_out_of_range(cuda_device):
    from autoindexer_b200 import read_status, token_logprobs

    x, tokens, _ = (t.to(cuda_device) for t in make((5,), 300, torch.float32, 2))
    plain = token_logprobs(x, tokens)
    tokens[0], tokens[1] = -1, -(2 ** 40)
    assert token_logprobs(x, tokens).logprobs[:2].tolist() == [0, 0] and read_status(cuda_device) == 0
    tokens[2], tokens[3] = 300, 2 ** 32 + 1
    got = token_logprobs(x, tokens, top_k=2, entropy=True)
    assert read_status(cuda_device) == -2
    assert got.logprobs[:4].tolist() == [0] * 4 and got.top_tokens[:4].eq(-1).all()
    assert got.logprobs[4] == plain.logprobs[4]
    _, tokens, _ = (t.to(cuda_device) for t in make((5,), 300, torch.float32, 2))
    tau = torch.tensor([0.0, -1.0, float("nan"), 1.0, 1.0], device=cuda_device)
    assert torch.equal(token_logprobs(x, tokens, tau).logprobs, plain.logprobs)
    assert read_status(cuda_device) == -2
    # Far temperatures: the most likely words share the mass, or all do.
    tau = torch.tensor([1e-45, 1e-30, 1e30, INF, 1.0], device=cuda_device)
    got = token_logprobs(x, x.argmax(-1), tau, entropy=True)
    assert got.logprobs[:2].tolist() == [0, 0] and got.entropy[:2].tolist() == [0, 0]
    close(got.logprobs[2:4].cpu().numpy(), -np.log(300), 1e-4, "uniform")
    assert read_status(cuda_device) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("lay", ["padded", "off", "transposed", "expanded", "stepped"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_strides(lay, dtype, cuda_device):
    from autoindexer_b200 import token_logprobs

    x, tokens, tau = (t.to(cuda_device) for t in make((3, 4), 1003, dtype, 12))
    base = None
    if lay == "padded":
        base = torch.full((3, 4, 1024), float("nan"), dtype=dtype, device=cuda_device)
        base[..., :1003] = x
        view = base[..., :1003]
    elif lay == "off":
        base = torch.full((3, 4, 1010), float("nan"), dtype=dtype, device=cuda_device)
        base[..., 5:1008] = x
        view = base[..., 5:1008]
    elif lay == "transposed":
        view = x.transpose(0, 1).contiguous().transpose(0, 1)
    elif lay == "expanded":
        x = x[:, :1].expand(3, 4, 1003)
        view = x
    else:
        base = torch.zeros(3, 4, 2006, dtype=dtype, device=cuda_device)
        base[..., ::2] = x
        view = base[..., ::2]
    view = view.detach().requires_grad_()
    out = token_logprobs(view, tokens, tau, top_k=3, entropy=True)
    check(x, tokens, tau, 3, out)
    ups = [torch.ones_like(out.logprobs), torch.ones_like(out.logprobs), torch.ones_like(out.top_logprobs)]
    d = torch.autograd.grad(out[:3], view, ups)[0]
    check_grad(x, tokens, tau, out.top_tokens, ups, d, dtype)


@pytest.mark.gpu
def test_offsets_past_31_bits(cuda_device):
    from autoindexer_b200 import token_logprobs

    far, V = 2 ** 31 + 5, 1000
    base = torch.empty(far + V, dtype=torch.bfloat16, device=cuda_device)
    x = base.as_strided((2, 1, V), (far, V, 1))
    src, tokens, _ = (t.to(cuda_device) for t in make((2, 1), V, torch.bfloat16, 4))
    x.copy_(src)
    x.requires_grad_()
    out = token_logprobs(x, tokens, top_k=3, entropy=True)
    check(src, tokens, None, 3, out)
    ups = [torch.ones_like(out.logprobs), None, None]
    d = torch.autograd.grad(out.logprobs, x, ups[0])[0]
    check_grad(src, tokens, None, out.top_tokens, ups, d, torch.bfloat16)


@pytest.mark.gpu
@pytest.mark.parametrize("shape,V,k", [((2,), 50001, 5), ((40, 20), 700, 0)])
def test_captured_graph_and_another_stream(shape, V, k, cuda_device):
    from autoindexer_b200 import token_logprobs

    x, tokens, tau = (t.to(cuda_device) for t in make(shape, V, torch.bfloat16, 8))
    other = make(shape, V, torch.bfloat16, 9)
    x.requires_grad_()
    g = torch.randn(shape, device=cuda_device)

    def step():
        out = token_logprobs(x, tokens, tau, top_k=k, entropy=True)
        d = torch.autograd.grad([out.logprobs, out.entropy], x, [g, g])
        return [o.detach() for o in out if o is not None] + list(d)

    step()
    torch.cuda.synchronize(cuda_device)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for values in (None, other):
        if values is not None:
            for a, b in zip((x.data, tokens, tau), values):
                a.copy_(b)
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
def test_saved_tensors_through_hooks(cuda_device):
    """Hooks may bring saved tensors back with other strides."""
    from autoindexer_b200 import token_logprobs

    x, tokens, tau = (t.to(cuda_device) for t in make((3, 4), 500, torch.bfloat16, 3))
    wide = torch.zeros(3, 4, 520, dtype=torch.bfloat16, device=cuda_device)
    wide[..., :500] = x
    a, b = wide[..., :500].detach().requires_grad_(), x.clone().requires_grad_()
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t.cpu(), lambda t: t.to(cuda_device)):
        out = token_logprobs(a, tokens, tau, top_k=2, entropy=True)
        got = torch.autograd.grad(out.logprobs.sum() + out.top_logprobs.sum(), a)[0]
    out = token_logprobs(b, tokens, tau, top_k=2, entropy=True)
    assert torch.equal(got, torch.autograd.grad(out.logprobs.sum() + out.top_logprobs.sum(), b)[0])


@pytest.mark.gpu
def test_gradients_that_do_not_exist(cuda_device):
    from autoindexer_b200 import token_logprobs

    x, tokens, tau = (t.to(cuda_device) for t in make((3,), 50, torch.float32, 3))
    with pytest.raises(RuntimeError, match="temperature"):
        token_logprobs(x, tokens, tau.clone().requires_grad_())
    with torch.no_grad():
        token_logprobs(x, tokens, tau.clone().requires_grad_())
    with forward_ad.dual_level(), pytest.raises(RuntimeError, match="forward"):
        token_logprobs(forward_ad.make_dual(x, torch.ones_like(x)), tokens, tau)
    y = x.clone().requires_grad_()
    d = torch.autograd.grad(token_logprobs(y, tokens).logprobs.sum(), y, create_graph=True)[0]
    with pytest.raises(RuntimeError, match="once_differentiable|does not require grad"):
        d.sum().backward()
    out = token_logprobs(y, tokens)
    y.data.add_(0)  # (unseen by autograd)
    with torch.no_grad():
        y.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.logprobs.sum().backward()


def refusals(x, tokens, tau):
    return [
        (ValueError, (x[0, 0], tokens)),
        (ValueError, (x[None], tokens)),
        (ValueError, (x[:, :0], tokens[:, :0])),
        (ValueError, (x, tokens[:, :1])),
        (ValueError, (x, tokens, tau[:1])),
        (ValueError, (x, tokens, None, -1)),
        (ValueError, (x, tokens, None, 129)),
        (TypeError, (x, tokens.int())),
        (TypeError, (x.double(), tokens)),
        (TypeError, (x, tokens, tau.double())),
    ]


@pytest.mark.gpu
def test_refusals(cuda_device):
    from autoindexer_b200 import token_logprobs

    x, tokens, tau = (t.to(cuda_device) for t in make((2, 3), 50, torch.bfloat16, 0))
    for error, args in refusals(x, tokens, tau) + [(RuntimeError, (x, tokens.cpu())), (RuntimeError, (x, tokens, tau.cpu()))]:
        with pytest.raises(error):
            token_logprobs(*args)


def test_cpu_tensors_are_refused():
    from autoindexer_b200 import token_logprobs

    x, tokens, _ = make((2, 3), 50, torch.bfloat16, 0)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        token_logprobs(x, tokens)


def test_c_abi_refusals():
    from autoindexer_b200 import _lib

    L = _lib.lib()

    def args(**over):
        a = _lib.AiScoreArgs()
        a.batch, a.seq_len, a.vocab, a.dtype, a.top_k = 2, 3, 100, _lib.DTYPE_BF16, 4
        a.logits = a.tokens = a.logprobs = a.top_logprobs = a.top_tokens = a.row_stats = 256
        for n, v in over.items():
            setattr(a, n, v)
        return a

    bad = (("batch", 0, 2), ("seq_len", 0, 2), ("vocab", 0, 2), ("vocab", 2 ** 31 - 1, 2), ("top_k", 129, 2), ("top_k", -1, 2),
           ("batch", 2 ** 30, 2), ("dtype", 3, 4), ("logits", None, 1), ("tokens", None, 1), ("stride_t", -1, 5),
           ("logits", 257, 6), ("row_stats", 264, 6))
    assert L.ai_token_logprobs(None, None) == 1 and L.ai_token_logprobs_bwd(None, None) == 1
    for field, value, code in bad + (("logprobs", None, 1), ("top_tokens", None, 1), ("top_logprobs", None, 1)):
        assert L.ai_token_logprobs(ctypes.byref(args(**{field: value})), None) == code, field

    def bwd(fwd, **over):
        g = _lib.AiScoreBwdArgs()
        g.fwd = fwd
        g.dlogits = g.g_logprobs = g.g_top = 256
        for n, v in over.items():
            setattr(g, n, v)
        return ctypes.byref(g)

    for field, value, code in bad + (("row_stats", None, 1), ("top_tokens", None, 1)):
        assert L.ai_token_logprobs_bwd(bwd(args(**{field: value})), None) == code, field
    for field, value, code in (("dlogits", None, 1), ("dstride_b", -1, 5), ("dlogits", 255, 6)):
        assert L.ai_token_logprobs_bwd(bwd(args(), **{field: value}), None) == code, field


def test_oracle_gradient_follows_its_values():
    """The oracle's gradient against differences of its own values."""
    rng = np.random.default_rng(0)
    x, k, step = rng.normal(size=40) * 2, 5, 1e-6
    _, _, ids, _ = O.score_row(x, 7, 0.7, k)
    g, h, t = 0.3, -1.1, rng.normal(size=k)
    d, _ = O.score_row_grad(x, 7, 0.7, ids, g, h, t)
    for v in (0, 7, int(ids[0])):
        def f(y):
            lp, e, _, top = O.score_row(y, 7, 0.7, k)
            return g * lp + h * e + top @ t
        e = np.eye(40)[v] * step
        assert abs((f(x + e) - f(x - e)) / (2 * step) - d[v]) < 1e-7
