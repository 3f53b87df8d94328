"""Verification of drafted tokens (``verify_draft``) against the definition in
64 bits, its distribution, and refusals.

Tolerances: float32 probabilities carry a few roundings of 2^-24 and the
rounding of ``(x - max) / tau`` (at most 2^-23 of an argument that matters
below 20), so a decision nearer than 2e-5 (relative) to its threshold may go
either way; the checks accept only those."""

import ctypes

import numpy as np
import pytest
import torch

from oracle import operator_oracle as O

TOL = 2e-5


def _case(B, L, V, dtype, draft, seed, device, spread=2.5):
    g = torch.Generator().manual_seed(seed)
    target = spread * torch.randn(B, L + 1, V, generator=g)
    dl = target[:, :L] + 0.7 * torch.randn(B, L, V, generator=g)
    race = torch.empty(B, L, V).exponential_(generator=g)
    tau = 0.5 + torch.rand(B, generator=g)
    tau[1::3] = 0.0
    tokens = (torch.softmax(dl, -1) / race).argmax(-1) if L else torch.zeros(B, 0, dtype=torch.long)
    u = torch.rand(B, L, generator=g)
    noise = torch.empty(B, V).exponential_(generator=g).clamp_min(1e-8)
    n = torch.randint(0, L + 1, (B,), generator=g).int()
    n[0] = L
    to = lambda x: x.to(device)  # noqa: E731
    return to(target.to(dtype)), to(tokens), to(u), to(noise), to(dl.to(dtype)) if draft else None, to(n), to(tau)


def _verify(target, tokens, u, noise, draft, n, tau, got):
    a, said, logp = (x.cpu().numpy() for x in got)
    B, L = tokens.shape
    for b in range(B):
        wrong = O.verify_check(target[b].double().cpu().numpy(), None if draft is None else draft[b].double().cpu().numpy(),
                               tokens[b].cpu().numpy(), u[b].double().cpu().numpy(), noise[b].double().cpu().numpy(),
                               1.0 if tau is None else float(tau[b]), L if n is None else int(n[b]), int(a[b]), said[b],
                               logp[b], TOL)
        assert not wrong, f"sequence {b}: {wrong}"


@pytest.mark.gpu
@pytest.mark.parametrize("B,L,V,dtype,draft", [
    (1, 1, 1, torch.float32, True),
    (1, 0, 37, torch.bfloat16, True),
    (3, 1, 2, torch.float32, False),
    (5, 3, 1001, torch.bfloat16, True),
    (4, 2, 4099, torch.float16, True),
    (7, 4, 32003, torch.bfloat16, False),
    (2, 5, 151936, torch.bfloat16, True),
    (1, 7, 151936, torch.float32, True),
    (33, 1, 20000, torch.float32, True),
    (2, 64, 500, torch.float16, True),
])
def test_against_definition(B, L, V, dtype, draft, cuda_device):
    from autoindexer_b200 import read_status, verify_draft

    t, x, u, e, d, n, tau = _case(B, L, V, dtype, draft, B + L + V, cuda_device)
    got = verify_draft(t, x, u, e, d, n, tau)
    assert read_status(cuda_device) == 0
    assert got[0].dtype == torch.int32 and got[1].dtype == torch.int64 and got[2].dtype == torch.float32
    _verify(t, x, u, e, d, n, tau, got)
    again = verify_draft(t, x, u, e, d, n, tau)
    assert all(torch.equal(p, q) for p, q in zip(got, again))
    _verify(t, x, u, e, d, None, None, verify_draft(t, x, u, e, d))


@pytest.mark.gpu
@pytest.mark.parametrize("pad", [1, 8])
def test_strided_logits(pad, cuda_device):
    """Rows of a padded vocabulary (off and on 16-byte boundaries)."""
    from autoindexer_b200 import verify_draft

    t, x, u, e, d, n, tau = _case(3, 2, 5003, torch.bfloat16, True, 11, cuda_device)
    want = verify_draft(t, x, u, e, d, n, tau)
    wt = torch.full((3, 3, 5003 + pad), float("nan"), dtype=t.dtype, device=cuda_device)
    wd = torch.full((3, 2, 5003 + 3 * pad), float("nan"), dtype=t.dtype, device=cuda_device)
    wt[..., :5003], wd[..., pad:5003 + pad] = t, d
    got = verify_draft(wt[..., :5003], x, u, e, wd[..., pad:5003 + pad], n, tau)
    _verify(t, x, u, e, d, n, tau, got)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.gpu
def test_masked_logits_ties_and_equal_distributions(cuda_device):
    from autoindexer_b200 import verify_draft

    B, V = 6, 3000
    inf = float("inf")
    t, x, u, e, d, _, _ = _case(B, 1, V, torch.float32, True, 5, cuda_device)
    t[0, :, :], d[0] = -inf, -inf                 # a row without any word: token 0, nothing accepted
    t[1, :, 17:] = -inf                           # a vocabulary mask; the drafted token is outside it
    x[1], x[2] = 900, 5
    t[2], d[2] = d[2].clone(), d[2].clone()       # p = q: u < 1 accepts always
    u[2] = 1 - 2.0 ** -24
    t[3, 0, :], d[3] = 0.0, 0.0                   # flat: ties everywhere
    t[3, 0, 1000:] = -1.0
    u[3], x[3] = 0.99999, 2999
    e[3] = 1.0
    t[4, 0], t[4, 1] = 1.0, 1.0                   # greedy over equal logits: the lowest index
    x[4] = 0
    t[5, 0, 40] = t[5, 0, 41] = 100.0
    x[5] = 41
    tau = torch.tensor([1.0, 1.0, 1.0, 1.0, 0.0, 0.0], device=cuda_device)
    a, said, logp = (y.cpu() for y in verify_draft(t, x, u, e, d, temperature=tau))
    assert a.tolist()[:2] == [0, 0] and int(said[0, 0]) == 0 and int(said[1, 0]) < 17
    assert int(a[2]) == 1
    assert int(a[3]) == 0 and int(said[3, 0]) == 0
    assert int(a[4]) == 1 and said[4].tolist() == [0, 0]
    assert int(a[5]) == 0 and said[5].tolist() == [40, -1]
    _verify(t[1:], x[1:], u[1:], e[1:], d[1:], None, tau[1:], (a[1:], said[1:], logp[1:]))


@pytest.mark.gpu
def test_token_outside_the_vocabulary(cuda_device):
    from autoindexer_b200 import read_status, verify_draft

    t, x, u, e, d, _, _ = _case(3, 2, 700, torch.bfloat16, False, 9, cuda_device)
    x[0, 1], x[1, 0], x[2, 0] = 700, -1, 2 ** 32 + 1
    u[0, 0] = 0.0
    read_status(cuda_device)
    got = verify_draft(t, x, u, e)
    assert read_status(cuda_device) == -2
    assert got[0].tolist() == [1, 0, 0]
    _verify(t, x, u, e, None, None, None, got)


@pytest.mark.gpu
@pytest.mark.parametrize("draft", [True, False])
def test_tokens_follow_the_target_distribution(draft, cuda_device):
    """The first token of 20,000 sequences follows the target's distribution
    whatever was drafted: a chi-square over 8 words (7 degrees of freedom)
    stays below 40 (a probability of 1e-6)."""
    from autoindexer_b200 import verify_draft

    B, V = 20000, 8
    g = torch.Generator().manual_seed(77)
    p = torch.tensor([2.0, 0.5, -1.0, 1.2, 0.0, -0.3, 1.9, 0.4])
    q = torch.tensor([0.0, 1.5, 0.3, -1.0, 1.1, 0.2, 0.1, 0.9])
    t = p.expand(B, 2, V).contiguous().to(cuda_device)
    d = q.expand(B, 1, V).contiguous().to(cuda_device) if draft else None
    x = torch.multinomial(torch.softmax(q, 0), B, replacement=True, generator=g)[:, None].to(cuda_device)
    u = torch.rand(B, 1, generator=g).to(cuda_device)
    e = torch.empty(B, V).exponential_(generator=g).clamp_min(1e-9).to(cuda_device)
    a, said, _ = verify_draft(t, x, u, e, d)
    seen = np.bincount(said[:, 0].cpu().numpy(), minlength=V)
    want = torch.softmax(p.double(), 0).numpy() * B
    assert float(((seen - want) ** 2 / want).sum()) < 40
    assert 0 < int((a == 0).sum()) < B


@pytest.mark.gpu
def test_refusals(cuda_device):
    from autoindexer_b200 import verify_draft

    t, x, u, e, d, n, tau = _case(2, 3, 100, torch.bfloat16, True, 1, cuda_device)
    for error, args in [
        (ValueError, (t[0], x, u, e)),
        (ValueError, (t, x[:, :2], u, e)),
        (ValueError, (t, x, u[:1], e)),
        (ValueError, (t, x, u, e[:, :50])),
        (ValueError, (t, x, u, e, d[:, :2])),
        (ValueError, (t, x, u, e, d, n[:1])),
        (ValueError, (t, x, u, e, d, n, tau[:1])),
        (ValueError, (t.new_zeros(1, 66, 4), x.new_zeros(1, 65), u.new_zeros(1, 65), e.new_ones(1, 4))),
        (TypeError, (t, x.int(), u, e)),
        (TypeError, (t, x, u.double(), e)),
        (TypeError, (t, x, u, e, d.float())),
        (TypeError, (t, x, u, e, d, n.long())),
        (TypeError, (t.double(), x, u, e)),
        (RuntimeError, (t, x.cpu(), u, e)),
        (RuntimeError, (t.cpu(), x, u, e)),
    ]:
        with pytest.raises(error):
            verify_draft(*args)


def test_oracle_check_finds_planted_mistakes():
    """The 64-bit check accepts the definition's results and refuses others."""
    rng = np.random.default_rng(0)
    V, L = 50, 2
    target, draft = rng.normal(size=(L + 1, V)) * 2, rng.normal(size=(L, V)) * 2
    tokens, u, noise = np.array([3, 4]), np.array([0.0, 0.999999]), rng.exponential(size=V)
    p, q = O.softmax(target[1], 1.0), O.softmax(draft[1], 1.0)
    draft[1, 4] += 8  # drafted far too often: refused
    q = O.softmax(draft[1], 1.0)
    nxt = int((np.maximum(p - q, 0) / noise).argmax())
    said = np.array([3, nxt, -1])
    logp = np.array([np.log(O.softmax(target[0], 1.0)[3]), np.log(p[nxt]), 0.0])
    args = (target, draft, tokens, u, noise, 1.0, 2)
    assert O.verify_check(*args, 1, said, logp, TOL) == ""
    assert O.verify_check(*args, 2, np.array([3, 4, nxt]), logp, TOL) != ""
    assert O.verify_check(*args, 1, np.array([3, (nxt + 1) % V, -1]), logp, TOL) != ""
    assert O.verify_check(*args, 1, said, logp + 1e-3, TOL) != ""
    assert O.verify_check(*args, 0, np.array([nxt, -1, -1]), logp, TOL) != ""


def test_c_abi_refusals():
    from autoindexer_b200 import _lib

    L = _lib.lib()

    def args(**over):
        a = _lib.AiVerifyArgs()
        a.batch, a.n_draft, a.vocab, a.dtype = 2, 3, 100, _lib.DTYPE_BF16
        a.target = a.tokens = a.uniforms = a.noise = a.accepted = a.out_tokens = a.logprobs = 256
        for n, v in over.items():
            setattr(a, n, v)
        return a

    assert L.ai_verify_draft(None, None) == 1
    for field, value, code in (("batch", 0, 2), ("n_draft", 65, 2), ("vocab", 0, 2), ("batch", 10000, 2), ("dtype", 3, 4),
                               ("noise", None, 1), ("tokens", None, 1), ("target_stride_t", -1, 5)):
        assert L.ai_verify_draft(ctypes.byref(args(**{field: value})), None) == code, field
    assert L.ai_verify_draft(ctypes.byref(args()), None) == 8  # no workspace
    n = ctypes.c_size_t(0)
    assert L.ai_verify_draft_workspace(ctypes.byref(args()), ctypes.byref(n)) == 0 and n.value > 0
