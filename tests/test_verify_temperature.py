"""``verify_draft`` over the whole range of temperatures: from subnormal ones,
where the distribution is the largest logit's, through ordinary ones to
infinity, where it is flat.

Tolerance: as in ``test_verify.py``.  A weight is ``2^((x - max) c)``: the
difference is rounded once (2^-24 of itself), ``c = log2(e) / tau`` once and
the product once, so the argument of a weight that matters (above 2^-29 of the
largest) is off by less than 30 * 3 * 2^-24, the weight by 4e-6 of itself."""

import numpy as np
import pytest
import torch

from test_verify import _case, _verify


@pytest.mark.gpu
@pytest.mark.parametrize("tau", [1e-1, 1e-3, 1e-4, 1e-6, 5e-8, 1e-8, 1e-10, 1e-20, 1e-38, 1e-40, 1e-45, 1e4, 1e20, 3e38])
@pytest.mark.parametrize("dtype,draft,V", [(torch.float32, True, 4099), (torch.bfloat16, True, 20000),
                                           (torch.float16, False, 5003), (torch.float32, False, 1001)])
def test_temperatures(tau, dtype, draft, V, cuda_device):
    """Logits of up to some hundreds; the largest of a row stands alone, so
    that the definition has no near ties at small temperatures."""
    from autoindexer_b200 import read_status, verify_draft

    B, L = 5, 3
    t, x, u, e, d, n, _ = _case(B, L, V, dtype, draft, 23, cuda_device, spread=40.0)
    top = t.float().argmax(-1)
    t.scatter_(-1, top[..., None], t.amax(-1, keepdim=True) + 8)
    if draft:
        dtop = d.float().argmax(-1)
        d.scatter_(-1, dtop[..., None], d.amax(-1, keepdim=True) + 8)
    x[0] = top[0, :L]        # drafted where the target is certain: all accepted
    x[1, 0], n[1] = top[1, 0], L
    if draft:
        d[0] = t[0, :L]
        d[1, 0] = t[1, 0]
    tau_t = torch.full((B,), tau, device=cuda_device)
    got = verify_draft(t, x, u, e, d, n, tau_t)
    assert read_status(cuda_device) == 0
    assert all(torch.isfinite(got[2]).flatten().tolist())
    _verify(t, x, u, e, d, n, tau_t, got)
    if tau < 1e-2:
        a, said = got[0].tolist(), got[1].tolist()
        assert a[0] == L and said[0][:L] == top[0, :L].tolist() and said[0][L] == int(top[0, L])
        assert a[1] >= 1


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("tau", [1e-6, 1e-8, 1e-12, 1e-39])
def test_a_tiny_temperature_decodes_as_zero_does(tau, dtype, cuda_device):
    """Many rows whose largest logits differ in size (what the offset of the
    exponent depends on): the tokens are those of temperature 0."""
    from autoindexer_b200 import verify_draft

    B, V = 64, 1777
    g = torch.Generator().manual_seed(3)
    t = 3 * torch.randn(B, 2, V, generator=g)
    t.scatter_(-1, t.argmax(-1, keepdim=True), torch.linspace(20, 300, 2 * B).reshape(B, 2, 1))
    t = t.to(dtype).to(cuda_device)
    x = t[:, :1].float().argmax(-1)
    x[::3] = (x[::3] + 1) % V
    u = torch.rand(B, 1, generator=g).to(cuda_device)
    e = torch.empty(B, V).exponential_(generator=g).clamp_min(1e-8).to(cuda_device)
    want = verify_draft(t, x, u, e, temperature=torch.zeros(B, device=cuda_device))
    got = verify_draft(t, x, u, e, temperature=torch.full((B,), tau, device=cuda_device))
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    assert torch.all(got[2] == 0)


@pytest.mark.gpu
def test_masked_words_at_the_ends_of_the_range(cuda_device):
    """-inf stays without weight, and a flat distribution (infinite
    temperature) is flat over the other words."""
    from autoindexer_b200 import verify_draft

    V = 1000
    t = torch.full((3, 1, V), -float("inf"), device=cuda_device)
    t[:, :, 100:200] = torch.linspace(-80, 80, 100, device=cuda_device)
    e = torch.ones(3, V, device=cuda_device)
    e[:, 150] = 0.5
    empty = torch.zeros(3, 0, device=cuda_device)
    tau = torch.tensor([1e-30, 1.0, float("inf")], device=cuda_device)
    a, said, logp = verify_draft(t, empty.long(), empty, e, temperature=tau)
    assert a.tolist() == [0, 0, 0] and said[:, 0].tolist() == [199, 199, 150]
    assert abs(float(logp[2, 0]) + np.log(100)) < 1e-5 and float(logp[0, 0]) == 0
