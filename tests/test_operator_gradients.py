"""What the operators do with inputs that carry gradients they cannot give:
none is lost silently."""

import pytest
import torch
from torch.autograd import forward_ad

from test_head_norm import _inputs
from test_paged import _cache
from test_verify import _case


@pytest.mark.gpu
@pytest.mark.parametrize("which", [0, 1, 2, 3])
def test_norm_refuses_forward_mode(which, cuda_device):
    from autoindexer_b200 import qk_norm_rope

    ins = list(_inputs(2, 5, 4, 2, 64, torch.float32, 1, cuda_device))
    want = qk_norm_rope(*ins)
    with forward_ad.dual_level():
        got = qk_norm_rope(*ins)  # without tangents nothing is refused
        assert all(torch.equal(x, y) for x, y in zip(got, want))
        ins[which] = forward_ad.make_dual(ins[which], torch.ones_like(ins[which]))
        for grad_mode in (torch.enable_grad(), torch.no_grad()):
            with grad_mode, pytest.raises(RuntimeError, match="forward"):
                qk_norm_rope(*ins)


def _attention(device):
    lens = [9, 20]
    q, kp, vp, prefix, table = _cache(2, 1, 4, 2, 64, 16, 20, lens, torch.float32, 6, device)
    return q, kp, vp, prefix, 20, table, torch.tensor(lens, dtype=torch.int32, device=device)


@pytest.mark.gpu
@pytest.mark.parametrize("which", [0, 1, 2])
def test_attention_refuses_the_backward(which, cuda_device):
    """Inputs that require a gradient are taken (a model may run outside
    ``no_grad``) and give the same values; a backward through them raises."""
    from autoindexer_b200 import shared_prefix_attention

    args = list(_attention(cuda_device))
    want, wlse = shared_prefix_attention(*args, return_lse=True)
    assert not want.requires_grad
    args[which] = args[which].detach().requires_grad_()
    out, lse = shared_prefix_attention(*args, return_lse=True)
    assert torch.equal(out, want) and torch.equal(lse, wlse)
    alone = shared_prefix_attention(*args)
    assert torch.equal(alone, want)
    for x in (out, lse, alone):
        with pytest.raises(RuntimeError, match="shared_prefix_attention has no backward"):
            x.sum().backward()
    with torch.no_grad():
        assert not shared_prefix_attention(*args).requires_grad
    with torch.inference_mode():
        assert torch.equal(shared_prefix_attention(*args), want)


@pytest.mark.gpu
def test_attention_refuses_forward_mode(cuda_device):
    from autoindexer_b200 import shared_prefix_attention

    args = list(_attention(cuda_device))
    with forward_ad.dual_level():
        shared_prefix_attention(*args)
        args[0] = forward_ad.make_dual(args[0], torch.ones_like(args[0]))
        with pytest.raises(RuntimeError, match="forward"):
            shared_prefix_attention(*args)


@pytest.mark.gpu
def test_verification_refuses_the_backward(cuda_device):
    from autoindexer_b200 import verify_draft

    t, x, u, e, d, n, tau = _case(3, 2, 100, torch.float32, True, 1, cuda_device)
    want = verify_draft(t, x, u, e, d, n, tau)
    got = verify_draft(t.requires_grad_(), x, u, e, d, n, tau)
    assert all(torch.equal(p, q) for p, q in zip(got, want))
    with pytest.raises(RuntimeError, match="verify_draft has no backward"):
        got[2].sum().backward()
    with forward_ad.dual_level():
        with pytest.raises(RuntimeError, match="forward"):
            verify_draft(forward_ad.make_dual(t.detach(), torch.ones_like(t)), x, u, e, d, n, tau)
