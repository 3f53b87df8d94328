"""What the operators do with inputs that carry gradients they cannot give:
none is lost silently."""

import pytest
import torch
from torch.autograd import forward_ad

from test_head_norm import _inputs


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
