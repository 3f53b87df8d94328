"""The backward of ``qk_norm_rope`` reads its saved tensors as they come back:
hooks on saved tensors (offloading, ``save_on_cpu``) may give back copies of
other strides."""

import pytest
import torch
from torch.autograd.graph import save_on_cpu, saved_tensors_hooks

from test_head_norm import _inputs, _table


def _sliced_positions(B, T, n, wide, device):
    g = torch.Generator().manual_seed(17)
    return torch.randint(0, n, (B, wide), generator=g).to(device)[:, 3:T + 3]


def _strides(t):
    return t.stride_b, t.stride_h, t.stride_t


@pytest.mark.parametrize("rows", [1, 3])
def test_backward_is_launched_with_the_saved_tensors_strides(rows, monkeypatch):
    """On the CPU with a recorded launch: every pointer of the backward goes
    with the strides of the tensor it points to."""
    from autoindexer_b200 import _call, head_norm, qk_norm_rope

    seen, given = [], {}
    monkeypatch.setattr(_call, "cuda_index", lambda name, x: -1)
    monkeypatch.setattr(_call, "status_ptr", lambda index: 0)
    monkeypatch.setattr(_call, "workspace", lambda *a: None)
    monkeypatch.setattr(_call, "launch", lambda fn, args, index, what: seen.append((what, type(args).from_buffer_copy(args))))
    monkeypatch.setattr(head_norm, "_PLANS", _call.Plans())
    B, T, D, n = 3, 5, 64, 40
    q, k, wq, wk = _inputs(B, T, 4, 2, D, torch.float32, 3, "cpu", "fused")
    rope = _table(n, D, "cpu")
    pos = _sliced_positions(rows, T, n, 1000, "cpu")
    for x in (q, k, wq, wk):
        x.requires_grad_()

    def back(x):
        # (an offloading hook brings a dense copy; one that keeps a layout of its own may transpose)
        y = x.clone(memory_format=torch.contiguous_format)
        if x.dim() == 4:
            y = x.transpose(-1, -2).contiguous().transpose(-1, -2)
        given[y.data_ptr()] = y
        return y

    with saved_tensors_hooks(lambda x: x, back):
        out = qk_norm_rope(q, k, wq, wk, rope, pos)
        assert seen[-1][0] == "ai_head_norm_fwd"
        assert seen[-1][1].pos.stride_b == (1000 if rows > 1 else 0)
        torch.autograd.grad(out, (q, k, wq, wk), [torch.ones_like(o) for o in out])
    what, args = seen[-1]
    assert what == "ai_head_norm_bwd"
    saved = given[args.fwd.pos.ptr]
    assert torch.equal(saved, pos) and saved.stride(0) == T
    assert args.fwd.pos.stride_b == (saved.stride(0) if rows > 1 else 0)
    # rows of q and k that lie one element apart are copied dense before the launch
    assert _strides(args.fwd.q) == (T * D * 4, T * D, D) and _strides(args.fwd.k) == (T * D * 2, T * D, D)
    # outside the hooks nothing has changed
    torch.autograd.grad(qk_norm_rope(q, k, wq, wk, rope, pos), (q,), [torch.ones_like(o) for o in out][:2])
    assert seen[-1][1].fwd.pos.stride_b == (1000 if rows > 1 else 0)
    assert _strides(seen[-1][1].fwd.q) == (q.stride(0), q.stride(1), q.stride(2))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_gradients_are_the_same_with_tensors_saved_on_the_host(dtype, cuda_device):
    from autoindexer_b200 import qk_norm_rope, read_status

    B, T, D, n = 4, 37, 128, 301
    q, k, wq, wk = _inputs(B, T, 8, 2, D, dtype, 5, cuda_device, "fused")
    rope = _table(n, D, cuda_device)
    pos = _sliced_positions(B, T, n, 1000, cuda_device)
    ins = [x.requires_grad_() for x in (q, k, wq, wk)]
    g = torch.Generator().manual_seed(2)
    gs = [torch.randn(x.shape, generator=g).to(dtype).to(cuda_device) for x in (q, k)]
    want = torch.autograd.grad(qk_norm_rope(*ins, rope, pos), ins, gs)
    with save_on_cpu():
        out = qk_norm_rope(*ins, rope, pos)
    got = torch.autograd.grad(out, ins, gs)
    assert read_status(cuda_device) == 0
    for x, y in zip(want, got):
        assert torch.equal(x, y)
