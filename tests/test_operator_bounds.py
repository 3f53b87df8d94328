"""The largest batches that the operators take, and the text that refuses larger ones."""

import pytest
import torch


@pytest.mark.gpu
def test_verification_batch(cuda_device):
    """B (2 L + 1) is at most 65535 with or without draft logits."""
    from autoindexer_b200 import read_status, verify_draft

    B, L, V = 13107, 2, 3
    t = torch.zeros(B + 1, L + 1, V, device=cuda_device)
    t[..., 1] = 5
    x = torch.ones(B + 1, L, dtype=torch.long, device=cuda_device)
    u, e = torch.zeros(B + 1, L, device=cuda_device), torch.ones(B + 1, V, device=cuda_device)
    for d in (None, t[:, :L]):
        a, said, _ = verify_draft(t[:B], x[:B], u[:B], e[:B], None if d is None else d[:B])
        assert bool((a == L).all()) and bool((said == 1).all())
        with pytest.raises(ValueError, match="65535"):
            verify_draft(t, x, u, e, d)
    assert read_status(cuda_device) == 0


@pytest.mark.gpu
def test_attention_batch(cuda_device):
    from autoindexer_b200 import read_status, shared_prefix_attention

    B, D = 65535, 32
    q = torch.zeros(B + 1, 1, 1, D, device=cuda_device)
    kp = torch.zeros(1, 1, 16, D, device=cuda_device)
    vp = torch.ones_like(kp)
    table = torch.zeros(B + 1, 1, dtype=torch.int32, device=cuda_device)
    lens = torch.ones(B + 1, dtype=torch.int32, device=cuda_device)
    out = shared_prefix_attention(q[:B], kp, vp, None, 0, table[:B], lens[:B])
    assert bool((out == 1).all()) and read_status(cuda_device) == 0
    with pytest.raises(ValueError, match="65535"):
        shared_prefix_attention(q, kp, vp, None, 0, table, lens)


@pytest.mark.gpu
@pytest.mark.parametrize("P", [0, 70, 3000])
@pytest.mark.parametrize("B,dtype", [(2, torch.bfloat16), (40, torch.float16), (2, torch.float32)])
def test_attention_without_room_for_own_keys(B, dtype, P, cuda_device):
    """A page table without columns: the prefix alone, or nothing."""
    from autoindexer_b200 import read_status, shared_prefix_attention

    g = torch.Generator(device=cuda_device).manual_seed(1)
    q = torch.randn(B, 8, 1, 64, generator=g, device=cuda_device).to(dtype)
    kp, vp = (torch.randn(50, 2, 64, 64, generator=g, device=cuda_device).to(dtype) for _ in range(2))
    prefix = torch.randperm(50, generator=g, device=cuda_device).int()
    none = torch.zeros(B, 0, dtype=torch.int32, device=cuda_device)
    one = torch.full((B, 1), 7, dtype=torch.int32, device=cuda_device)
    lens = torch.zeros(B, dtype=torch.int32, device=cuda_device)
    out, lse = shared_prefix_attention(q, kp, vp, prefix, P, none, lens, return_lse=True)
    want, wlse = shared_prefix_attention(q, kp, vp, prefix, P, one, lens, return_lse=True)
    assert read_status(cuda_device) == 0
    if P == 0:
        assert bool((out == 0).all()) and bool(torch.isneginf(lse).all())
    # (the two may cut the prefix at other places)
    assert float((out.float() - want.float()).abs().max()) <= 2.0 ** -7 and torch.allclose(lse, wlse, atol=1e-4)
