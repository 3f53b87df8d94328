"""The cache in 4 bits at the ends of what its calls take."""

import ctypes

import pytest
import torch


@pytest.mark.parametrize("D", [32, 64, 128])
def test_the_largest_page(D):
    """A slot lies at most 2^30 bytes behind its page's start."""
    from autoindexer_b200 import _lib
    from autoindexer_b200.paged4 import MAX_PAGE, _pool

    def pool(size, p):
        meta = dict(device="meta")
        codes = torch.empty(1, 1, size, D // 2, dtype=torch.uint8, **meta)
        scales = torch.empty(1, 1, size, D // 32, dtype=torch.float16, **meta)
        table = torch.empty(1, 1, dtype=torch.int32, **meta)
        return _pool(p, codes, codes, scales, scales, table, 1, 1, D, codes.get_device())

    p = _lib.AiPool4()
    pool(MAX_PAGE, p)
    assert p.page_size == MAX_PAGE and (MAX_PAGE - 1) * D // 2 < 2 ** 30
    with pytest.raises(ValueError, match="page_size must be a power of two from 16 to"):
        pool(2 * MAX_PAGE, _lib.AiPool4())
    a = _lib.AiPaged4Args()
    a.batch = a.seq_len = a.num_kv_heads = 1
    a.head_dim, a.dtype = D, _lib.DTYPE_BF16
    a.k.ptr = a.v.ptr = a.lens = 256
    for name in ("k_codes", "v_codes", "k_scales", "v_scales"):
        t = getattr(p, name)
        t.ptr = 256
    p.page_table = 256
    a.pool = p
    a.pool.page_size = 2 * MAX_PAGE
    L = _lib.lib()
    for fn in (L.ai_paged_append_4bit, L.ai_paged_read_4bit):
        assert fn(ctypes.byref(a), None) == 2
    b = _lib.AiPagedAttn4Args()
    b.batch = b.seq_len = b.num_q_heads = b.num_kv_heads = 1
    b.head_dim, b.dtype, b.scale = D, _lib.DTYPE_BF16, 0.1
    b.q.ptr = b.out.ptr = b.lens = 256
    b.pool = p
    n = ctypes.c_size_t(0)
    assert L.ai_paged_attn_4bit_workspace(ctypes.byref(b), ctypes.byref(n)) == 0
    b.pool.page_size = 2 * MAX_PAGE
    assert L.ai_paged_attn_4bit_workspace(ctypes.byref(b), ctypes.byref(n)) == 2
    assert L.ai_paged_attn_4bit(ctypes.byref(b), None) == 2


@pytest.mark.gpu
@pytest.mark.parametrize("T", [1, 2])
def test_the_longest_list(T, cuda_device):
    """2^31 - 1 keys (the pages repeat): the one slot past them is not looked at."""
    from autoindexer_b200 import paged_attention_4bit, read_status

    D, S, keys = 32, 2 ** 20, 2 ** 31 - 1
    g = torch.Generator().manual_seed(3)
    codes = [torch.randint(0, 256, (2, 1, S, D // 2), generator=g, dtype=torch.uint8) for _ in range(2)]
    scales = [0.05 + 0.2 * torch.rand(2, 1, S, 1, generator=g) for _ in range(2)]
    cache = [x.to(cuda_device) for x in (*codes, *(x.half() for x in scales))]
    for x in cache:
        x[1] = x[0]
    cache[2][1, 0, S - 1] = cache[3][1, 0, S - 1] = float("nan")
    table = torch.zeros(1, keys // S + 1, dtype=torch.int32, device=cuda_device)
    table[0, -1] = 1
    q = (0.3 * torch.randn(1, 2, T, D, generator=g)).to(torch.bfloat16).to(cuda_device)
    n = torch.tensor([keys], dtype=torch.int32, device=cuda_device)
    out, lse = paged_attention_4bit(q, *cache, table, n, return_lse=True)
    once, of_page = paged_attention_4bit(q, *cache, table[:, :1], torch.full_like(n, S), return_lse=True)
    assert read_status(cuda_device) == 0
    # A page 2048 times has the page's mean, and ln 2048 more; a key more or less changes 2^-20 of
    # it.  (Two values that close, each rounded by half a step at most, are a step apart at most:
    # bf16's step is 2^-7 of a value or less.)
    assert bool(((out - once)[:, -1].abs() <= 2.0 ** -7 * once[:, -1].abs() + 1e-5).all())
    more = torch.log(torch.tensor(2048.0)).item()
    assert bool(((lse - of_page)[..., -1] - more).abs().le(1e-4).all())
    if T > 1:
        assert bool(out[:, 0].isfinite().all())


def test_n_tokens_is_a_whole_number():
    from autoindexer_b200 import paged_read_4bit

    cache = [torch.zeros(2, 1, 16, 16, dtype=torch.uint8)] * 2 + [torch.zeros(2, 1, 16, 1, dtype=torch.float16)] * 2
    table, lens = torch.zeros(1, 1, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    for bad in (2.5, 2.0, "2", None, torch.tensor(2.0)):
        with pytest.raises(TypeError):
            paged_read_4bit(*cache, table, lens, bad, torch.bfloat16)


@pytest.mark.gpu
def test_n_tokens_of_a_tensor_that_changes(cuda_device):
    from autoindexer_b200 import paged_read_4bit

    cache = [torch.zeros(2, 1, 16, 16, dtype=torch.uint8, device=cuda_device)] * 2
    cache += [torch.zeros(2, 1, 16, 1, dtype=torch.float16, device=cuda_device)] * 2
    table, lens = (torch.zeros(*n, dtype=torch.int32, device=cuda_device) for n in ((1, 1), (1,)))
    n = torch.tensor(3)
    assert paged_read_4bit(*cache, table, lens, n, torch.bfloat16)[0].shape[2] == 3
    n.fill_(5)
    assert paged_read_4bit(*cache, table, lens, n, torch.bfloat16)[0].shape[2] == 5


@pytest.mark.gpu
@pytest.mark.parametrize("which", [2, 3])
def test_scales_that_require_a_gradient(which, cuda_device):
    """A backward that would reach them raises, as one to the query does."""
    from autoindexer_b200 import paged_attention_4bit

    cache = [torch.randint(0, 256, (2, 1, 16, 16), dtype=torch.uint8, device=cuda_device) for _ in range(2)]
    cache += [torch.ones(2, 1, 16, 1, dtype=torch.float16, device=cuda_device) for _ in range(2)]
    table, lens = (torch.full(n, 1, dtype=torch.int32, device=cuda_device) for n in ((1, 1), (1,)))
    q = torch.randn(1, 2, 1, 32, device=cuda_device).bfloat16()
    want = paged_attention_4bit(q, *cache, table, lens)
    assert not want.requires_grad
    cache[which].requires_grad_()
    out = paged_attention_4bit(q, *cache, table, lens)
    assert torch.equal(out, want)
    with pytest.raises(RuntimeError, match="paged_attention_4bit has no backward"):
        out.sum().backward()
    with torch.no_grad():
        assert not paged_attention_4bit(q, *cache, table, lens).requires_grad
