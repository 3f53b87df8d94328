"""Per-head norms with the rotation (``qk_norm_rope``): forward and gradients
against the 64-bit formula, the gradients against differences of the kernel's
own forward, and refusals.

Tolerances: an output is rounded once to its type (relative ``u``: half
the type's epsilon); before that every step is float32, a
few roundings of the terms it adds (their magnitudes come with the oracle's
results): at most D terms in the row sum, so ``C = D + 32`` units of 2^-24."""

import ctypes

import numpy as np
import pytest
import torch

from oracle import operator_oracle as O

U = {dtype: torch.finfo(dtype).eps / 2 for dtype in (torch.bfloat16, torch.float16, torch.float32)}
TINY = {torch.bfloat16: 0.0, torch.float16: 2.0 ** -25, torch.float32: 0.0}
EPS = 1e-6


def _table(n, D, device):
    a = torch.arange(n, dtype=torch.float64)[:, None] * 1e4 ** (-torch.arange(0, D, 2, dtype=torch.float64) / D)
    return a.cos().float().to(device), a.sin().float().to(device)


def _inputs(B, T, Hq, Hkv, D, dtype, seed, device, layout="bthd"):
    g = torch.Generator().manual_seed(seed)

    def heads(H):
        x = torch.randn(B, T, H, D, generator=g) * 1.5
        if layout == "bthd":
            return x.to(dtype).to(device).transpose(1, 2)
        if layout == "bhtd":
            return x.to(dtype).to(device).transpose(1, 2).contiguous()
        if layout == "fused":  # a slice of one projection's output
            wide = torch.zeros(B, T, H, 3 * D, dtype=dtype, device=device)
            wide[..., D:2 * D] = x.to(dtype).to(device)
            return wide[..., D:2 * D].transpose(1, 2)
        odd = torch.zeros(B, T, H, D + 3, dtype=dtype, device=device)  # rows off every 16-byte boundary
        odd[..., 1:D + 1] = x.to(dtype).to(device)
        return odd[..., 1:D + 1].transpose(1, 2)

    w = [(1 + 0.3 * torch.randn(D, generator=g)).to(dtype).to(device) for _ in range(2)]
    return heads(Hq), heads(Hkv), w[0], w[1]


def _np(x):
    return None if x is None else x.detach().double().cpu().numpy()


def _close(got, want, mag, dtype, D, extra=0):
    err = np.abs(_np(got) - want)
    tol = U[dtype] * np.abs(want) + (D + 32 + extra) * 2.0 ** -24 * mag + TINY[dtype]
    assert np.all(err <= tol), float((err / np.maximum(tol, 1e-300)).max())


CASES = [
    # B, T, Hq, Hkv, D, dtype, layout, positions
    (1, 1, 1, 1, 128, torch.bfloat16, "bthd", "shared"),
    (8, 1, 32, 8, 128, torch.bfloat16, "bthd", "rows"),
    (2, 37, 32, 8, 128, torch.bfloat16, "bthd", "rows"),
    (3, 5, 7, 3, 128, torch.float16, "bhtd", "int32"),
    (2, 19, 12, 4, 64, torch.float16, "fused", "rows"),
    (1, 23, 6, 2, 32, torch.bfloat16, "odd", "shared"),
    (2, 11, 5, 5, 64, torch.float32, "odd", "rows"),
    (1, 1300, 16, 2, 128, torch.float32, "bthd", "shared"),
    (2, 700, 24, 8, 64, torch.bfloat16, "bthd", "rows"),
    (1, 2500, 4, 1, 32, torch.float32, "bthd", "int32"),
]


def _positions(kind, B, T, n, device):
    g = torch.Generator().manual_seed(B + T)
    if kind == "shared":
        return torch.randint(0, n, (T,), generator=g).to(device)
    p = torch.randint(0, n, (B, T), generator=g)
    return (p.int() if kind == "int32" else p).to(device)


@pytest.mark.gpu
@pytest.mark.parametrize("B,T,Hq,Hkv,D,dtype,layout,kind", CASES)
def test_forward_and_gradients(B, T, Hq, Hkv, D, dtype, layout, kind, cuda_device):
    from autoindexer_b200 import qk_norm_rope, read_status

    q, k, wq, wk = _inputs(B, T, Hq, Hkv, D, dtype, 3, cuda_device, layout)
    cos, sin = _table(211, D, cuda_device)
    pos = _positions(kind, B, T, 211, cuda_device)
    for x in (q, k, wq, wk):
        x.requires_grad_()
    g = torch.Generator().manual_seed(9)
    gq, gk = (torch.randn(x.shape, generator=g).to(dtype).to(cuda_device) for x in (q, k))
    out = qk_norm_rope(q, k, wq, wk, (cos, sin), pos, eps=EPS)
    assert out[0].dtype == dtype and out[0].shape == q.shape and out[1].shape == k.shape
    with torch.no_grad():
        again = qk_norm_rope(q, k, wq, wk, (cos, sin), pos, eps=EPS)
    assert torch.equal(out[0], again[0]) and torch.equal(out[1], again[1])
    grads = torch.autograd.grad(out, (q, k, wq, wk), (gq, gk), retain_graph=True)
    same = torch.autograd.grad(out, (q, k, wq, wk), (gq, gk))
    for x, y in zip(grads, same):  # fixed summation order
        assert torch.equal(x, y)
    p = _np(pos).astype(np.int64)
    p = np.broadcast_to(p, (B, T))
    for x, w, o, gx, dx, dw in ((q, wq, out[0], gq, grads[0], grads[2]), (k, wk, out[1], gk, grads[1], grads[3])):
        want, mag = O.head_norm(_np(x), _np(w), _np(cos), _np(sin), p, EPS)
        _close(o, want, mag, dtype, D)
        rdx, rdw, mdx, mdw = O.head_norm_grad(_np(x), _np(w), _np(cos), _np(sin), p, EPS, _np(gx))
        _close(dx, rdx, mdx, dtype, D, extra=D)
        # a lane adds at most B T H / 4 rows one after another, the rest in trees
        _close(dw, rdw, mdw, dtype, D, extra=B * T * x.shape[1] // 4)
    assert read_status(cuda_device) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("which", ["no rope", "no weights", "query only", "one weight", "fp32 weights"])
def test_parts(which, cuda_device):
    from autoindexer_b200 import qk_norm_rope

    B, T, D = 2, 9, 128
    q, k, wq, wk = _inputs(B, T, 8, 2, D, torch.bfloat16, 5, cuda_device)
    cos, sin = _table(64, D, cuda_device)
    pos = _positions("rows", B, T, 64, cuda_device)
    rope = (cos, sin)
    if which == "no rope":
        rope = pos = cos = sin = None
    if which == "no weights":
        wq = wk = None
    if which == "query only":
        k = wk = None
    if which == "one weight":
        wq = None
    if which == "fp32 weights":
        wq, wk = wq.float() + 1e-4, wk.float() - 1e-4
    ins = [x for x in (q, k, wq, wk) if x is not None]
    for x in ins:
        x.requires_grad_()
    outs = qk_norm_rope(q, k, wq, wk, rope, pos)
    assert (outs[1] is None) == (k is None)
    real = [o for o in outs if o is not None]
    gs = [torch.randn_like(o) for o in real]
    grads = dict(zip(map(id, ins), torch.autograd.grad(real, ins, gs)))
    p = None if pos is None else _np(pos).astype(np.int64)
    for x, w, o, g in zip((q, k), (wq, wk), outs, gs):
        if x is None:
            continue
        want, mag = O.head_norm(_np(x), _np(w), _np(cos), _np(sin), p, EPS)
        _close(o, want, mag, torch.bfloat16, D)
        rdx, rdw, mdx, mdw = O.head_norm_grad(_np(x), _np(w), _np(cos), _np(sin), p, EPS, _np(g))
        _close(grads[id(x)], rdx, mdx, torch.bfloat16, D, extra=D)
        if w is not None:
            assert grads[id(w)].dtype == w.dtype
            _close(grads[id(w)], rdw, mdw, w.dtype, D, extra=B * T * 2)


@pytest.mark.gpu
def test_gradients_against_differences(cuda_device):
    """Central differences of the float32 forward along random directions: the
    step moves a row by about 0.7 % of its length, so the truncation is below
    1e-4 of the derivative's scale, rounding below 1e-4 too; 1e-3 is asked."""
    from autoindexer_b200 import qk_norm_rope

    B, T, D, h = 2, 13, 64, 1e-2
    q, k, wq, wk = _inputs(B, T, 6, 3, D, torch.float32, 21, cuda_device, "bhtd")
    rope = _table(40, D, cuda_device)
    pos = _positions("rows", B, T, 40, cuda_device)
    ins = [x.detach().clone().requires_grad_() for x in (q, k, wq, wk)]
    outs = qk_norm_rope(*ins, rope, pos)
    gen = torch.Generator().manual_seed(4)
    gs = [torch.randn(o.shape, generator=gen).to(cuda_device) for o in outs]
    grads = torch.autograd.grad(outs, ins, gs)

    def loss(xs):
        with torch.no_grad():
            return sum(float((o.double() * g.double()).sum()) for o, g in zip(qk_norm_rope(*xs, rope, pos), gs))

    for i, (x, d) in enumerate(zip(ins, grads)):
        step = torch.randn(x.shape, generator=gen).to(cuda_device)
        xs = [[y.detach() + (s * h * step if j == i else 0) for j, y in enumerate(ins)] for s in (1, -1)]
        got = (loss(xs[0]) - loss(xs[1])) / (2 * h)
        want = float((d.double() * step.double()).sum())
        scale = float(d.double().norm() * step.double().norm()) / x.numel() ** 0.5
        assert abs(got - want) <= 1e-3 * scale, (i, got, want, scale)


@pytest.mark.gpu
def test_broadcast_inputs_and_gradients(cuda_device):
    """One key head expanded over several, and an expanded output gradient."""
    from autoindexer_b200 import qk_norm_rope

    q, k, wq, wk = _inputs(2, 6, 4, 1, 64, torch.float32, 8, cuda_device)
    wide = k.detach().expand(2, 4, 6, 64)
    base = k.detach().clone().requires_grad_()
    qa, ka = qk_norm_rope(q, base.expand(2, 4, 6, 64), wq, wk)
    qb, kb = qk_norm_rope(q, wide.contiguous(), wq, wk)
    assert torch.equal(qa, qb) and torch.equal(ka, kb)
    (dk,) = torch.autograd.grad(ka.sum(), base)  # its gradient arrives with zero strides
    rdx = O.head_norm_grad(_np(k), _np(wk), None, None, None, EPS, np.ones(k.shape))
    _close(dk, 4 * rdx[0], 4 * rdx[2], torch.float32, 64, extra=64)


@pytest.mark.gpu
def test_position_outside_the_table(cuda_device):
    from autoindexer_b200 import qk_norm_rope, read_status

    q, k, wq, wk = _inputs(1, 3, 4, 2, 64, torch.bfloat16, 2, cuda_device)
    rope = _table(10, 64, cuda_device)
    read_status(cuda_device)
    bad = torch.tensor([1, 2 ** 32 + 3, 5], device=cuda_device)  # would be row 3 if it wrapped
    got = qk_norm_rope(q, k, wq, wk, rope, bad)
    assert read_status(cuda_device) == -2
    want = qk_norm_rope(q, k, wq, wk, rope, torch.tensor([1, 0, 5], device=cuda_device))
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    assert read_status(cuda_device) == 0


@pytest.mark.gpu
def test_zero_rows_and_large_values(cuda_device):
    """A zero row gives zeros (eps keeps the norm finite); magnitudes whose
    squares still fit float32 are normalised exactly as others are."""
    from autoindexer_b200 import qk_norm_rope

    q, k, wq, wk = _inputs(1, 4, 4, 2, 128, torch.bfloat16, 12, cuda_device)
    q = q.contiguous()
    q[:, :, 0] = 0
    q[:, :, 1] *= 2.0 ** 50
    out, _ = qk_norm_rope(q, k, wq, wk)
    assert torch.all(out[:, :, 0] == 0)
    want, mag = O.head_norm(_np(q), _np(wq), None, None, None, EPS)
    _close(out, want, mag, torch.bfloat16, 128)


@pytest.mark.gpu
def test_other_stream(cuda_device):
    from autoindexer_b200 import qk_norm_rope

    q, k, wq, wk = _inputs(2, 400, 32, 8, 128, torch.bfloat16, 6, cuda_device)
    want = qk_norm_rope(q, k, wq, wk)
    s = torch.cuda.Stream(cuda_device)
    s.wait_stream(torch.cuda.current_stream(cuda_device))
    with torch.cuda.stream(s):
        got = qk_norm_rope(q, k, wq, wk)
    torch.cuda.current_stream(cuda_device).wait_stream(s)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.gpu
def test_refusals(cuda_device):
    from autoindexer_b200 import qk_norm_rope

    q, k, wq, wk = _inputs(2, 5, 4, 2, 64, torch.bfloat16, 1, cuda_device)
    rope = _table(8, 64, cuda_device)
    pos = torch.zeros(2, 5, dtype=torch.long, device=cuda_device)
    for error, args in [
        (ValueError, (q[..., :48], k[..., :48])),
        (ValueError, (q, k[:, :, :3], wq, wk)),
        (ValueError, (q, None, wq, wk)),
        (ValueError, (q[:, :0], k, wq, wk)),
        (ValueError, (q, k, wq[:32], wk)),
        (ValueError, (q, k, wq, wk, rope)),
        (ValueError, (q, k, wq, wk, None, pos)),
        (ValueError, (q, k, wq, wk, rope, pos[:, :3])),
        (ValueError, (q, k, wq, wk, (rope[0][:, :16], rope[1]), pos)),
        (TypeError, (q, k.float(), wq, wk)),
        (TypeError, (q.double(), k.double())),
        (TypeError, (q, k, wq.half(), wk.half())),
        (TypeError, (q, k, wq.float(), wk)),
        (TypeError, (q, k, wq, wk, rope, pos.float())),
        (RuntimeError, (q, k, wq.cpu(), wk)),
        (RuntimeError, (q.cpu(), k.cpu())),
    ]:
        with pytest.raises(error):
            qk_norm_rope(*args)


def test_cpu_tensors_are_refused():
    from autoindexer_b200 import qk_norm_rope

    with pytest.raises(RuntimeError):
        qk_norm_rope(torch.zeros(1, 2, 3, 64), torch.zeros(1, 2, 3, 64))


def test_c_abi_refusals():
    from autoindexer_b200 import _lib

    L = _lib.lib()

    def args(**over):
        a = _lib.AiHeadNormArgs()
        a.batch, a.seq_len, a.num_q_heads, a.num_kv_heads, a.head_dim = 1, 4, 4, 2, 64
        a.dtype = a.weight_dtype = _lib.DTYPE_BF16
        for t in ("q", "k", "q_out", "k_out"):
            getattr(a, t).ptr = 256
        for n, v in over.items():
            setattr(a, n, v)
        return a

    assert L.ai_head_norm_fwd(None, None) == 1
    for field, value, code in (("batch", 0, 2), ("num_kv_heads", -1, 2), ("head_dim", 48, 3), ("dtype", 5, 4),
                               ("weight_dtype", 1, 4), ("rope_cos", 256, 1)):
        assert L.ai_head_norm_fwd(ctypes.byref(args(**{field: value})), None) == code
    assert L.ai_head_norm_fwd(ctypes.byref(args(rope_cos=256, rope_sin=256)), None) == 1  # no positions
    a = args()
    a.k.stride_h = -1
    assert L.ai_head_norm_fwd(ctypes.byref(a), None) == 5
    g = _lib.AiHeadNormBwdArgs()
    g.fwd = args(q_weight=256)
    for t in ("dq_out", "dk_out", "dq", "dk"):
        getattr(g, t).ptr = 256
    assert L.ai_head_norm_bwd(ctypes.byref(g), None) == 1  # no room for the weight's gradient
    g.dq_weight = 256
    n = ctypes.c_size_t(0)
    assert L.ai_head_norm_bwd_workspace(ctypes.byref(g), ctypes.byref(n)) == 0 and n.value > 0
    assert L.ai_head_norm_bwd(ctypes.byref(g), None) == 8
