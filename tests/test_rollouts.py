"""The operators together, as ``examples/shared_prompt_rollouts.py`` runs them:
drafted greedy rollouts equal undrafted ones and a plain float64 decoder, and
the training step's gradients reach the norms' weights."""

import importlib.util
import os

import pytest
import torch

from conftest import ROOT


def _example():
    spec = importlib.util.spec_from_file_location("shared_prompt_rollouts",
                                                  os.path.join(ROOT, "examples", "shared_prompt_rollouts.py"))
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod


def _plain_logits(model, ids):
    """A dense float64 forward of the example's model over one sequence."""
    layer = model.layers[0]
    D, G = layer.head_dim, layer.heads // layer.kv_heads
    T = ids.shape[0]
    w = {k: v.double() for k, v in model.state_dict().items()}
    ang = torch.arange(T).double()[:, None] * 1e4 ** (-torch.arange(0, D, 2).double() / D)
    cos, sin = ang.cos(), ang.sin()

    def rms(x, g, eps):
        return x / (x.pow(2).mean(-1, keepdim=True) + eps).sqrt() * g

    def rot(x):
        a, b = x[..., :D // 2], x[..., D // 2:]
        return torch.cat([a * cos[:, None] - b * sin[:, None], b * cos[:, None] + a * sin[:, None]], -1)

    x = w["embed.weight"][ids]
    small = torch.finfo(torch.float32).eps  # nn.RMSNorm's default for the weights' type
    for i in range(len(model.layers)):
        p = f"layers.{i}."
        y = (rms(x, w[p + "norm1.weight"], small) @ w[p + "qkv.weight"].T).reshape(T, -1, D)
        q, k, v = y[:, :layer.heads], y[:, layer.heads:layer.heads + layer.kv_heads], y[:, layer.heads + layer.kv_heads:]
        q, k = rot(rms(q, w[p + "q_norm"], 1e-6)), rot(rms(k, w[p + "k_norm"], 1e-6))
        s = torch.einsum("thd,shd->hts", q, k.repeat_interleave(G, 1)) * D ** -0.5
        s = s.masked_fill(torch.ones(T, T).triu(1).bool(), float("-inf"))
        o = torch.einsum("hts,shd->thd", s.softmax(-1), v.repeat_interleave(G, 1)).reshape(T, -1)
        x = x + o @ w[p + "o.weight"].T
        h = rms(x, w[p + "norm2.weight"], small) @ w[p + "up.weight"].T
        x = x + (h * torch.sigmoid(h)) @ w[p + "down.weight"].T
    return x @ w["head.weight"].T


@pytest.mark.gpu
def test_greedy_rollouts_with_and_without_drafts(cuda_device):
    """float32 and greedy: the drafted run emits what the undrafted one does,
    and each token is the largest logit of a float64 forward (or within the
    float32 model's error of it: 1e-4 of logits of order 1)."""
    from autoindexer_b200 import read_status

    ex = _example()
    torch.manual_seed(3)
    model = ex.Model(vocab=61, hidden=128, heads=4, kv_heads=2, head_dim=64).to(cuda_device)
    prompt = torch.randint(0, 61, (150,)).tolist()
    plain, none = ex.rollouts(model, prompt, 3, 20, 0, 0.0)
    drafted, took = ex.rollouts(model, prompt, 3, 20, 4, 0.0)
    assert read_status(cuda_device) == 0
    assert none == 0 and plain == drafted
    assert plain[0] == plain[1] == plain[2]  # greedy: every continuation is the same
    logits = _plain_logits(model.cpu(), torch.tensor(prompt + plain[0]))
    for i, t in enumerate(plain[0]):
        row = logits[len(prompt) + i - 1]
        assert float(row.max() - row[t]) <= 1e-4


@pytest.mark.gpu
def test_sampled_rollouts_run_in_bfloat16(cuda_device):
    from autoindexer_b200 import read_status

    ex = _example()
    torch.manual_seed(1)
    model = ex.Model(vocab=97, hidden=128, heads=8, kv_heads=2, head_dim=128).to(cuda_device, torch.bfloat16)
    prompt = torch.randint(0, 97, (333,)).tolist()
    texts, _ = ex.rollouts(model, prompt, 5, 16, 3, 1.0, seed=2)
    again, _ = ex.rollouts(model, prompt, 5, 16, 3, 1.0, seed=2)
    assert texts == again and len({tuple(t) for t in texts}) > 1
    assert all(len(t) == 16 and all(0 <= x < 97 for x in t) for t in texts)
    assert read_status(cuda_device) == 0


@pytest.mark.gpu
def test_training_step_reaches_the_norm_weights(cuda_device):
    from autoindexer_b200 import read_status

    ex = _example()
    torch.manual_seed(2)
    model = ex.Model(hidden=128, heads=4, kv_heads=2, head_dim=128).to(cuda_device, torch.bfloat16)
    loss = ex.training_step(model)
    assert torch.isfinite(loss) and read_status(cuda_device) == 0
    for layer in model.layers:
        for w in (layer.q_norm, layer.k_norm, layer.qkv.weight):
            assert torch.isfinite(w.grad).all() and float(w.grad.float().abs().max()) > 0


def test_lookup_drafts():
    ex = _example()
    assert ex.lookup([5, 1, 2, 3, 9, 1], 2) == [2, 3]
    assert ex.lookup([5, 1, 2, 1], 4) == [2, 1]
    assert ex.lookup([1, 2, 3], 4) == []
