"""The operators together, as ``examples/rollouts_and_distillation.py`` runs them:
every call that a rollout and a learning step make is checked against the
definition on the arguments it got, and the objective's gradient against float64
autograd and differences."""

import importlib.util
import os

import pytest
import torch

import test_distill
import test_paged4
import test_scoring
from conftest import ROOT
from test_scoring import REL


def _example():
    spec = importlib.util.spec_from_file_location("rollouts_and_distillation",
                                                  os.path.join(ROOT, "examples", "rollouts_and_distillation.py"))
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod


class Watched:
    """The package, its calls compared with the definition."""

    def __init__(self, ab):
        self.ab, self.calls = ab, []

    def __getattr__(self, name):
        return getattr(self.ab, name)

    def paged_append_4bit(self, key, value, *rest, new_lens):
        *pools, table, lens = rest
        self.ab.paged_append_4bit(key, value, *rest, new_lens=new_lens)
        test_paged4.check_held(key, value, pools, table.cpu(), lens.tolist(), new_lens.tolist(), key.shape[-1])
        self.calls.append("append")

    def paged_attention_4bit(self, query, *rest, query_lens):
        *pools, table, lens = rest
        out, lse = self.ab.paged_attention_4bit(query, *rest, query_lens=query_lens, return_lse=True)
        test_paged4.check_attention(query, pools, table, lens.tolist(), query_lens.tolist(), query.shape[-1] ** -0.5, out, lse)
        self.calls.append("attend")
        return out

    def token_logprobs(self, logits, tokens, temperature=None, top_k=0, entropy=False):
        got = self.ab.token_logprobs(logits, tokens, temperature, top_k, entropy)
        test_scoring.check(logits.detach(), tokens, temperature, top_k, type(got)(*(None if x is None else x.detach() for x in got)))
        self.calls.append("score")
        return got

    def distill_loss(self, logits, words, logprobs):
        loss = self.ab.distill_loss(logits, words, logprobs)
        test_distill.check(logits, words, logprobs, None, None, "bucket", loss.detach(), None)
        self.calls.append("distill")
        return loss


@pytest.mark.gpu
@pytest.mark.parametrize("head_dim,dtype", [(64, torch.bfloat16), (128, torch.float16)])
def test_rollout_and_learning_step(head_dim, dtype, cuda_device, monkeypatch):
    from autoindexer_b200 import read_status

    ex = _example()
    watch = Watched(ex.ab)
    monkeypatch.setattr(ex, "ab", watch)
    torch.manual_seed(4)
    shape = dict(vocab=211, hidden=128, heads=4, kv_heads=2, head_dim=head_dim)
    model = ex.Model(**shape).to(cuda_device, dtype)
    teacher = ex.Model(**shape, layers=3).to(cuda_device, dtype)
    prompts = [torch.randint(0, 211, (n,)).tolist() for n in (1, 64, 90, 17)]
    ids, targets, old = ex.sample(model, prompts, 5, 0.8, seed=1)
    assert watch.calls.count("append") == watch.calls.count("attend") == 2 * 5 and watch.calls.count("score") == 5
    for b, p in enumerate(prompts):
        assert ids[b, :len(p)].tolist() == p and not bool(ids[b, len(p) + 5:].any())
        live = (targets[b] >= 0).nonzero()[:, 0].tolist()
        assert live == list(range(len(p) - 1, len(p) + 4)) and torch.equal(targets[b, live], ids[b, len(p):len(p) + 5])
        assert bool((old[b, live] < 0).all())
    monkeypatch.setattr(ex, "ab", watch.ab)
    assert all(torch.equal(x, y) for x, y in zip(ex.sample(model, prompts, 5, 0.8, seed=1), (ids, targets, old)))
    monkeypatch.setattr(ex, "ab", watch)
    loss = ex.learn(model, teacher, ids, targets, old, torch.tensor([1.0, -0.5, 0.3, -1.2], device=cuda_device), 0.8, top=7)
    assert watch.calls[-3:] == ["score", "score", "distill"] and torch.isfinite(loss) and read_status(cuda_device) == 0
    for name, w in model.named_parameters():
        assert torch.isfinite(w.grad).all() and float(w.grad.float().abs().max()) > 0, name
    assert all(w.grad is None for w in teacher.parameters())


def plain_objective(logits, targets, old, advantage, words, word_logprobs, temperature, bonus=0.01, pull=0.5, clip=0.2):
    """The example's objective in the logits' type."""
    lp = torch.log_softmax(logits / temperature, -1)
    some = targets >= 0
    now = lp.gather(-1, targets.clamp_min(0)[..., None])[..., 0]
    ratio = (now - old).exp()
    gain = torch.minimum(ratio * advantage[:, None], ratio.clamp(1 - clip, 1 + clip) * advantage[:, None])
    lq = torch.log_softmax(logits, -1)
    p = word_logprobs.exp() * (words >= 0)
    listed = torch.zeros_like(logits).scatter_add(-1, words.clamp_min(0), (words >= 0).to(logits.dtype)) > 0
    rest, lq_rest = 1 - p.sum(-1), lq.masked_fill(listed, -float("inf")).logsumexp(-1)
    pulled = (p * (word_logprobs.masked_fill(words < 0, 0) - lq.gather(-1, words.clamp_min(0)))).sum(-1) + rest * (rest.log() - lq_rest)
    return ((pull * pulled - gain + bonus * (lp.exp() * lp).sum(-1))[some]).sum() / some.sum()


@pytest.mark.gpu
def test_gradient_of_the_objective(cuda_device):
    """Of a row's three parts each is good to 4 REL of its terms' magnitude, and the
    ratio, an exponential of a log-probability, to REL (1 + |logprob|)."""
    ex = _example()
    g = torch.Generator().manual_seed(7)
    B, T, V, K, tau = 3, 6, 401, 9, 0.7
    x = 2 * torch.randn(B, T, V, generator=g)
    targets = torch.randint(0, V, (B, T), generator=g)
    targets[0, 4:], targets[2, 0] = -100, -100
    advantage = torch.tensor([1.5, -0.7, 0.4])
    top, words = torch.log_softmax(2 * torch.randn(B, T, V, generator=g), -1).topk(K)
    words, top = words.masked_fill(targets[..., None] < 0, -1), top.masked_fill(targets[..., None] < 0, -float("inf"))
    now = torch.log_softmax(x.double() / tau, -1).gather(-1, targets.clamp_min(0)[..., None])[..., 0]
    old = (now + 0.3 * torch.randn(B, T, generator=g)).float().masked_fill(targets < 0, 0)
    y = x.to(cuda_device).requires_grad_()
    loss = ex.objective(y, *(t.to(cuda_device) for t in (targets, old, advantage, words, top)), temperature=tau)
    got = torch.autograd.grad(loss, y)[0].double().cpu()
    z = x.double().requires_grad_()
    want_loss = plain_objective(z, targets, old.double(), advantage.double(), words, top.double(), tau)
    want = torch.autograd.grad(want_loss, z)[0]
    size = float(now.abs().max())
    mag = (2 * 1.2 * 1.5 / tau + 0.01 * 2 * (size + 6) / tau + 2 * 0.5) / int((targets >= 0).sum())
    bound = (4 + 1 + size) * REL * mag
    assert float((got - want).abs().max()) <= bound and not bool(got[0, 4:].any()) and not bool(got[2, 0].any())
    assert abs(float(loss.detach()) - float(want_loss.detach())) <= (4 + 1 + size) * REL * (1 + size)
    way, step = torch.randn(x.shape, generator=g, dtype=torch.float64), 1e-6

    def f(v):
        return float(plain_objective(v, targets, old.double(), advantage.double(), words, top.double(), tau))

    slope = (f(x.double() + step * way) - f(x.double() - step * way)) / (2 * step)
    assert abs(slope - float((got * way).sum())) <= 1e-4 * (1 + abs(slope))


@pytest.mark.gpu
def test_streams_at_once_and_graphs_that_share_memory(cuda_device):
    """The same calls on two streams that overlap, and in two graphs of one memory pool
    replayed in turns, give what they give alone."""
    import autoindexer_b200 as ab

    def inputs(seed, lens):
        cache, table = test_paged4.filled(len(lens), 2, 64, 16, lens, torch.bfloat16, seed, cuda_device)
        q = test_paged4.heads(len(lens), 8, 1, 64, torch.bfloat16, seed, cuda_device)
        x, ids, t, w, tau = (y.to(cuda_device) for y in test_distill.make((40,), 5003, 6, torch.bfloat16, seed))
        return q, cache, table, test_paged4.ints(lens, cuda_device), x, ids, t, w, tau

    def step(q, cache, table, lens, x, ids, t, w, tau):
        score = ab.token_logprobs(x, ids[:, 0].clamp_min(0), tau, top_k=6, entropy=True)
        return [ab.paged_attention_4bit(q, *cache, table, lens), *score, *ab.distill_loss_and_grad(x, ids, t, w, tau)]

    both = [inputs(1, [700, 33, 1500]), inputs(2, [5, 2049, 64, 900])]
    want = [step(*given) for given in both]
    torch.cuda.synchronize(cuda_device)
    streams = [torch.cuda.Stream(cuda_device) for _ in both]
    got = [[], []]
    for _ in range(20):
        for i, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                got[i].append(step(*both[i]))
    torch.cuda.synchronize(cuda_device)
    for i in range(2):
        assert all(torch.equal(a, b) for out in got[i] for a, b in zip(out, want[i]))
    del got
    graphs, outs = [torch.cuda.CUDAGraph() for _ in both], []
    for i, graph in enumerate(graphs):
        with torch.cuda.graph(graph, pool=graphs[0].pool() if i else None):
            outs.append(step(*both[i]))
    for i in (0, 1, 1, 0):
        graphs[i].replay()
        torch.cuda.synchronize(cuda_device)
        assert all(torch.equal(a, b) for a, b in zip(outs[i], want[i]))
    del outs
    for graph in graphs:
        graph.reset()
    assert ab.read_status(cuda_device) == 0
