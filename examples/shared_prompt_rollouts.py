"""Several continuations of one prompt with drafted tokens, and a training
step, on the operators around the attention kernels.

A small Qwen3-like decoder (random weights, grouped-query attention, per-head
query / key norms) samples a batch of rollouts: the prompt's keys and values
are written once to pages that every sequence shares, each sequence's own
tokens go to its own pages, and every step runs the last token plus a few
drafted ones (looked up in what the sequence has so far) through the model and
keeps what the target distribution allows:

    qk_norm_rope            queries: norm + rotation
    paged_append            keys: norm + rotation on the way into the pages
    shared_prefix_attention prompt keys read once for the whole batch
    verify_draft            accepted drafts and the next token

Rejected drafts need no clean-up: the sequence's length does not count them
and the next step writes over their slots.

    python examples/shared_prompt_rollouts.py [--batch 8] [--tokens 32] [--draft 4] [--temperature 0.8]
"""

import argparse
import os
import sys

import torch
from torch import nn

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

import autoindexer_b200 as ab  # noqa: E402

PAGE = 64


class Layer(nn.Module):
    def __init__(self, hidden, heads, kv_heads, head_dim):
        super().__init__()
        self.heads, self.kv_heads, self.head_dim = heads, kv_heads, head_dim
        self.norm1, self.norm2 = nn.RMSNorm(hidden), nn.RMSNorm(hidden)
        self.qkv = nn.Linear(hidden, (heads + 2 * kv_heads) * head_dim, bias=False)
        self.o = nn.Linear(heads * head_dim, hidden, bias=False)
        self.up, self.down = nn.Linear(hidden, 2 * hidden, bias=False), nn.Linear(2 * hidden, hidden, bias=False)
        self.q_norm, self.k_norm = nn.Parameter(torch.ones(head_dim)), nn.Parameter(torch.ones(head_dim))

    def split(self, x):
        """Queries, keys and values as (B, H, T, D) views of one projection."""
        y = self.qkv(self.norm1(x)).unflatten(-1, (self.heads + 2 * self.kv_heads, self.head_dim)).transpose(1, 2)
        return y.split((self.heads, self.kv_heads, self.kv_heads), dim=1)

    def finish(self, x, attended):
        x = x + self.o(attended.flatten(2))
        return x + self.down(nn.functional.silu(self.up(self.norm2(x))))


class Model(nn.Module):
    def __init__(self, vocab=512, hidden=256, layers=2, heads=8, kv_heads=2, head_dim=64):
        super().__init__()
        self.embed = nn.Embedding(vocab, hidden)
        self.layers = nn.ModuleList(Layer(hidden, heads, kv_heads, head_dim) for _ in range(layers))
        self.head = nn.Linear(hidden, vocab, bias=False)


class Cache:
    """One page pool per layer, the prompt's page list and each sequence's."""

    def __init__(self, model, prompt_len, batch, own_tokens, dtype, device):
        layer = model.layers[0]
        shared, own = -(-prompt_len // PAGE), -(-own_tokens // PAGE)
        shape = (len(model.layers), shared + batch * own, layer.kv_heads, PAGE, layer.head_dim)
        self.k, self.v = (torch.empty(shape, dtype=dtype, device=device) for _ in range(2))
        ids = torch.arange(shape[1], dtype=torch.int32, device=device)
        self.prefix, self.table = ids[:shared].contiguous(), ids[shared:].reshape(batch, own)
        self.prefix_len = prompt_len
        self.lens = torch.zeros(batch, dtype=torch.int32, device=device)  # own tokens held


def forward(model, cache, tokens, n_new, positions, rope, prompt=False):
    """Logits of ``tokens`` (B, T), the first ``n_new`` of each sequence real;
    appends them to the cache (to the shared pages when ``prompt``)."""
    x = model.embed(tokens)
    table = cache.prefix[None] if prompt else cache.table
    held = torch.zeros_like(n_new) if prompt else cache.lens
    for i, layer in enumerate(model.layers):
        q, k, v = layer.split(x)
        q, _ = ab.qk_norm_rope(q, None, layer.q_norm, None, rope, positions)
        ab.paged_append(k, v, cache.k[i], cache.v[i], table, held, rope=rope, positions=positions, new_lens=n_new,
                        key_weight=layer.k_norm)
        attended = ab.shared_prefix_attention(q, cache.k[i], cache.v[i], None if prompt else cache.prefix,
                                              0 if prompt else cache.prefix_len, table, held + n_new, query_lens=n_new)
        x = layer.finish(x, attended)
    return model.head(x)


def lookup(history, length):
    """Up to ``length`` tokens that followed the last earlier occurrence of the
    history's last token."""
    for i in range(len(history) - 2, -1, -1):
        if history[i] == history[-1]:
            return history[i + 1:i + 1 + length]
    return []


@torch.no_grad()
def rollouts(model, prompt, batch, new_tokens, draft, temperature, seed=0):
    """``batch`` continuations of ``prompt`` (a list of ids) of at least
    ``new_tokens`` tokens each, and how many drafted tokens were accepted."""
    device, dtype = model.embed.weight.device, model.embed.weight.dtype
    layer = model.layers[0]
    total = len(prompt) + new_tokens + 2 * (draft + 1)
    rotary = ab.SectionedRope(layer.head_dim, 1e4, [torch.arange(total)], [(0, layer.head_dim // 2)], device=device)
    rope = ab.rope_table(rotary, 0, total - 1, layer.head_dim, device)
    cache = Cache(model, len(prompt), batch, new_tokens + 2 * (draft + 1), dtype, device)
    gen = torch.Generator(device=device).manual_seed(seed)
    tau = torch.full((batch,), float(temperature), device=device)
    ids = torch.tensor([prompt], device=device)
    logits = forward(model, cache, ids, torch.tensor([len(prompt)], dtype=torch.int32, device=device),
                     torch.arange(len(prompt), device=device), rope, prompt=True)[:, -1:]
    vocab = logits.shape[-1]

    def noise():
        return torch.empty(batch, vocab, device=device).exponential_(generator=gen).clamp_min_(1e-20)

    # The first token of every sequence: a verification without drafts.
    empty = torch.zeros(batch, 0, device=device)
    _, first, _ = ab.verify_draft(logits.expand(batch, 1, vocab), empty.long(), empty, noise(), temperature=tau)
    out = [[t] for t in first[:, 0].tolist()]
    accepted = steps = 0
    while min(map(len, out)) < new_tokens:
        drafts = [lookup(prompt + o, draft) for o in out]
        n = [len(d) for d in drafts]
        block = torch.tensor([[o[-1], *d, *[0] * (draft - len(d))] for o, d in zip(out, drafts)], device=device)
        n_draft = torch.tensor(n, dtype=torch.int32, device=device)
        positions = len(prompt) + cache.lens[:, None] + torch.arange(draft + 1, device=device)
        logits = forward(model, cache, block, n_draft + 1, positions.clamp_max(total - 1), rope)
        uniforms = torch.rand(batch, draft, generator=gen, device=device)
        took, said, _ = ab.verify_draft(logits, block[:, 1:], uniforms, noise(), draft_lens=n_draft, temperature=tau)
        # The last token and the accepted drafts stay in the cache; a sequence
        # that has enough waits for the others.
        done = torch.tensor([len(o) >= new_tokens for o in out], device=device)
        cache.lens += torch.where(done, 0, took + 1)
        for o, a, row, stop in zip(out, took.tolist(), said.tolist(), done.tolist()):
            if not stop:
                o.extend(row[:a + 1])
                accepted += a
                steps += 1
    return [o[:new_tokens] for o in out], accepted / max(1, steps)


def training_step(model, batch=2, length=256, seed=0):
    """One step through the differentiable operators: per-head norms, then the
    chain-of-edits attention (which rotates inside its kernels)."""
    device = model.embed.weight.device
    layer = model.layers[0]
    gen = torch.Generator(device=device).manual_seed(seed)
    ids = torch.randint(0, model.head.out_features, (batch, length + 1), generator=gen, device=device)
    blocks = ab.document_blocks([length], position_ids=range(length))
    rotary = ab.SectionedRope(layer.head_dim, 1e4, [torch.arange(length)], [(0, layer.head_dim // 2)], device=device)
    x = model.embed(ids[:, :-1])
    for block in model.layers:
        q, k, v = block.split(x)
        q, k = ab.qk_norm_rope(q, k, block.q_norm, block.k_norm)
        attended, _ = ab.fused_chain_of_edits_attn_b200(rotary, q, k, v, blocks)
        x = block.finish(x, attended)
    loss = nn.functional.cross_entropy(model.head(x).flatten(0, 1).float(), ids[:, 1:].flatten())
    loss.backward()
    return loss.detach()


def main():
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--batch", type=int, default=8)
    ap.add_argument("--tokens", type=int, default=32)
    ap.add_argument("--draft", type=int, default=4)
    ap.add_argument("--temperature", type=float, default=0.8)
    args = ap.parse_args()
    torch.manual_seed(0)
    model = Model().to("cuda", torch.bfloat16)
    prompt = torch.randint(0, 512, (700,)).tolist()
    texts, accepted = rollouts(model, prompt, args.batch, args.tokens, args.draft, args.temperature)
    print(f"{len(texts)} rollouts of {len(texts[0])} tokens; {accepted:.2f} drafted tokens accepted per step")
    print("training loss", float(training_step(model)))
    status = ab.read_status(torch.device("cuda", torch.cuda.current_device()))
    assert status == 0, f"device status {status}"


if __name__ == "__main__":
    main()
