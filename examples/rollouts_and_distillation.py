"""Rollouts over a cache in 4 bits, scored and learnt from.

A small decoder (that of ``shared_prompt_rollouts.py``) continues a batch of
prompts of different lengths from a key / value cache in 4 bits, and takes a
policy-gradient step on what it sampled, towards a teacher at the same time:

    paged_append_4bit     keys and values of the prompts, then of every token
    paged_attention_4bit  prompts and single tokens over the cache
    token_logprobs        of the sampled tokens, as they are sampled and again as
                          the policy learns (with its entropy); the teacher's
                          likeliest words
    distill_loss          towards those, on the tokens that the student chose

    python examples/rollouts_and_distillation.py [--batch 8] [--tokens 32] [--top 16] [--temperature 1.0]
"""

import argparse
import os
import sys

import torch

sys.path[:0] = [os.path.dirname(os.path.dirname(os.path.abspath(__file__))), os.path.dirname(os.path.abspath(__file__))]

import autoindexer_b200 as ab  # noqa: E402
from shared_prompt_rollouts import PAGE, Model  # noqa: E402


class Cache:
    """Pools of codes and scales per layer, and each sequence's pages."""

    def __init__(self, model, batch, tokens, device):
        layer, per = model.layers[0], -(-tokens // PAGE)
        shape, D = (len(model.layers), batch * per, layer.kv_heads, PAGE), layer.head_dim
        self.codes = [torch.empty(*shape, D // 2, dtype=torch.uint8, device=device) for _ in range(2)]
        self.scales = [torch.empty(*shape, D // 32, dtype=torch.float16, device=device) for _ in range(2)]
        self.table = torch.arange(batch * per, dtype=torch.int32, device=device).view(batch, per)
        self.lens = torch.zeros(batch, dtype=torch.int32, device=device)

    def layer(self, i):
        return *(x[i] for x in self.codes), *(x[i] for x in self.scales), self.table


def forward(model, cache, tokens, n_new, rope):
    """Logits of ``tokens`` (B, T), the first ``n_new`` of each sequence real,
    behind what the cache holds; appends them."""
    x = model.embed(tokens)
    positions = (cache.lens[:, None] + torch.arange(tokens.shape[1], device=tokens.device)).clamp_max(cache.table.shape[1] * PAGE - 1)
    held = cache.lens + n_new
    for i, layer in enumerate(model.layers):
        q, k, v = layer.split(x)
        q, k = ab.qk_norm_rope(q, k, layer.q_norm, layer.k_norm, rope, positions)
        ab.paged_append_4bit(k, v, *cache.layer(i), cache.lens, new_lens=n_new)
        x = layer.finish(x, ab.paged_attention_4bit(q, *cache.layer(i), held, query_lens=n_new))
    cache.lens = held
    return model.head(x)


@torch.no_grad()
def sample(model, prompts, new_tokens, temperature, seed=0):
    """``new_tokens`` tokens behind each of ``prompts`` (lists of ids).  Returns
    the sequences (B, L), padded with 0; the tokens to learn (B, L - 1), -100
    where there is none, as targets of the positions before them; and their
    log-probabilities."""
    device, batch = model.embed.weight.device, len(prompts)
    layer, lens = model.layers[0], [len(p) for p in prompts]
    cache = Cache(model, batch, max(lens) + new_tokens, device)
    total = cache.table.shape[1] * PAGE
    rotary = ab.SectionedRope(layer.head_dim, 1e4, [torch.arange(total)], [(0, layer.head_dim // 2)], device=device)
    rope = ab.rope_table(rotary, 0, total - 1, layer.head_dim, device)
    gen = torch.Generator(device=device).manual_seed(seed)
    tau = torch.full((batch,), float(temperature), device=device)
    none = torch.zeros(batch, 0, device=device)
    ids = torch.zeros(batch, max(lens) + new_tokens, dtype=torch.int64, device=device)
    for b, p in enumerate(prompts):
        ids[b, :len(p)] = torch.tensor(p)
    rows, first = torch.arange(batch, device=device), torch.tensor(lens, device=device)
    targets = torch.full((batch, ids.shape[1] - 1), -100, device=device)
    logprobs = torch.zeros(targets.shape, device=device)
    logits = forward(model, cache, ids[:, :max(lens)], first.int(), rope)[rows, first - 1]
    one = torch.ones(batch, dtype=torch.int32, device=device)
    for t in range(new_tokens):
        noise = torch.empty(logits.shape, device=device).exponential_(generator=gen).clamp_min_(1e-20)
        token = ab.verify_draft(logits[:, None], none.long(), none, noise, temperature=tau)[1][:, 0].long()
        ids[rows, first + t] = token
        targets[rows, first + t - 1] = token
        logprobs[rows, first + t - 1] = ab.token_logprobs(logits, token, tau).logprobs
        if t + 1 < new_tokens:
            logits = forward(model, cache, token[:, None], one, rope)[:, 0]
    return ids, targets, logprobs


def logits_of(model, ids):
    """Logits of whole sequences, differentiable (padding comes last: nothing sees it)."""
    layer, length = model.layers[0], ids.shape[1]
    blocks = ab.document_blocks([length], position_ids=range(length))
    rotary = ab.SectionedRope(layer.head_dim, 1e4, [torch.arange(length)], [(0, layer.head_dim // 2)], device=ids.device)
    x = model.embed(ids)
    for block in model.layers:
        q, k, v = block.split(x)
        q, k = ab.qk_norm_rope(q, k, block.q_norm, block.k_norm)
        x = block.finish(x, ab.fused_chain_of_edits_attn_b200(rotary, q, k, v, blocks)[0])
    return model.head(x)


def objective(logits, targets, old, advantage, words, word_logprobs, temperature=1.0, bonus=0.01, pull=0.5, clip=0.2):
    """Clipped policy gradient with an entropy bonus, and the divergence from the
    teacher's list, per token that was sampled."""
    tau = torch.full((logits.shape[0],), float(temperature), device=logits.device)
    now = ab.token_logprobs(logits, targets, tau, entropy=True)
    ratio, advantage = (now.logprobs - old).exp(), advantage[:, None]
    gain = torch.minimum(ratio * advantage, ratio.clamp(1 - clip, 1 + clip) * advantage)
    pulled = ab.distill_loss(logits, words, word_logprobs)
    # (rows without a target give 0 in all three, and an empty list)
    some = targets >= 0
    return ((pull * pulled - gain - bonus * now.entropy) * some).sum() / some.sum()


def learn(model, teacher, ids, targets, old, advantage, temperature=1.0, top=16):
    """Gradients of the objective on sampled sequences."""
    with torch.no_grad():
        known = ab.token_logprobs(logits_of(teacher, ids[:, :-1]), targets, top_k=top)
    loss = objective(logits_of(model, ids[:, :-1]), targets, old, advantage, known.top_tokens, known.top_logprobs, temperature)
    loss.backward()
    return loss.detach()


def main():
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--batch", type=int, default=8)
    ap.add_argument("--tokens", type=int, default=32)
    ap.add_argument("--top", type=int, default=16)
    ap.add_argument("--temperature", type=float, default=1.0)
    args = ap.parse_args()
    torch.manual_seed(0)
    model, teacher = Model().to("cuda", torch.bfloat16), Model(layers=3).to("cuda", torch.bfloat16)
    prompts = [torch.randint(0, 512, (40 + 13 * b,)).tolist() for b in range(args.batch)]
    ids, targets, old = sample(model, prompts, args.tokens, args.temperature)
    # (a stand-in for a reward: the share of even tokens)
    reward = ((targets >= 0) & (targets % 2 == 0)).sum(1) / args.tokens
    advantage = (reward - reward.mean()) / (reward.std() + 1e-6)
    print(f"{args.batch} rollouts of {args.tokens} tokens, mean log-probability {float(old.sum() / (targets >= 0).sum()):.2f}")
    print("objective", float(learn(model, teacher, ids, targets, old, advantage, args.temperature, args.top)))
    status = ab.read_status(torch.device("cuda", torch.cuda.current_device()))
    assert status == 0, f"device status {status}"


if __name__ == "__main__":
    main()
