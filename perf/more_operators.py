"""Cases of the operators for rollouts and what is learnt from them: log-probabilities of given tokens (with entropy
and the likeliest alternatives, and their gradient), distillation from a teacher's likeliest tokens, and a paged cache
held in 4 bits with the attention that reads it.

``run`` computes a case in plain fp32 torch operations, or with the library's operators where ``own`` is true;
``exact`` restates it in 64 bits.  Sizes are those of the library's benchmark layer (32 query heads, 8 KV heads,
head_dim 128, vocabulary 151936, sequences up to 32768) and smaller or odd ones.

The 4-bit format: 32 dims of a head row share an fp16 scale d, minus an eighth of their value of largest magnitude
(the negative one of two); a dim's code c in 0..15 stands for (c - 8) d.  Of a row of D dims, dim 32 c + 4 g + j (g < 8,
j < 4) lies in byte g D / 16 + 2 c + j / 2, in the low half for even j."""

import math

import torch

own = False

_DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}
NONE = -math.inf


# ------------------------------------------------------------------ cases
def listed():
    layer = {"Hq": 32, "Hkv": 8, "D": 128}
    return [
        # one decode step of 8 requests that asked for the alternatives' probabilities: latency
        dict(name="score step", op="score", B=8, T=1, V=151936, dtype="bf16", k=20, tau=True, train=False),
        # 64 rollouts of up to 64 tokens in policy training: log-probabilities and entropy, forward and backward
        dict(name="score train", op="score", B=64, T=64, V=151936, dtype="bf16", k=0, tau=True, train=True),
        # a teacher's pass over one document: its 32 likeliest tokens per position, fp32 logits
        dict(name="score teacher", op="score", B=1, T=509, V=151936, dtype="fp32", k=32, tau=False, train=False),
        # a draft model's update from 16 positions just verified: latency
        dict(name="distill step", op="distill", B=4, T=4, V=151936, dtype="bf16", k=8, tail="bucket", fused=True),
        # distillation of a batch: 4096 positions, 32 teacher tokens each, loss and gradient in one call
        dict(name="distill train", op="distill", B=8, T=512, V=151936, dtype="bf16", k=32, tail="bucket", fused=True),
        # a smaller vocabulary of odd size in fp16, through autograd (loss, then its backward)
        dict(name="distill odd", op="distill", B=3, T=341, V=32003, dtype="fp16", k=64, tail="renormalize", fused=False),
        # the cache write of one decode step of 64 sequences, and the values that the cache then holds
        dict(layer, name="append decode", op="append", B=64, T=1, M=512, S=64, dtype="bf16"),
        # the same of a prefill of ragged prompts
        dict(layer, name="append prefill", op="append", B=8, T=2047, M=2304, S=16, dtype="fp16"),
        # four edits of one short document, one token each: latency
        dict(layer, name="attend small", op="attend", B=4, T=1, M=322, S=16, dtype="bf16"),
        # 64 sequences of up to 8192 tokens, one token each
        dict(layer, name="attend batch", op="attend", B=64, T=1, M=8192, S=64, dtype="bf16"),
        # 32 long documents, one token each
        dict(layer, name="attend long", op="attend", B=32, T=1, M=32768, S=64, dtype="bf16"),
        # 64 sequences with drafted tokens (up to five query tokens each): more rows meet each key
        dict(layer, name="attend drafted", op="attend", B=64, T=5, M=8192, S=32, dtype="fp16"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    op = rng.choice(["score", "distill", "append", "attend"])
    if op in ("score", "distill"):
        dtype = rng.choice(["bf16", "fp16", "fp32"])
        V = _log(rng, 1000, 151936)
        B = _log(rng, 1, 64)
        if op == "score":
            k = rng.choice([0, 0, 1, 5, 20, 64])
            T = _log(rng, 1, max(1, (512 if k else 4096 if dtype != "fp32" else 2048) // B))
            return dict(op=op, B=B, T=T, V=V, dtype=dtype, k=k, tau=rng.random() < 0.5, train=rng.random() < 0.6)
        T = _log(rng, 1, max(1, (4096 if dtype != "fp32" else 2048) // B))
        return dict(op=op, B=B, T=T, V=V, dtype=dtype, k=_log(rng, 1, 128), tail=rng.choice(["bucket", "renormalize"]),
                    fused=rng.random() < 0.6)
    Hq, Hkv = rng.choice([(32, 8), (16, 2), (8, 8), (24, 8), (4, 1)])
    case = dict(op=op, Hq=Hq, Hkv=Hkv, D=rng.choice([32, 64, 128, 128]), dtype=rng.choice(["bf16", "fp16"]))
    B, S = _log(rng, 1, 64), rng.choice([16, 32, 64, 128])
    if op == "append":
        T = _log(rng, 1, max(1, 16384 // B))
        return dict(case, B=B, T=T, M=T + _log(rng, 1, 512), S=S)
    T = rng.choice([1, 1, 2, 3, 5])
    return dict(case, B=B, T=T, M=_log(rng, T, min(32768, 2 ** 19 // B)), S=S)


def _spread(n, lo, hi, phase=0.0):
    """n whole numbers over [lo, hi], evenly spread, in no order."""
    return [lo + int((hi - lo + 1) * ((i * 0.6180339887 + phase) % 1.0)) for i in range(n)]


def _real(case):
    """Rows that count of each sequence of T (the others are padding)."""
    return _spread(case["B"], max(1, 3 * case["T"] // 4), case["T"], 0.9)


def _lens(case):
    """Tokens of each sequence (the new ones among them; those before them, for an append) and how many of its T
    new tokens are real."""
    B, T, M = case["B"], case["T"], case["M"]
    n = [T] * B if T == 1 else _spread(B, 1, T, 0.9)
    if case["op"] == "append":
        return _spread(B, 0, M - T, 0.4), n
    return [max(a, b) for a, b in zip(_spread(B, 1, M, 0.5), n)], n


# ------------------------------------------------------------------ the 4-bit format
def _quantize(x):
    """(..., D) -> codes (..., D) int64 and scales (..., D / 32) fp16."""
    v = x.double().unflatten(-1, (-1, 32))
    top, low = v.amax(-1), v.amin(-1)
    d = (torch.where(top > -low, top, low) / -8).float().half()
    q = torch.where(d[..., None] == 0, 0.0, v / d[..., None].double())
    return (torch.round(q).clamp(-8, 7) + 8).long().flatten(-2), d


def _values(codes, d):
    return ((codes.float() - 8).unflatten(-1, (-1, 32)) * d.float()[..., None]).flatten(-2)


def _pack(codes):
    x = codes.to(torch.uint8).unflatten(-1, (-1, 8, 2, 2))
    x = x[..., 0] | (x[..., 1] << 4)
    return x.transpose(-3, -2).flatten(-3).contiguous()


def _unpack(pages):
    x = pages.unflatten(-1, (8, -1, 2)).transpose(-3, -2)
    return torch.stack((x & 15, x >> 4), -1).flatten(-4)


# ------------------------------------------------------------------ inputs
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _heads(g, B, T, H, D, dt, scale=1.0):
    """What a projection gives: (B, T, H, D) in memory, seen as (B, H, T, D)."""
    return (torch.randn(B, T, H, D, generator=g, device="cuda") * scale).to(dt).transpose(1, 2)


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _logits(g, B, T, V, dt):
    out = torch.empty(B, T, V, dtype=dt, device="cuda")
    for row in out.view(-1, V).split(256):
        row.copy_(2.5 * torch.randn(row.shape, generator=g, device="cuda"))
    return out


def _prepare_rows(s, case, g, dt):
    B, T, V, k = (case[n] for n in ("B", "T", "V", "k"))
    real = torch.arange(T, device="cuda") < torch.tensor(_real(case), device="cuda")[:, None]
    s["logits"] = _logits(g, B, T, V, dt)
    if case["op"] == "score":
        s["tau"] = 0.6 + 0.8 * torch.rand(B, generator=g, device="cuda") if case["tau"] else None
        tokens = torch.randint(0, V, (B, T, 1), generator=g, device="cuda")
        # (sampled tokens are likely ones)
        s["logits"].scatter_add_(-1, tokens, (8 * torch.rand(B, T, 1, generator=g, device="cuda")).to(dt))
        s["tokens"] = torch.where(real, tokens[..., 0], -100)
        s["g_logprob"] = torch.randn(B, T, generator=g, device="cuda")
        s["g_entropy"] = 0.1 * torch.rand(B, T, generator=g, device="cuda")
        s["g_top"] = torch.randn(B, T, k, generator=g, device="cuda") if k else None
        s["logits"].requires_grad_(own and case["train"])
        return
    # The teacher's likeliest tokens and their log-probabilities, best first; the student roughly agrees.
    step = 2 * torch.randint(0, max(1, V // (2 * k)), (B, T, 1), generator=g, device="cuda") + 1
    first = torch.randint(0, V, (B, T, 1), generator=g, device="cuda")
    s["ids"] = (first + step * torch.arange(k, device="cuda")) % V
    t = torch.sort(2 * torch.randn(B, T, k, generator=g, device="cuda"), dim=-1, descending=True)[0]
    t = t - 0.1 * torch.arange(k, device="cuda")
    kept = 0.7 + 0.28 * torch.rand(B, T, 1, generator=g, device="cuda")
    s["teacher"] = torch.log_softmax(t, -1) + kept.log()
    s["logits"].scatter_(-1, s["ids"], (9 + t + 0.5 * torch.randn(B, T, k, generator=g, device="cuda")).to(dt))
    s["weights"] = torch.where(real, 0.5 + torch.rand(B, T, generator=g, device="cuda"), 0.0)
    s["ids"] = torch.where(real[..., None], s["ids"], -1)
    s["logits"].requires_grad_(own and not case["fused"])


def prepare(case, seed):
    g, dt, op = _gen(seed), _DT[case["dtype"]], case["op"]
    s = {"case": case}
    if op in ("score", "distill"):
        _prepare_rows(s, case, g, dt)
        return s
    B, T, Hq, Hkv, D, S, M = (case[k] for k in ("B", "T", "Hq", "Hkv", "D", "S", "M"))
    lens, n = _lens(case)
    s["lens"], s["n"] = _ints(lens), _ints(n)
    per = -(-M // S)
    held = [-(-(a + (b if op == "append" else 0)) // S) for a, b in zip(lens, n)]
    pages = sum(held) + 2
    order = torch.randperm(pages, generator=g, device="cuda").int()
    s["table"] = torch.zeros(B, per, dtype=torch.int32, device="cuda")
    at = 0
    for b, h in enumerate(held):
        s["table"][b, :h] = order[at:at + h]
        at += h
    for name in ("k", "v"):
        codes = torch.empty(pages, Hkv, S, D // 2, dtype=torch.uint8, device="cuda")
        scales = torch.empty(pages, Hkv, S, D // 32, dtype=torch.float16, device="cuda")
        step = max(1, 2 ** 25 // (Hkv * S * D))
        for c, d in zip(codes.split(step), scales.split(step)):
            x = torch.randn(*c.shape[:3], D, generator=g, device="cuda")
            q, e = _quantize(x.to(dt))
            c.copy_(_pack(q))
            d.copy_(e)
        s[name + "_pages"], s[name + "_scales"] = codes, scales
    if op == "append":
        s["k"], s["v"] = _heads(g, B, T, Hkv, D, dt, 1.5), _heads(g, B, T, Hkv, D, dt)
    else:
        s["q"] = _heads(g, B, T, Hq, D, dt, 1.5)  # sharper than noise, as trained heads are
    return s


# ------------------------------------------------------------------ plain forms, 32 bits
def _best(x, k):
    """The k largest of each row and where they are, equal ones by index; -1 past the unmasked ones."""
    value, at = [], []
    for rows in x.flatten(0, -2).split(128):
        v, i = torch.sort(rows, dim=-1, descending=True, stable=True)
        value.append(v[:, :k])
        at.append(i[:, :k])
    value, at = torch.cat(value).view(*x.shape[:-1], -1), torch.cat(at).view(*x.shape[:-1], -1)
    return value, torch.where(value == NONE, -1, at)


def _plain_score(s):
    c, tokens = s["case"], s["tokens"]
    inv = 1.0 if s["tau"] is None else (1 / s["tau"])[:, None, None]
    real = tokens >= 0
    x = s["logits"].detach().float()
    z = (x - x.amax(-1, keepdim=True)) * inv
    logp = z - torch.log(torch.exp(z).sum(-1, keepdim=True))
    del z
    p = torch.exp(logp)
    given = tokens.clamp_min(0)[..., None]
    out = [torch.where(real, logp.gather(-1, given)[..., 0], 0.0)]
    entropy = -(p * logp).sum(-1)
    out.append(torch.where(real, entropy, 0.0))
    ids = None
    if c["k"]:
        _, ids = _best(x, c["k"])
        top = torch.where(ids >= 0, logp.gather(-1, ids.clamp_min(0)), NONE)
        out += [torch.where(real[..., None], top, NONE), torch.where(real[..., None], ids, -1)]
    if c["train"]:
        g, h = s["g_logprob"][..., None], s["g_entropy"][..., None]
        total = g + (s["g_top"].sum(-1, keepdim=True) if c["k"] else 0.0)
        d = -p * (total + h * (logp + entropy[..., None]))
        d.scatter_add_(-1, given, g)
        if c["k"]:
            d.scatter_add_(-1, ids, s["g_top"])
        out.append(torch.where(real[..., None], d * inv, 0.0).to(s["logits"].dtype))
    return out


def _plain_distill(s):
    ids, w = s["ids"], s["weights"]
    real = ids[..., 0] >= 0
    at, x = ids.clamp_min(0), s["logits"].detach().float()
    z = x - x.amax(-1, keepdim=True)
    q = torch.exp(z)
    zk = z.gather(-1, at)
    if s["case"]["tail"] == "renormalize":
        logp = s["teacher"] - s["teacher"].amax(-1, keepdim=True)
        logp = logp - torch.log(torch.exp(logp).sum(-1, keepdim=True))
        total = q.sum(-1, keepdim=True)
        p = torch.exp(logp)
        loss = (p * (logp - zk + torch.log(total))).sum(-1)
        d = q / total
        d.scatter_add_(-1, at, -p)
    else:
        p = torch.exp(s["teacher"])
        left = (1 - p.double().sum(-1, keepdim=True)).float()
        qk = torch.exp(zk)
        q.scatter_(-1, at, 0.0)
        rest = q.sum(-1, keepdim=True)  # (the other words' sum by itself: a difference would lose it)
        total = rest + qk.sum(-1, keepdim=True)
        loss = (p * (s["teacher"] - zk + torch.log(total))).sum(-1)
        loss = loss + (left * (torch.log(left) - torch.log(rest / total)))[..., 0]
        d = q * (1 / total - left / rest)
        d.scatter_(-1, at, qk / total - p)
    d = torch.where(real[..., None], d * w[..., None], 0.0).to(s["logits"].dtype)
    return [torch.where(real, loss, 0.0), d]


def _plain_append(s):
    T, S = s["case"]["T"], s["case"]["S"]
    t = torch.arange(T, device="cuda")
    b, t = torch.nonzero(t < s["n"][:, None], as_tuple=True)
    at = s["lens"][b] + t
    page = s["table"][b, at // S].long()
    out = []
    for name in ("k", "v"):
        codes, d = _quantize(s[name])
        s[name + "_pages"][page, :, at % S] = _pack(codes)[b, :, t]
        s[name + "_scales"][page, :, at % S] = d[b, :, t]
        held = _values(_unpack(s[name + "_pages"][page, :, at % S]), s[name + "_scales"][page, :, at % S])
        x = torch.zeros(s[name].shape, dtype=s[name].dtype, device="cuda")
        x[b, :, t] = held.to(x.dtype)
        out.append(x)
    return out


def _plain_attend(s):
    c = s["case"]
    B, T, Hq, Hkv, D = (c[k] for k in ("B", "T", "Hq", "Hkv", "D"))
    G = Hq // Hkv
    out = torch.empty(B, T, Hq, D, dtype=s["q"].dtype, device="cuda")
    step = max(1, 2 ** 30 // (s["table"].shape[1] * c["S"] * Hkv * D))
    for b0 in range(0, B, step):
        b = slice(b0, b0 + step)
        k, v = (_values(_unpack(s[x + "_pages"][s["table"][b].long()]), s[x + "_scales"][s["table"][b].long()])
                .transpose(1, 2).flatten(2, 3) for x in ("k", "v"))
        q = (s["q"][b].float() * D ** -0.5).reshape(-1, Hkv, G * T, D)
        score = q @ k.transpose(-1, -2)
        t = torch.arange(T, device="cuda").repeat(G)
        lens, n = s["lens"][b, None], s["n"][b, None]
        seen = torch.arange(k.shape[2], device="cuda") <= (lens - n + t)[..., None]
        score = score.masked_fill(~seen[:, None], NONE)
        e = torch.exp(score - score.amax(-1, keepdim=True))
        o = (e @ v) / e.sum(-1, keepdim=True)
        o = o.masked_fill(~(t < n)[:, None, :, None], 0.0)
        out[b] = o.reshape(-1, Hq, T, D).transpose(1, 2).to(out.dtype)
    return out


_PLAIN = {"score": _plain_score, "distill": _plain_distill, "append": _plain_append, "attend": _plain_attend}


# ------------------------------------------------------------------ the library's operators
def _own_score(ab, s):
    c = s["case"]
    got = ab.token_logprobs(s["logits"], s["tokens"], temperature=s["tau"], top_k=c["k"], entropy=True)
    out, grads = [got.logprobs, got.entropy], [s["g_logprob"], s["g_entropy"]]
    if c["k"]:
        out.append(got.top_logprobs)
        grads.append(s["g_top"])
    d = torch.autograd.grad(out, s["logits"], grads) if c["train"] else ()
    out = [x.detach() for x in out]
    if c["k"]:
        out.append(got.top_tokens)
    return [*out, *d]


def _own_distill(ab, s):
    tail = s["case"]["tail"]
    if s["case"]["fused"]:
        return ab.distill_loss_and_grad(s["logits"], s["ids"], s["teacher"], s["weights"], tail=tail)
    loss = ab.distill_loss(s["logits"], s["ids"], s["teacher"], tail=tail)
    return [loss.detach(), *torch.autograd.grad(loss, s["logits"], s["weights"])]


def _own_append(ab, s):
    cache = (s["k_pages"], s["v_pages"], s["k_scales"], s["v_scales"], s["table"], s["lens"])
    ab.paged_append_4bit(s["k"], s["v"], *cache, new_lens=s["n"])
    return ab.paged_read_4bit(*cache, s["case"]["T"], s["k"].dtype, read_lens=s["n"])


def _own_attend(ab, s):
    return ab.paged_attention_4bit(s["q"], s["k_pages"], s["v_pages"], s["k_scales"], s["v_scales"], s["table"], s["lens"],
                                   query_lens=s["n"])


_OWN = {"score": _own_score, "distill": _own_distill, "append": _own_append, "attend": _own_attend}


def run(state):
    op = state["case"]["op"]
    if not own:
        with torch.no_grad():
            return _PLAIN[op](state)
    import autoindexer_b200

    return _OWN[op](autoindexer_b200, state)


# ------------------------------------------------------------------ 64 bits, from the definitions
def _exact_score(s):
    c, V = s["case"], s["case"]["V"]
    B, T, k = c["B"], c["T"], c["k"]
    dev = dict(dtype=torch.float64, device="cuda")
    logprob, entropy = torch.zeros(B, T, **dev), torch.zeros(B, T, **dev)
    top, ids = torch.full((B, T, k), NONE, **dev), torch.full((B, T, k), -1, device="cuda")
    grad = torch.zeros(B, T, V, **dev) if c["train"] else None
    for b, n in enumerate(_real(c)):
        for t0 in range(0, n, 64):
            r = slice(t0, min(n, t0 + 64))
            tau = 1.0 if s["tau"] is None else s["tau"][b].double()
            x = s["logits"][b, r].double().requires_grad_()
            y = x / tau
            lse = torch.logsumexp(y, -1, keepdim=True)
            lp = y - lse
            a = lp.gather(-1, s["tokens"][b, r, None])[:, 0]
            h = lse[:, 0] - (torch.exp(lp) * y).sum(-1)
            total = (a * s["g_logprob"][b, r].double()).sum() + (h * s["g_entropy"][b, r].double()).sum()
            if k:
                # the best by value, then by index: whole numbers that order a row's words
                order = torch.argsort(x.detach(), dim=-1, descending=True, stable=True)[:, :k]
                e = lp.gather(-1, order)
                total = total + (e * s["g_top"][b, r].double()).sum()
                top[b, r, :order.shape[1]], ids[b, r, :order.shape[1]] = e.detach(), order
            logprob[b, r], entropy[b, r] = a.detach(), h.detach()
            if c["train"]:
                grad[b, r] = torch.autograd.grad(total, x)[0]
    out = [logprob, entropy] + ([top, ids] if k else [])
    return out + ([grad] if c["train"] else [])


def _exact_distill(s):
    c, V = s["case"], s["case"]["V"]
    B, T = c["B"], c["T"]
    loss = torch.zeros(B, T, dtype=torch.float64, device="cuda")
    grad = torch.zeros(B, T, V, dtype=torch.float64, device="cuda")
    for b, n in enumerate(_real(c)):
        for t0 in range(0, n, 64):
            r = slice(t0, min(n, t0 + 64))
            x = s["logits"][b, r].double().requires_grad_()
            logq = torch.log_softmax(x, -1)
            at, t = s["ids"][b, r], s["teacher"][b, r].double()
            if c["tail"] == "renormalize":
                t = torch.log_softmax(t, -1)
                kl = (t.exp() * (t - logq.gather(-1, at))).sum(-1)
            else:
                other = torch.ones_like(x, dtype=torch.bool).scatter_(-1, at, False)
                left = 1 - t.exp().sum(-1)
                rest = torch.logsumexp(logq.masked_fill(~other, NONE), -1)
                kl = (t.exp() * (t - logq.gather(-1, at))).sum(-1) + left * (left.log() - rest)
            loss[b, r] = kl.detach()
            grad[b, r] = torch.autograd.grad(kl, x, s["weights"][b, r].double())[0]
    return [loss, grad]


def _exact_append(s):
    out = []
    for x in (s["k"].double(), s["v"].double()):
        y = torch.zeros(x.shape, dtype=torch.float64, device="cuda")
        for b, n in enumerate(s["n"].tolist()):
            group = x[b, :, :n].reshape(*x[b, :, :n].shape[:-1], -1, 32)
            mag, first = group.abs().max(-1, keepdim=True)
            peak = torch.where((group == -mag).any(-1, keepdim=True), -mag, mag)
            scale = (peak / -8).to(torch.float16).double()
            steps = torch.where(scale == 0, torch.zeros_like(group), group / torch.where(scale == 0, 1.0, scale))
            y[b, :, :n] = (steps.round().clamp(min=-8, max=7) * scale).reshape(x[b, :, :n].shape)
        out.append(y)
    return out


def _exact_attend(s):
    c = s["case"]
    T, Hq, Hkv, D, S = (c[k] for k in ("T", "Hq", "Hkv", "D", "S"))
    out = torch.zeros(c["B"], T, Hq, D, dtype=torch.float64, device="cuda")
    dim = torch.arange(D, device="cuda")
    group, g, j = dim // 32, dim % 32 // 4, dim % 4
    byte, shift = g * (D // 16) + 2 * group + j // 2, 4 * (j % 2)
    for b, (size, n) in enumerate(zip(s["lens"].tolist(), s["n"].tolist())):
        pages = s["table"][b, :-(-size // S)].long()
        for h in range(Hkv):
            kv = []
            for x in ("k", "v"):
                codes = s[x + "_pages"][pages, h].reshape(-1, D // 2)[:size]
                scales = s[x + "_scales"][pages, h].reshape(-1, D // 32)[:size].double()
                kv.append((((codes[:, byte].int() >> shift) & 15) - 8) * scales[:, group])
            mine = slice(h * Hq // Hkv, (h + 1) * Hq // Hkv)
            past = torch.arange(size, device="cuda") > size - n + torch.arange(n, device="cuda")[:, None]
            x = s["q"][b, mine, :n].double() @ kv[0].T / math.sqrt(D)
            out[b, :n, mine] = (torch.softmax(x.masked_fill(past, NONE), -1) @ kv[1]).transpose(0, 1)
    return out


_EXACT = {"score": _exact_score, "distill": _exact_distill, "append": _exact_append, "attend": _exact_attend}


def exact(case, seed):
    global own
    was, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = was
    return _EXACT[case["op"]](s)


# ------------------------------------------------------------------ the work a pass cannot do without
def work(case):
    e, op = _BYTES[case["dtype"]], case["op"]
    if op in ("score", "distill"):
        rows, V, k = sum(_real(case)), case["V"], case["k"]
        grad = case["train"] if op == "score" else True
        # (the gradient's padding rows are written too)
        logits = (rows + (case["B"] * case["T"] if grad else 0)) * V * e
        small = rows * (24 + 12 * k)
        return {"bytes": logits + small, "flops": rows * V * (12 if grad else 6)}
    B, T, Hkv, D = (case[k] for k in ("B", "T", "Hkv", "D"))
    lens, n = _lens(case)
    row = D // 2 + D // 16  # a key or value of a head
    if op == "append":
        # read, written to the cache, and all T slots of the values that come back
        return {"bytes": 2 * Hkv * (sum(n) * (D * e + row) + B * T * D * e), "flops": 20 * sum(n) * Hkv * D}
    Hq = case["Hq"]
    keys = sum(k * (a - k) + k * (k + 1) // 2 for a, k in zip(lens, n))
    return {"bytes": 2 * sum(lens) * Hkv * row + (sum(n) + B * T) * Hq * D * e, "flops": 4 * D * Hq * keys}
