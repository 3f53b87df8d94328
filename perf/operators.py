"""Cases of the serving and training operators around the attention kernels: per-head query / key norms with the
position rotation, the paged key / value cache, attention of a batch that shares a prefix, and the verification of
drafted tokens.

``run`` computes a case in plain fp32 torch operations, or with the library's operators where ``own`` is true;
``exact`` restates it in 64 bits.  Sizes are those of the library's benchmark layer (32 query heads, 8 KV heads,
head_dim 128, vocabulary 151936, documents of 64 to 2048 tokens, sequences up to 32768) and smaller or odd ones."""

import math

import torch

own = False

_DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}
EPS = 1e-6
THETA = 1e6


# ------------------------------------------------------------------ cases
def listed():
    layer = {"Hq": 32, "Hkv": 8, "D": 128}
    return [
        # one decode step of 8 sequences: the norms before the attention, launch latency
        dict(layer, name="norm decode", op="norm", B=8, T=1, dtype="bf16", train=False),
        # the benchmark layer's training step (four rows of 4096 tokens), forward and backward
        dict(layer, name="norm train", op="norm", B=4, T=4096, dtype="bf16", train=True),
        # a small fp32 model in training, odd length, head_dim 64, more query heads per KV head
        dict(name="norm train fp32", op="norm", B=2, T=1021, Hq=16, Hkv=2, D=64, dtype="fp32", train=True),
        # the cache write of one decode step of 64 sequences
        dict(layer, name="append decode", op="append", B=64, T=1, M=512, S=64, dtype="bf16", norm=True),
        # the cache write of a prefill of ragged prompts, no key norm (a Llama-like model)
        dict(layer, name="append prefill", op="append", B=8, T=2047, M=2304, S=16, dtype="fp16", norm=False),
        # four edits of one short document, one token each: latency
        dict(layer, name="prefix small", op="prefix", B=4, T=1, P=257, M=65, S=16, dtype="bf16"),
        # 16 rollouts of one prompt, one token each
        dict(layer, name="prefix rollouts", op="prefix", B=16, T=1, P=4096, M=512, S=64, dtype="bf16"),
        # 64 rollouts of a long document, one token each: the own keys weigh as much as the prefix
        dict(layer, name="prefix long", op="prefix", B=64, T=1, P=32768, M=2048, S=64, dtype="bf16"),
        # the same with drafted tokens (up to five query tokens a sequence): many rows share each key
        dict(layer, name="prefix drafted", op="prefix", B=64, T=5, P=32768, M=2048, S=64, dtype="fp16"),
        # one sequence, three drafted tokens: latency
        dict(name="verify one", op="verify", B=1, L=3, V=151936, dtype="bf16", draft=True),
        # 64 sequences, four drafted tokens from a draft model
        dict(name="verify batch", op="verify", B=64, L=4, V=151936, dtype="bf16", draft=True),
        # fp32 logits, tokens drafted by lookup in the prompt (no draft distribution)
        dict(name="verify lookup", op="verify", B=16, L=7, V=151936, dtype="fp32", draft=False),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    op = rng.choice(["norm", "append", "prefix", "verify"])
    Hq, Hkv = rng.choice([(32, 8), (16, 2), (8, 8), (24, 8), (4, 1)])
    D = rng.choice([64, 128, 128])
    if op == "norm":
        B = _log(rng, 1, 8)
        return dict(op=op, B=B, T=_log(rng, 1, 16384 // B), Hq=Hq, Hkv=Hkv, D=D, dtype=rng.choice(["bf16", "fp16", "fp32"]),
                    train=rng.random() < 0.6)
    if op == "append":
        B = _log(rng, 1, 64)
        T = _log(rng, 1, max(1, 16384 // B))
        return dict(op=op, B=B, T=T, M=T + _log(rng, 1, 512), Hq=Hq, Hkv=Hkv, D=D, S=rng.choice([16, 32, 64, 128]),
                    dtype=rng.choice(["bf16", "fp16"]), norm=rng.random() < 0.5)
    if op == "prefix":
        T = rng.choice([1, 1, 2, 3, 5])
        return dict(op=op, B=_log(rng, 1, 64), T=T, P=_log(rng, 1, 32768), M=_log(rng, T, 2048), Hq=Hq, Hkv=Hkv, D=D,
                    S=rng.choice([16, 32, 64, 128]), dtype=rng.choice(["bf16", "fp16"]))
    return dict(op=op, B=_log(rng, 1, 48), L=rng.randint(1, 5), V=_log(rng, 1000, 151936),
                dtype=rng.choice(["bf16", "fp16", "fp32"]), draft=rng.random() < 0.6)


def _spread(n, lo, hi, phase=0.0):
    """n whole numbers over [lo, hi], evenly spread, in no order."""
    return [lo + int((hi - lo + 1) * ((i * 0.6180339887 + phase) % 1.0)) for i in range(n)]


def _lens(case):
    """Own tokens of each sequence (the new ones among them) and how many of its T query tokens are real."""
    B, T, M = case["B"], case["T"], case["M"]
    n = [T] * B if T == 1 else _spread(B, 1, T, 0.9)
    if case["op"] == "append":
        return _spread(B, 0, M - T, 0.4), n
    lens = _spread(B, 1, M, 0.5)
    return [max(a, b) for a, b in zip(lens, n)], n


# ------------------------------------------------------------------ inputs
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _heads(g, B, T, H, D, dt, scale=1.0):
    """What a projection gives: (B, T, H, D) in memory, seen as (B, H, T, D)."""
    return (torch.randn(B, T, H, D, generator=g, device="cuda") * scale).to(dt).transpose(1, 2)


def _weight(g, D, dt):
    return (1 + 0.2 * torch.randn(D, generator=g, device="cuda")).to(dt)


def _rope(n, D):
    inv = THETA ** (-torch.arange(0, D, 2, device="cuda", dtype=torch.float64) / D)
    a = torch.arange(n, device="cuda", dtype=torch.float64)[:, None] * inv
    return a.cos().float().contiguous(), a.sin().float().contiguous()


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def prepare(case, seed):
    g, dt, op = _gen(seed), _DT[case["dtype"]], case["op"]
    s = {"case": case}
    if op == "verify":
        B, L, V = case["B"], case["L"], case["V"]
        base = 3 * torch.randn(B, L + 1, V, generator=g, device="cuda")
        drafted = base[:, :L] + 0.6 * torch.randn(B, L, V, generator=g, device="cuda")
        race = torch.empty(B, L, V, device="cuda").exponential_(generator=g)
        s["target"] = base.to(dt)
        s["draft"] = drafted.to(dt) if case["draft"] else None
        s["tau"] = 0.6 + 0.4 * torch.rand(B, generator=g, device="cuda")
        s["tau"][3::4] = 0.0  # every fourth sequence decodes greedily
        pick = torch.softmax(drafted / torch.where(s["tau"] > 0, s["tau"], 0.05)[:, None, None], -1) / race
        s["tokens"] = pick.argmax(-1)
        s["n"] = _ints([L] * B if B < 4 else _spread(B, max(1, L - 2), L, 0.9))
        s["u"] = torch.rand(B, L, generator=g, device="cuda")
        s["noise"] = torch.empty(B, V, device="cuda").exponential_(generator=g).clamp_min_(1e-10)
        return s
    B, T, Hq, Hkv, D = (case[k] for k in ("B", "T", "Hq", "Hkv", "D"))
    if op == "norm":
        s["q"], s["k"] = _heads(g, B, T, Hq, D, dt, 1.5), _heads(g, B, T, Hkv, D, dt, 1.5)
        s["wq"], s["wk"] = _weight(g, D, dt), _weight(g, D, dt)
        s["rope"] = _rope(T + 64, D)
        start = torch.randint(0, 64, (B, 1), generator=g, device="cuda")
        s["pos"] = start + torch.arange(T, device="cuda")
        if case["train"]:
            s["gq"], s["gk"] = _heads(g, B, T, Hq, D, dt), _heads(g, B, T, Hkv, D, dt)
            for name in ("q", "k", "wq", "wk"):
                s[name].requires_grad_(own)
        return s
    S, M = case["S"], case["M"]
    P = case.get("P", 0)
    lens, n = _lens(case)
    per, shared = -(-M // S), -(-P // S)
    pages = shared + B * per + 2
    order = torch.randperm(pages, generator=g, device="cuda").int()
    s["k_pages"] = torch.randn(pages, Hkv, S, D, generator=g, device="cuda", dtype=dt)
    s["v_pages"] = torch.randn(pages, Hkv, S, D, generator=g, device="cuda", dtype=dt)
    s["table"] = order[shared:shared + B * per].reshape(B, per).contiguous()
    s["lens"], s["n"] = _ints(lens), _ints(n)
    if op == "append":
        s["k"], s["v"] = _heads(g, B, T, Hkv, D, dt, 1.5), _heads(g, B, T, Hkv, D, dt)
        s["wk"] = _weight(g, D, dt) if case["norm"] else None
        s["rope"] = _rope(M + 64, D)
        s["pos"] = torch.randint(0, 64, (B, 1), generator=g, device="cuda") + s["lens"][:, None] + torch.arange(T, device="cuda")
        return s
    s["prefix"] = order[:shared].contiguous()
    s["q"] = _heads(g, B, T, Hq, D, dt, 2.0)  # sharper than noise, as trained heads are
    return s


# ------------------------------------------------------------------ plain forms, 32 bits
def _rotate(y, cos, sin):
    a, b = y.chunk(2, -1)
    return torch.cat((a * cos - b * sin, b * cos + a * sin), -1)


def _norm(x, w):
    r = torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS)
    return x * r * w


def _norm_grad(x, w, g, cos, sin):
    g = _rotate(g, cos, -sin)
    r = torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS)
    n, u = x * r, g * w
    return r * (u - n * (u * n).mean(-1, keepdim=True)), (g * n).sum((0, 1, 2))


def _plain_norm(s):
    cos, sin = (t[s["pos"]].unsqueeze(1) for t in s["rope"])
    dt = s["q"].dtype
    q, k, wq, wk = (s[n].float() for n in ("q", "k", "wq", "wk"))
    out = [_rotate(_norm(q, wq), cos, sin).to(dt), _rotate(_norm(k, wk), cos, sin).to(dt)]
    if s["case"]["train"]:
        dq, dwq = _norm_grad(q, wq, s["gq"].float(), cos, sin)
        dk, dwk = _norm_grad(k, wk, s["gk"].float(), cos, sin)
        out += [dq.to(dt), dk.to(dt), dwq.to(dt), dwk.to(dt)]
    return out


def _plain_append(s):
    T, S = s["case"]["T"], s["case"]["S"]
    k = s["k"].float()
    if s["wk"] is not None:
        k = _norm(k, s["wk"].float())
    cos, sin = (t[s["pos"]].unsqueeze(1) for t in s["rope"])
    k = _rotate(k, cos, sin).to(s["k"].dtype)
    t = torch.arange(T, device="cuda")
    at = s["lens"][:, None] + t
    b, t = torch.nonzero(t < s["n"][:, None], as_tuple=True)
    at = at[b, t]
    page = s["table"][b, at // S].long()
    s["k_pages"][page, :, at % S] = k[b, :, t]
    s["v_pages"][page, :, at % S] = s["v"][b, :, t]
    return [s["k_pages"], s["v_pages"]]


def _gathered(pages, table):
    """(..., pages of a row) -> (..., Hkv, keys, D) in fp32."""
    x = pages[table.long()].float().movedim(-3, -4)
    return x.flatten(-3, -2)


def _plain_prefix(s):
    c, q = s["case"], s["q"].float()
    B, T, Hq, Hkv, D, P = (c[k] for k in ("B", "T", "Hq", "Hkv", "D", "P"))
    G = Hq // Hkv
    q = (q * D ** -0.5).reshape(B, Hkv, G * T, D)
    kp, vp = (_gathered(s[n], s["prefix"])[:, :P] for n in ("k_pages", "v_pages"))
    ko, vo = (_gathered(s[n], s["table"]) for n in ("k_pages", "v_pages"))
    across = q.transpose(0, 1).reshape(Hkv, B * G * T, D)
    sp = (across @ kp.transpose(-1, -2)).reshape(Hkv, B, G * T, P).transpose(0, 1)
    so = q @ ko.transpose(-1, -2)
    t = torch.arange(T, device="cuda").repeat(G)
    last = s["lens"][:, None] - s["n"][:, None] + t  # the row's last own key
    live = t < s["n"][:, None]
    seen = torch.arange(ko.shape[2], device="cuda") <= last[..., None]
    so = so.masked_fill(~seen[:, None], float("-inf"))
    m = torch.maximum(sp.amax(-1, keepdim=True), so.amax(-1, keepdim=True))
    ep, eo = torch.exp(sp - m), torch.exp(so - m)
    total = ep.sum(-1, keepdim=True) + eo.sum(-1, keepdim=True)
    op = (ep.transpose(0, 1).reshape(Hkv, B * G * T, P) @ vp).reshape(Hkv, B, G * T, D).transpose(0, 1)
    o = (op + eo @ vo) / total
    o = o.masked_fill(~live[:, None, :, None], 0.0).reshape(B, Hq, T, D)
    return o.transpose(1, 2).to(s["q"].dtype)


def _plain_verify(s):
    L, V = s["case"]["L"], s["case"]["V"]
    tau = s["tau"][:, None, None]
    warm = torch.where(tau > 0, tau, 1.0)
    words = torch.arange(V, device="cuda")

    def probabilities(logits):
        x = logits.float() / warm
        e = torch.exp(x - x.amax(-1, keepdim=True))
        p = e / e.sum(-1, keepdim=True)
        return torch.where(tau > 0, p, (words == logits.float().argmax(-1, keepdim=True)).float())

    p = probabilities(s["target"])
    tokens = s["tokens"]
    q = probabilities(s["draft"]) if s["draft"] is not None else (words == tokens[..., None]).float()
    px, qx = (x.gather(-1, tokens[..., None])[..., 0] for x in (p[:, :L], q))
    i = torch.arange(L + 1, device="cuda")
    good = (s["u"] * qx < px) & (i[:L] < s["n"][:, None])
    a = good.long().cumprod(-1).sum(-1)
    pa = p.gather(1, a[:, None, None].expand(-1, 1, V))[:, 0]
    qa = q.gather(1, a.clamp_max(L - 1)[:, None, None].expand(-1, 1, V))[:, 0]
    r = torch.where((a < s["n"])[:, None], (pa - qa).clamp_min(0), pa)
    r = torch.where((r > 0).any(-1, keepdim=True), r, pa)
    nxt = torch.where(r > 0, r / s["noise"], 0.0).argmax(-1)
    said = torch.cat((tokens, nxt[:, None]), 1).scatter(1, a[:, None], nxt[:, None])
    said = torch.where(i <= a[:, None], said, -1)
    logp = torch.log(p.gather(-1, said.clamp_min(0)[..., None])[..., 0])
    return [a.int(), said, torch.where(i <= a[:, None], logp, 0.0)]


_PLAIN = {"norm": _plain_norm, "append": _plain_append, "prefix": _plain_prefix, "verify": _plain_verify}


# ------------------------------------------------------------------ the library's operators
def _own_norm(ab, s):
    if not s["case"]["train"]:
        return ab.qk_norm_rope(s["q"], s["k"], s["wq"], s["wk"], s["rope"], s["pos"], eps=EPS)
    out = ab.qk_norm_rope(s["q"], s["k"], s["wq"], s["wk"], s["rope"], s["pos"], eps=EPS)
    grads = torch.autograd.grad(out, (s["q"], s["k"], s["wq"], s["wk"]), (s["gq"], s["gk"]))
    return [out[0].detach(), out[1].detach(), *grads]


def _own_append(ab, s):
    ab.paged_append(s["k"], s["v"], s["k_pages"], s["v_pages"], s["table"], s["lens"], rope=s["rope"], positions=s["pos"],
                    new_lens=s["n"], key_weight=s["wk"], eps=EPS)
    return [s["k_pages"], s["v_pages"]]


def _own_prefix(ab, s):
    return ab.shared_prefix_attention(s["q"], s["k_pages"], s["v_pages"], s["prefix"], s["case"]["P"], s["table"], s["lens"],
                                      query_lens=s["n"])


def _own_verify(ab, s):
    return ab.verify_draft(s["target"], s["tokens"], s["u"], s["noise"], draft_logits=s["draft"], draft_lens=s["n"],
                           temperature=s["tau"])


_OWN = {"norm": _own_norm, "append": _own_append, "prefix": _own_prefix, "verify": _own_verify}


def run(state):
    op = state["case"]["op"]
    if not own:
        with torch.no_grad():
            return _PLAIN[op](state)
    import autoindexer_b200

    return _OWN[op](autoindexer_b200, state)


# ------------------------------------------------------------------ 64 bits, from the definitions
def _turned(x, table, pos):
    """Each pair (i, i + D/2) of the last axis as a complex number, turned by its position's angle."""
    cos, sin = (t.double()[pos] for t in table)
    h = x.shape[-1] // 2
    z = torch.complex(x[..., :h].contiguous(), x[..., h:].contiguous()) * torch.complex(cos, sin)
    return torch.cat((z.real, z.imag), -1)


def _scaled(x, w):
    d = x.shape[-1]
    return x / ((x ** 2).sum(-1, keepdim=True) / d + EPS) ** 0.5 * w


def _exact_norm(s):
    out, grads, weights = [], [], []
    for x, w, g in (("q", "wq", "gq"), ("k", "wk", "gk")):
        a = s[x].detach().double().requires_grad_()
        b = s[w].detach().double().requires_grad_()
        y = _turned(_scaled(a, b), s["rope"], s["pos"][:, None])
        out.append(y.detach())
        if s["case"]["train"]:
            da, db = torch.autograd.grad(y, (a, b), s[g].double())
            grads.append(da)
            weights.append(db)
    return out + grads + weights


def _exact_append(s):
    S, kp, vp = s["case"]["S"], s["k_pages"].double(), s["v_pages"].double()
    k = s["k"].double()
    k = _turned(k if s["wk"] is None else _scaled(k, s["wk"].double()), s["rope"], s["pos"][:, None])
    for b, (first, n) in enumerate(zip(s["lens"].tolist(), s["n"].tolist())):
        at = torch.arange(first, first + n, device="cuda")
        page = s["table"][b].long()[at // S]
        kp[page, :, at % S] = k[b, :, :n].transpose(0, 1)
        vp[page, :, at % S] = s["v"][b, :, :n].double().transpose(0, 1)
    return [kp, vp]


def _exact_prefix(s):
    c = s["case"]
    T, Hq, Hkv, D, P = (c[k] for k in ("T", "Hq", "Hkv", "D", "P"))
    out = torch.zeros(c["B"], T, Hq, D, dtype=torch.float64, device="cuda")
    k, v = s["k_pages"], s["v_pages"]
    flat = lambda x, pages, n: x[pages.long()].transpose(1, 2).reshape(-1, Hkv, D)[:n].double()  # noqa: E731
    kp, vp = (flat(x, s["prefix"], P) for x in (k, v))
    for b, (size, n) in enumerate(zip(s["lens"].tolist(), s["n"].tolist())):
        kb, vb = (torch.cat((shared, flat(x, s["table"][b], size))) for x, shared in ((k, kp), (v, vp)))
        past = torch.arange(P + size, device="cuda") > P + size - n + torch.arange(n, device="cuda")[:, None]
        for h in range(Hkv):
            mine = slice(h * Hq // Hkv, (h + 1) * Hq // Hkv)
            x = s["q"][b, mine, :n].double() @ kb[:, h].T / math.sqrt(D)
            out[b, :n, mine] = (torch.softmax(x.masked_fill(past, -math.inf), -1) @ vb[:, h]).transpose(0, 1)
    return out


def _exact_verify(s):
    B, L = s["case"]["B"], s["case"]["L"]
    a = torch.zeros(B, dtype=torch.int32, device="cuda")
    said = torch.full((B, L + 1), -1, dtype=torch.int64, device="cuda")
    logp = torch.zeros(B, L + 1, dtype=torch.float64, device="cuda")

    def distribution(row, t):
        if t > 0:
            return torch.softmax(row.double() / t, -1)
        p = torch.zeros(row.shape[-1], dtype=torch.float64, device="cuda")
        p[row.float().argmax()] = 1
        return p

    for b, (t, n) in enumerate(zip(s["tau"].tolist(), s["n"].tolist())):
        i = 0
        while True:
            p = distribution(s["target"][b, i], t)
            if i == n:
                r = p
                break
            x = int(s["tokens"][b, i])
            if s["draft"] is None:
                q = torch.zeros_like(p)
                q[x] = 1
            else:
                q = distribution(s["draft"][b, i], t)
            if not bool(s["u"][b, i].double() * q[x] < p[x]):
                r = (p - q).clamp_min(0)
                break
            said[b, i], logp[b, i] = x, p[x].log()
            i += 1
        if not bool((r > 0).any()):
            r = p
        nxt = int((r / s["noise"][b].double()).argmax())
        a[b], said[b, i], logp[b, i] = i, nxt, p[nxt].log()
    return [a, said, logp]


_EXACT = {"norm": _exact_norm, "append": _exact_append, "prefix": _exact_prefix, "verify": _exact_verify}


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
    if op == "verify":
        B, L, V = case["B"], case["L"], case["V"]
        rows = (L + 1) + (L if case["draft"] else 0)
        return {"bytes": B * V * (rows * e + 4), "flops": 4 * B * V * rows}
    B, T, Hq, Hkv, D = (case[k] for k in ("B", "T", "Hq", "Hkv", "D"))
    if op == "norm":
        x = B * T * (Hq + Hkv) * D
        table = (T + 64) * D * 4 + 8 * B * T
        return {"bytes": x * e * (5 if case["train"] else 2) + table, "flops": x * (30 if case["train"] else 10)}
    lens, n = _lens(case)
    if op == "append":
        new = sum(n) * Hkv * D
        return {"bytes": 4 * new * e + sum(n) * (4 * D + 8), "flops": 10 * new}
    keys = sum(k * case["P"] + k * (a - k) + k * (k + 1) // 2 for a, k in zip(lens, n))
    kv = (case["P"] + sum(lens)) * Hkv * D * 2
    return {"bytes": (kv + 2 * sum(n) * Hq * D) * e, "flops": 4 * D * Hq * keys}
