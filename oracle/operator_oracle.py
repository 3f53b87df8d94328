"""64-bit numpy restatements of the operators around the attention kernels:
per-head norms with the rotation, the paged cache, attention over a shared
prefix and the verification of drafted tokens.  Each also returns the bounds
its tests need (sums of magnitudes, decision margins)."""

import numpy as np


def rotate(x, cos, sin):
    """Rotate-half rotation of ``(..., D)`` by ``(..., D/2)`` tables."""
    h = x.shape[-1] // 2
    a, b = x[..., :h], x[..., h:]
    return np.concatenate([a * cos - b * sin, b * cos + a * sin], -1)


def head_norm(x, w, cos, sin, pos, eps):
    """``x`` (B, H, T, D); ``w`` (D,) or None; tables (n_pos, D/2) or None;
    ``pos`` (B, T).  Returns out and the magnitude of the terms it sums."""
    y = x
    if w is not None:
        y = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * w
    if cos is None:
        return y, np.abs(y)
    c, s = cos[pos][:, None], sin[pos][:, None]
    h = y.shape[-1] // 2
    a = np.abs(y)
    m = np.abs(np.concatenate([c, c], -1)) * a + np.abs(np.concatenate([s, s], -1)) * np.roll(a, h, -1)
    return rotate(y, c, s), m


def head_norm_grad(x, w, cos, sin, pos, eps, g):
    """Gradients (dx, dw) of ``sum(head_norm(...) * g)`` and the magnitudes of
    their terms."""
    gm = np.abs(g)
    if cos is not None:
        c, s = cos[pos][:, None], sin[pos][:, None]
        h = x.shape[-1] // 2
        gm = np.abs(np.concatenate([c, c], -1)) * gm + np.abs(np.concatenate([s, s], -1)) * np.roll(gm, h, -1)
        g = rotate(g, c, -s)
    if w is None:
        return g, None, gm, None
    r = 1 / np.sqrt((x * x).mean(-1, keepdims=True) + eps)
    n, u = x * r, g * w
    um = gm * np.abs(w)
    dx = r * (u - n * (u * n).mean(-1, keepdims=True))
    dxm = r * (um + np.abs(n) * (um * np.abs(n)).mean(-1, keepdims=True))
    return dx, (g * n).sum((0, 1, 2)), dxm, (gm * np.abs(n)).sum((0, 1, 2))


def append_slots(lens, new_lens, page_table, page_size):
    """(sequence, token, page, slot) of every appended token."""
    for b, n in enumerate(new_lens):
        for t in range(int(n)):
            at = int(lens[b]) + t
            yield b, t, int(page_table[b, at // page_size]), at % page_size


def gather(pages, table, n):
    """The first n tokens of a page list: (Hkv, n, D)."""
    x = pages[np.asarray(table, dtype=np.int64)]
    x = x.transpose(1, 0, 2, 3).reshape(pages.shape[1], -1, pages.shape[3])
    return x[:, :n]


def prefix_attention(q, k_pages, v_pages, prefix_pages, prefix_len, page_table, lens, query_lens, scale):
    """Returns out (B, T, Hq, D), lse (B, Hq, T), the magnitude ``sum p |v|``
    of each output and the largest ``scale * sum |q k|``."""
    B, Hq, T, D = q.shape
    Hkv, S = k_pages.shape[1], k_pages.shape[2]
    G = Hq // Hkv
    out, mag = np.zeros((B, T, Hq, D)), np.zeros((B, T, Hq, D))
    lse = np.full((B, Hq, T), -np.inf)
    most = 0.0
    kp, vp = (gather(p, prefix_pages[:-(-prefix_len // S)] if prefix_len else [], prefix_len) for p in (k_pages, v_pages))
    for b in range(B):
        n = int(query_lens[b])
        own = [gather(p, page_table[b, :-(-int(lens[b]) // S)], int(lens[b])) for p in (k_pages, v_pages)]
        k, v = np.concatenate([kp, own[0]], 1), np.concatenate([vp, own[1]], 1)
        for t in range(n):
            m = prefix_len + max(0, int(lens[b]) - n + t + 1)
            if m == 0:
                continue
            for h in range(Hq):
                kk, vv = k[h // G, :m], v[h // G, :m]
                s = kk @ q[b, h, t] * scale
                most = max(most, float((np.abs(kk) @ np.abs(q[b, h, t])).max() * scale))
                top = s.max()
                p = np.exp(s - top)
                out[b, t, h] = p @ vv / p.sum()
                mag[b, t, h] = p @ np.abs(vv) / p.sum()
                lse[b, h, t] = top + np.log(p.sum())
    return out, lse, mag, most


def softmax(x, tau):
    if tau <= 0:
        p = np.zeros(x.shape)
        p[int(np.argmax(x))] = 1.0
        return p
    if not np.isfinite(x).any():
        return np.zeros(x.shape)
    e = np.exp((x - x.max()) / tau)
    return e / e.sum()


def verify_check(target, draft, tokens, u, noise, tau, n, accepted, said, logp, tol):
    """Checks one sequence's results (accepted count, tokens, logprobs)
    against the definition in 64 bits.  A decision closer than ``tol``
    (relative) to its threshold may go either way, and the next token may be
    any whose race value is within ``tol`` of the best.  Returns a text for
    what is wrong, or ''."""
    L = tokens.shape[0]
    if not 0 <= accepted <= n:
        return f"accepted {accepted} of {n}"
    for i in range(accepted + (accepted < n)):
        p = softmax(target[i], tau)
        x = int(tokens[i])
        if not 0 <= x < p.shape[0]:
            if i < accepted:
                return f"token {i} outside the vocabulary accepted"
            continue
        q = 1.0 if draft is None else softmax(draft[i], tau)[x]
        lhs, rhs = u[i] * q, p[x]
        if tau <= 0:
            lhs, rhs = 0.0, p[x]
        near = abs(lhs - rhs) <= tol * max(lhs, rhs) and tau > 0
        if not near and (lhs < rhs) != (i < accepted):
            return f"token {i}: u q = {lhs}, p = {rhs}, accepted {accepted}"
    p = softmax(target[accepted], tau)
    r, bar = p, 0.0
    if accepted < n and tau > 0:
        q = np.zeros_like(p)
        if draft is not None:
            q = softmax(draft[accepted], tau)
        elif 0 <= int(tokens[accepted]) < p.shape[0]:
            q[int(tokens[accepted])] = p[int(tokens[accepted])]
        r = np.maximum(p - q, 0)
        bar = tol * np.maximum(p, q)  # what rounding may leave of a difference
        if not (r > 0).any():
            r, bar = p, 0.0
    nxt = int(said[accepted])
    if not 0 <= nxt < p.shape[0]:
        return f"next token {nxt}"
    race, slack = r / noise, (bar + tol * r) / noise
    best = float((race - slack).max())
    if race[nxt] + slack[nxt] < best:
        return f"next token {nxt} with {race[nxt]}, best {race.argmax()} with {race.max()}"
    if list(said[:accepted]) != [int(x) for x in tokens[:accepted]] or any(int(x) != -1 for x in said[accepted + 1:]):
        return f"tokens {said}"
    for i in range(L + 1):
        want = 0.0
        if i <= accepted and tau > 0:
            pi = softmax(target[i], tau)[int(said[i])]
            want = np.log(pi) if pi > 0 else -np.inf
        if not (logp[i] == want or abs(logp[i] - want) <= 1e-5 * (1 + abs(want))):
            return f"logprob {i}: {logp[i]}, expected {want}"
    return ""
