"""64-bit numpy restatements of the operators for rollouts and what is learnt
from them: token log-probabilities with their gradient, distillation from a
teacher's likeliest words, and the cache in 4 bits.  Rows are taken one at a
time; each function also returns the magnitudes its tests' bounds need."""

import numpy as np


def log_softmax(x, tau):
    """``ln softmax(x / tau)`` of one row; ``None`` without an unmasked word,
    NaN everywhere for a row with a NaN or a +inf."""
    if np.isnan(x).any() or (x == np.inf).any():
        return np.full(x.shape, np.nan)
    if (x == -np.inf).all():
        return None
    z = (x - x.max()) / tau
    return z - np.log(np.exp(z).sum())


def entropy_of(lp):
    p = np.exp(lp)
    return float(-(p * np.where(p > 0, lp, 0.0)).sum())


def score_row(x, token, tau, k):
    """(logprob, entropy, top ids, top logprobs) of one row."""
    ids, top = np.full(k, -1, dtype=np.int64), np.full(k, -np.inf)
    if not 0 <= token < x.shape[0]:
        return 0.0, 0.0, ids, top
    lp = log_softmax(x, tau)
    if lp is None:
        return -np.inf, 0.0, ids, top
    if np.isnan(lp).any():
        return np.nan, np.nan, ids, np.full(k, np.nan)
    order = np.lexsort((np.arange(x.shape[0]), -x))[:k]
    order = order[x[order] > -np.inf]
    ids[:len(order)], top[:len(order)] = order, lp[order]
    return float(lp[token]), entropy_of(lp), ids, top


def score_row_grad(x, token, tau, ids, g_logprob, g_entropy, g_top):
    """Gradient of one row, and the magnitude of the terms that each entry sums."""
    d, mag = np.zeros(x.shape), np.zeros(x.shape)
    if not 0 <= token < x.shape[0] or not (g_logprob or g_entropy or np.any(g_top)):
        return d, mag
    lp = log_softmax(x, tau)
    if lp is None:
        return d, mag
    if np.isnan(lp).any():
        return np.full(x.shape, np.nan), mag
    p, h = np.exp(lp), entropy_of(lp)
    flat = np.where(p > 0, lp, 0.0)
    live = ids >= 0
    total = g_logprob + g_top[live].sum()
    d -= p * (total + g_entropy * (flat + h))
    mag += p * (abs(g_logprob) + np.abs(g_top[live]).sum() + abs(g_entropy) * (np.abs(flat) + h))
    for v, g in [(token, g_logprob), *zip(ids[live], g_top[live])]:
        d[v] += g
        mag[v] += abs(g)
    return d / tau, mag / tau


def distill_entries(ids, t, vocab):
    """Indices of the entries that count."""
    seen, keep = set(), []
    for j, v in enumerate(ids):
        if 0 <= v < vocab and t[j] != -np.inf and int(v) not in seen:
            seen.add(int(v))
            keep.append(j)
    return keep


def distill_row(x, ids, t, tau, tail, weight=1.0):
    """(loss, gradient of weight * loss, magnitude of its terms, magnitude of
    the loss's terms) of one row."""
    d, mag = np.zeros(x.shape), np.zeros(x.shape)
    keep = distill_entries(ids, t, x.shape[0])
    if not keep or weight == 0:
        return 0.0, d, mag, 0.0
    at, t = ids[keep], t[keep]
    lq = log_softmax(x, tau)
    if lq is None:
        return np.inf, d, mag, 0.0
    if np.isnan(lq).any() or np.isnan(t).any():
        return np.nan, np.full(x.shape, np.nan), mag, 0.0
    if tail == "renormalize":
        t = t - t.max()
        t = t - np.log(np.exp(t).sum())
    p, q = np.exp(t), np.exp(lq)
    other = np.ones(x.shape, dtype=bool)
    other[at] = False
    left = 1 - p.sum() if tail == "bucket" else 0.0
    if left <= 2.0 ** -23 + 2.0 ** -24 * (p * np.abs(t)).sum() or not (x[other] > -np.inf).any():
        left = 0.0
    some = p > 0
    loss = float((p[some] * (t[some] - lq[at][some])).sum())
    big = float((p[some] * (np.abs(t[some]) + np.abs(lq[at][some]))).sum())
    mass = p.sum() + left
    d += mass * q
    mag += mass * q
    if left > 0:
        # (relative to their largest one: far below the listed words a sum's logarithm would vanish in lq)
        z = (x[other] - x[other].max()) / tau
        share = np.exp(z) / np.exp(z).sum()
        rest = lq[other].max() + np.log(np.exp(z).sum())
        loss += left * (np.log(left) - rest)
        big += left * (abs(np.log(left)) + abs(rest))
        d[other] -= left * share
        mag[other] += left * share
    d[at] -= p
    mag[at] += p
    return loss, weight / tau * d, abs(weight) / tau * mag, big


# ------------------------------------------------------------------ the 4-bit format
def byte_of(D):
    """(byte, shift, group) of each dim of a row."""
    d = np.arange(D)
    c, g, j = d // 32, d % 32 // 4, d % 4
    return g * (D // 16) + 2 * c + j // 2, 4 * (j % 2), c


def quantize(x):
    """``x`` (..., D) float64 -> (codes uint8 (..., D / 2), scales float16 (..., D / 32))."""
    D = x.shape[-1]
    v = x.reshape(*x.shape[:-1], D // 32, 32)
    with np.errstate(invalid="ignore", over="ignore"):
        top, low = v.max(-1), v.min(-1)
        scale = np.clip(np.where(top > -low, top, low) / -8, -65504, 65504).astype(np.float16)
    bad = ~np.isfinite(v).all(-1)
    scale[bad] = np.nan
    d = scale.astype(np.float64)[..., None]
    whole = np.isfinite(d) & (d != 0)
    with np.errstate(invalid="ignore", divide="ignore"):
        q = np.where(whole, np.rint(np.where(whole, v, 0.0) / np.where(whole, d, 1.0)), 0.0)
    codes = (np.clip(q, -8, 7) + 8).astype(np.uint8).reshape(x.shape)
    byte, shift, _ = byte_of(D)
    out = np.zeros((*x.shape[:-1], D // 2), dtype=np.uint8)
    for i in range(D):
        out[..., byte[i]] |= codes[..., i] << np.uint8(shift[i])
    return out, scale


def values(codes, scales):
    """What codes (..., D / 2) and scales (..., D / 32) stand for, float64."""
    D = 2 * codes.shape[-1]
    byte, shift, group = byte_of(D)
    return (((codes[..., byte] >> shift.astype(np.uint8)) & 15).astype(np.float64) - 8) * scales.astype(np.float64)[..., group]


def attention(q, k, v, seen, scale):
    """``q`` (T, D) of one head over keys and values (n, D), row t over the
    first ``seen[t]``: out (T, D), lse (T,), the magnitude ``sum p |v|`` and the
    largest ``scale * sum |q k|``."""
    out, lse, mag, most = np.zeros(q.shape), np.full(q.shape[0], -np.inf), np.zeros(q.shape), 0.0
    for t, n in enumerate(seen):
        if n <= 0:
            continue
        s = k[:n] @ q[t] * scale
        most = max(most, float((np.abs(k[:n]) @ np.abs(q[t])).max() * scale))
        p = np.exp(s - s.max())
        out[t], mag[t] = p @ v[:n] / p.sum(), p @ np.abs(v[:n]) / p.sum()
        lse[t] = s.max() + np.log(p.sum())
    return out, lse, mag, most
