"""64-bit restatement (numpy) of the operators on rows of logits, for tests/test_gpu_logits.py."""
import numpy as np

GRID = 2.0 ** 30
LOG2E = np.float32(1.4426950408889634)


def unpack_mask(words, vocab):
    """bool [vocab] of u64 mask words (bit i % 64 of word i / 64)."""
    w = np.asarray(words).view(np.uint64)
    i = np.arange(vocab)
    return ((w[i // 64] >> (i % 64).astype(np.uint64)) & np.uint64(1)).astype(bool)


def pack_mask(bits):
    n = len(bits)
    b = np.zeros((n + 63) // 64 * 64, dtype=np.uint8)
    b[:n] = bits
    return np.packbits(b, bitorder="little").view(np.int64)


def allowed_logits(z, bits=None):
    z = np.asarray(z, np.float64).copy()
    z[np.isnan(z)] = -np.inf
    if bits is not None:
        z[~bits] = -np.inf
    return z


def order(z):
    """Ids by (logit descending, id ascending); -0 and +0 are equal."""
    return np.argsort(-(z + 0.0), kind="stable")


def logsumexp(x):
    m = x.max() if len(x) else -np.inf
    if not np.isfinite(m):
        return m
    return m + np.log(np.exp(x - m).sum())


def top(z, k, temperature, bits=None):
    z = allowed_logits(z, bits)
    o = order(z)[:k]
    o = o[z[o] > -np.inf]
    values, ids = np.full(k, -np.inf), np.full(k, -1, np.int32)
    values[:len(o)], ids[:len(o)] = z[o], o
    return values, ids, logsumexp(z / temperature)


def distill(z, ids, t, lse, temperature, weight=1.0):
    """(loss, stats, grad, magnitude of the loss's terms) of one row."""
    z, t = np.asarray(z, np.float64), np.asarray(t, np.float64)
    have = np.asarray(ids) >= 0
    ids, t = np.asarray(ids)[have], t[have] / temperature
    x = z / temperature
    L = logsumexp(x)
    logq = x - L
    norm = logsumexp(t) if lse is None else float(lse)
    logp = t - norm if lse is not None or norm > -np.inf else np.full(len(t), -np.inf)
    p = np.exp(logp)
    with np.errstate(invalid="ignore"):
        terms = np.where(p > 0, p * (logp - logq[ids]), 0.0)
    loss, mag, off = terms.sum(), np.abs(terms).sum(), 1.0
    whole = p.sum()  # the loss is a sum over the entries alone: its p are a part (or nothing) of a distribution
    if lse is not None:
        p_r = 1.0 - p.sum()
        out = np.ones(len(z), bool)
        out[ids] = False
        q_r = np.exp(logq[out]).sum()
        if p_r > 0 and q_r > 0:
            loss += p_r * (np.log(p_r) - np.log(q_r))
            mag += abs(p_r * np.log(p_r)) + abs(p_r * np.log(q_r))
            off, whole = 1.0 - p_r / q_r, None
    g = np.exp(logq) * (off if whole is None else whole)
    g[ids] = np.exp(logq[ids]) * (1.0 if whole is None else whole) - p
    return loss, (L, off), g * weight / temperature, mag


def sample_weights(z, temperature, top_k, top_p, min_p, bits=None, nudge=0.0):
    """Kept weights per id in units of 2^-30.  `nudge` moves the limits of top-p and min-p by that much
    of themselves (for a cut that lies within rounding of its limit)."""
    z = allowed_logits(z, bits)
    V = len(z)
    kept = np.zeros(V)
    if V == 0 or z.max() == -np.inf:
        return kept
    m = z.max()
    if not temperature > 0:
        kept[int(order(z)[0])] = GRID
        return kept
    with np.errstate(invalid="ignore", over="ignore", divide="ignore"):
        scale = LOG2E / np.float32(temperature)
        d = ((z.astype(np.float32) - np.float32(m)) * scale).astype(np.float64)
    d[z == m] = 0.0
    e = np.where(z == -np.inf, 0.0, np.exp2(np.where(np.isnan(d), -np.inf, d)))
    w = np.rint(e * GRID)
    o = order(z)
    ws = w[o].copy()
    if top_k > 0:
        ws[top_k:] = 0.0
    if top_p < 1.0:
        need = max(1.0, np.ceil(float(np.float32(top_p)) * ws.sum()) * (1.0 + nudge))
        c = np.cumsum(ws)
        ws[(c - ws) >= need] = 0.0
    mp = float(np.float32(min_p))
    ws[e[o] < min(mp, 1.0) * (1.0 + min(nudge, 0.0) if mp >= 1.0 else 1.0 + nudge)] = 0.0
    kept[o] = ws
    return kept
