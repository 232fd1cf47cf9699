"""Float64 numpy definitions of the quantized-page operators, for the tests."""
import numpy as np


def block_bytes(bits, hd, page):
    return page * (2 * (hd * bits // 8) + 8)


def split_block(pool, bits, hd, page):
    """(codes K, codes V) as integers the scales multiply, (scales K, scales
    V), from a uint8 pool (n_pages, n_kv, block_bytes)."""
    nb = hd * bits // 8
    out = []
    for i in (0, 1):
        raw = pool[:, :, i * page * nb:(i + 1) * page * nb].reshape(*pool.shape[:2], page, nb)
        if bits == 8:
            c = raw.view(np.int8).astype(np.int64)
        else:
            c = np.empty((*raw.shape[:3], hd), np.int64)
            c[..., 0::2] = 2 * (raw & 15).astype(np.int64) - 15
            c[..., 1::2] = 2 * (raw >> 4).astype(np.int64) - 15
        a = 2 * page * nb + 4 * page * i
        s = np.ascontiguousarray(pool[:, :, a:a + 4 * page]).view(np.float32)
        out.append((c, s))
    return out


def rows_of(pool, table, length, bits, hd, page):
    """K and V of tokens 0 .. length - 1: (length, n_kv, hd) float64."""
    res = []
    t = np.arange(length)
    pg, off = table[t // page], t % page
    for c, s in split_block(pool, bits, hd, page):
        res.append(c[pg, :, off].astype(np.float64) * s[pg, :, off].astype(np.float64)[..., None])
    return res


def norm_rope(x, w, cos, sin, eps):
    """x (n, heads, hd) float64; cos / sin (n, hd / 2)."""
    if w is not None:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * w
    h = x.shape[-1] // 2
    a, b, c, s = x[..., :h], x[..., h:], cos[:, None], sin[:, None]
    return np.concatenate([a * c - b * s, a * s + b * c], -1)


def attend(q, k, v, length, scale, cap=0.0, slopes=None, window=0, prefix=0):
    """q (n, heads, hd), k / v (length, n_kv, hd), all float64."""
    n, nh, hd = q.shape
    out = np.zeros((n, nh, hd))
    if length == 0:
        return out
    pos = np.arange(length - n, length)
    j = np.arange(length)
    see = j[None] <= pos[:, None]
    if window:
        see &= j[None] > pos[:, None] - window
    see |= (j < prefix)[None]
    for h in range(nh):
        kv = h // (nh // k.shape[1])
        x = q[:, h] @ k[:, kv].T * scale
        if cap:
            x = cap * np.tanh(x / cap)
        if slopes is not None:
            x = x - slopes[h] * np.abs(pos[:, None] - j[None])
        x = np.where(see, x, -np.inf)
        m = x.max(-1, keepdims=True)
        p = np.exp(x - np.where(np.isneginf(m), 0, m))
        d = p.sum(-1, keepdims=True)
        vv = np.where(see.any(0)[:, None], v[:, kv], 0)
        out[:, h] = (p @ vv) / np.where(d == 0, 1, d)
    return out


def adjust(logits, history, repeat, frequency, presence, bias, allowed):
    """One row in float64. history: tokens; bias: (token, value) pairs in
    order; allowed: bool (vocab) or None."""
    x = logits.astype(np.float64).copy()
    V = x.size
    tok, n = np.unique([t for t in history if 0 <= t < V], return_counts=True)
    for t, c in zip(tok.astype(int), n):
        x[t] = x[t] / repeat if x[t] > 0 else x[t] * repeat
        x[t] -= frequency * c + presence
    for t, b in dict(bias).items():
        if 0 <= t < V:
            x[t] += b
    if allowed is not None:
        x[~allowed] = -np.inf
    return x
