"""Plain 64-bit forms of the 8-bit key/value cache's operators (include/pxq.h,
"attention over an 8-bit key/value cache"), one sequence and head at a time."""
import numpy as np

BLOCK = 32


def values(x):
    """Rows [t, H, D] fp32 -> the fp32 values the cache stands for."""
    x = np.asarray(x, np.float32)
    out = np.empty_like(x)
    for b in range(0, x.shape[0], BLOCK):
        for h in range(x.shape[1]):
            blk = x[b:b + BLOCK, h].astype(np.float64)
            if not np.isfinite(blk).all():
                out[b:b + BLOCK, h] = np.nan
                continue
            a = np.abs(blk).max() if blk.size else 0.0
            if a < 2.0 ** -118:
                out[b:b + BLOCK, h] = 0
                continue
            d = np.float64(np.float32(a / 127.0))
            out[b:b + BLOCK, h] = (np.rint(blk / d) * d).astype(np.float32)
    return out


def attention(q, k, v, heads, causal):
    """q [n, heads, D], k, v [t, H, D] (values) -> out [n, heads, D], weights [H, t], in 64 bits."""
    n, _, D = q.shape
    t, H = k.shape[:2]
    G = heads // H
    out = np.zeros((n, heads, D))
    w = np.zeros((H, t))
    for i in range(n):
        lim = max(0, t - n + i + 1) if causal else t
        if lim == 0:
            continue
        for h in range(heads):
            z = k[:lim, h // G].astype(np.float64) @ q[i, h].astype(np.float64) / np.sqrt(D)
            p = np.exp(z - z.max())
            p /= p.sum()
            out[i, h] = p @ v[:lim, h // G].astype(np.float64)
            w[h // G, :lim] += p
    return out, w


def kept(w, keep, recent):
    """Indices that an eviction keeps of one (sequence, head) with weights w [t]."""
    t = len(w)
    c = min(t, keep)
    rec = min(recent, c)
    old = t - rec
    key = np.where(np.isnan(w[:old]), -np.inf, w[:old]).astype(np.float64)
    best = np.argsort(-key, kind="stable")[:c - rec]
    return np.sort(np.concatenate([best, np.arange(old, t)]).astype(np.int64))
