"""Attention over a key-value cache, and eviction from it, in plain float64: what the tests of those entry points
compare with. Arrays hold values (widened 16-bit operands); a query's unseen keys take no part at all."""
import numpy as np


def seen(L, length, window, sinks, S):
    """(L, S): which keys each query sees."""
    p = np.arange(L)[:, None] + length - L
    j = np.arange(S)[None, :]
    return (j <= p) & (j < length) & ((j > p - window) | (j < sinks))


def attend(q, keys, values):
    """One query's (result, weights, sum of weight x |value|, largest sum of |products| behind a score)."""
    s = keys @ q / np.sqrt(q.size)
    with np.errstate(invalid="ignore", over="ignore"):
        w = np.exp(s - s.max())
        w = w / w.sum()
        return w @ values, w, w @ np.abs(values), float(np.max(np.abs(keys) @ np.abs(q))) / np.sqrt(q.size)


def attention(q, k, v, lens=None, window=None, sinks=0, prefix_k=None, prefix_v=None):
    """-> (out (N, H, L, D), weights (N, Hk, S), scale of the output's errors (N, H, L, D), the scores' (N, H, L, 1))."""
    N, H, L, D = q.shape
    Hk, S = k.shape[1], k.shape[2]
    G = H // Hk
    window = S if window is None else window
    out, size, score = np.zeros(q.shape), np.zeros(q.shape), np.zeros((N, H, L, 1))
    weights = np.zeros((N, Hk, S))
    for n in range(N):
        length = S if lens is None else min(max(int(lens[n]), 0), S)
        see = seen(L, length, window, sinks, S)
        for h in range(H):
            for i in range(L):
                at = np.nonzero(see[i])[0]
                keys, values = k[n, h // G, at], v[n, h // G, at]
                if prefix_k is not None:
                    keys, values = np.concatenate([prefix_k[0, h // G], keys]), np.concatenate([prefix_v[0, h // G], values])
                if len(keys) == 0:
                    continue
                out[n, h, i], w, size[n, h, i], score[n, h, i] = attend(q[n, h, i], keys, values)
                if prefix_k is None:
                    weights[n, h // G, at] += w
    return out, weights, size, score


def evict(weights, lens, keep, recent):
    """-> kept (N, Hk, keep) int32, -1 past the last."""
    N, Hk, S = weights.shape
    kept = np.full((N, Hk, keep), -1, np.int32)
    for n in range(N):
        length = S if lens is None else min(max(int(lens[n]), 0), S)
        for h in range(Hk):
            chosen = list(range(length))
            if length > keep:
                old = length - recent
                rank = np.where(np.isnan(weights[n, h, :old]), -np.inf, weights[n, h, :old].astype(np.float64))
                first = sorted(range(old), key=lambda i: (not np.isnan(weights[n, h, i]), rank[i], -i), reverse=True)
                chosen = sorted(first[:keep - recent] + list(range(old, length)))
            kept[n, h, :len(chosen)] = chosen
    return kept
