"""Normed and rotated heads, attention weights, eviction and log probabilities in numpy, 64 bits: the oracle of their
tests, written from the statements in include/sera_attn.h and include/sera_logprobs.h.
"""
import numpy as np

HALVES, NEIGHBOURS = 0, 1


def heads_turned(x, gamma, eps, inv_freq, pairing, positions):
    """(values, tolerance without the final rounding) of heads x [rows, heads, dim] (float64).

    Tolerance. The mean of squares: at most 8 + 5 additions in fp32, halved by the root, and three more roundings: 10 steps
    of 2^-24; times x and gamma two more: 12. Sine and cosine: the angle is rounded once in half turns, 2^-25 pi, and
    the functions are good to two steps, together below 2^-22; the products and their sum two steps of 2^-24. In
    all (12 + 4 + 2) 2^-24 < 2^-19 of |a| + |b|. 64 bits leave position * inv_freq off by 2^-52 of it: 2^-24 at 2^28."""
    y = np.asarray(x, np.float64)
    if gamma is not None:
        with np.errstate(all="ignore"):
            y = y / np.sqrt((y * y).mean(-1, keepdims=True) + eps) * gamma.astype(np.float64)
    out, size = y.copy(), np.abs(y)
    if inv_freq is not None:
        half = len(inv_freq)
        angle = np.asarray(positions, np.float64)[:, None, None] * inv_freq.astype(np.float64)
        c, s = np.cos(angle), np.sin(angle)
        i, j = (slice(0, half), slice(half, 2 * half)) if pairing == HALVES else (slice(0, 2 * half, 2), slice(1, 2 * half, 2))
        out[..., i], out[..., j] = y[..., i] * c - y[..., j] * s, y[..., i] * s + y[..., j] * c
        both = np.abs(y[..., i]) + np.abs(y[..., j])
        size[..., i], size[..., j] = both, both
    return out, size * 2.0 ** -19


def weights_of(K, q, length, scale, window, sinks):
    """(sums, tolerance) [kv heads, length] of one sequence's new rows q [n, heads, dim], keys K [kv heads, length, dim].

    Tolerance. As for attention a weight is off by 2 * 2^-19 (sum|q k| scale + 1) of itself (its score, and the scores of
    the sum that it is divided by). Sums of m weights in fp32: m 2^-24 of them."""
    n, heads, _ = q.shape
    g = heads // K.shape[0]
    w, tol = np.zeros((K.shape[0], length)), np.zeros((K.shape[0], length))
    for i in range(n):
        p = length - n + i
        if p < 0:
            continue
        j = np.arange(length)
        see = j <= p
        if window > 0:
            see &= (j > p - window) | (j < sinks)
        for h in range(heads):
            k = K[h // g][see]
            with np.errstate(all="ignore"):
                s = (k @ q[i, h]) * scale
                e = np.exp(s - s.max())
                e /= e.sum()
                a = (np.abs(k) @ np.abs(q[i, h])).max() * abs(scale)
            w[h // g, see] += e
            tol[h // g, see] += e * (2 * 2.0 ** -19 * (a + 1))
    return w, tol + w * (n * g + 8) * 2.0 ** -24 + 1e-36


def kept_of(weights, length, keep, recent, sinks):
    """The positions that stay, of one sequence and kv head."""
    if length <= keep:
        return list(range(length))
    middle = range(sinks, length - recent)

    def rank(j):
        w = float(weights[j])
        return (1, 0.0, j) if w != w else (0, -w, j)

    best = sorted(middle, key=rank)[:keep - sinks - recent]
    return sorted(list(range(sinks)) + best + list(range(length - recent, length)))


def scores(x, tokens, top):
    """(log probabilities of tokens, entropy, top ids, their log probabilities) of one row x (float64)."""
    if np.isnan(x).any() or (x == np.inf).any() or not (x > -np.inf).any():
        return np.full(len(tokens), np.nan), np.nan, np.full(top, -1), np.full(top, np.nan)
    with np.errstate(all="ignore"):
        d = x - x.max()
        e = np.exp(d)
        log_z = np.log(e.sum())
        lp = d - log_z
        entropy = -np.sum(np.where(e > 0, e / e.sum() * np.where(e > 0, lp, 0), 0))
    given = np.array([lp[t] if 0 <= t < len(x) else np.nan for t in tokens])
    ids = np.lexsort((np.arange(len(x)), -x))[:top]
    return given, entropy, ids, lp[ids]
