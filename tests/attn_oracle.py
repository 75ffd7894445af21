"""The paged cache and its attention in numpy, 64 bits: the oracle of the cache
and attention tests, and their input maker. Written from the statement in
include/sera_attn.h, position by position.
"""
import numpy as np

F16, Q8 = 1, 264
F32T, F16T, BF16T = 0, 1, 30
# half a step of each row type, relative
HALF_STEP = {F32T: 2.0 ** -24, F16T: 2.0 ** -11, BF16T: 2.0 ** -8}


def head_bytes(kind, page, dim):
    return page * dim * 4 if kind == F16 else page * dim * 2 + 8 * page


def views(pool, kind, page, heads, dim):
    """(K, V, K scale, V scale) of a pool [pages, heads, head bytes] uint8, as writable views."""
    pages = pool.shape[0]
    t = np.float16 if kind == F16 else np.int8
    n = page * dim * np.dtype(t).itemsize
    k = pool[:, :, :n].view(t).reshape(pages, heads, page, dim)
    v = pool[:, :, n:2 * n].view(t).reshape(pages, heads, page // 16, dim, 16)
    assert np.shares_memory(k, pool) and np.shares_memory(v, pool)
    if kind == F16:
        return k, v, None, None
    return k, v, pool[:, :, 2 * n:2 * n + 4 * page].view(np.float32), pool[:, :, 2 * n + 4 * page:].view(np.float32)


def codes(x):
    """(int8 codes, float32 scale) of one vector."""
    x = np.asarray(x, np.float32)
    if not np.all(np.isfinite(x)):
        return np.zeros(x.shape, np.int8), np.float32(np.nan)
    d = np.float32(np.max(np.abs(x)) / np.float32(127)) if x.size else np.float32(0)
    if d == 0:
        return np.zeros(x.shape, np.int8), d
    return np.clip(np.rint(x.astype(np.float64) / np.float64(d)), -127, 127).astype(np.int8), d


def write(pool, kind, page, heads, dim, table, starts, lens, k, v):
    """The new rows of every sequence into the pool; k, v [rows, heads * dim] float32."""
    kk, vv, ks, vs = views(pool, kind, page, heads, dim)
    for b, length in enumerate(lens):
        n = starts[b + 1] - starts[b]
        for i in range(n):
            j = length - n + i
            if j < 0:
                continue
            p, o = table[b][j // page], j % page
            if not 0 <= p < pool.shape[0]:
                continue
            for h in range(heads):
                x, y = (a[starts[b] + i, h * dim:(h + 1) * dim] for a in (k, v))
                if kind == F16:
                    with np.errstate(over="ignore"):
                        kk[p, h, o], vv[p, h, o // 16, :, o % 16] = x.astype(np.float16), y.astype(np.float16)
                else:
                    kk[p, h, o], ks[p, h, o] = codes(x)
                    vv[p, h, o // 16, :, o % 16], vs[p, h, o] = codes(y)


def values(pool, kind, page, heads, dim, table, b, n):
    """(K, V) [heads, n, dim] float64 of positions 0..n-1 of sequence b; NaN on pages outside the pool."""
    kk, vv, ks, vs = views(pool, kind, page, heads, dim)
    K, V = np.full((heads, n, dim), np.nan), np.full((heads, n, dim), np.nan)
    for j0 in range(0, n, page):
        p, m = table[b][j0 // page], min(page, n - j0)
        if not 0 <= p < pool.shape[0]:
            continue
        x = kk[p].astype(np.float64)
        y = vv[p].astype(np.float64).transpose(0, 1, 3, 2).reshape(heads, page, dim)
        if kind == Q8:
            with np.errstate(invalid="ignore"):
                x, y = x * ks[p].astype(np.float64)[..., None], y * vs[p].astype(np.float64)[..., None]
        K[:, j0:j0 + m], V[:, j0:j0 + m] = x[:, :m], y[:, :m]
    return K, V


def attend(K, V, q, length, scale, window, sinks, kind_bits, flip=False):
    """(out, tolerance) [n, heads, dim] of one sequence's new rows q [n, heads, dim] (float64 of the given values).

    Tolerance. A score's terms are q k; the device holds q in 22 bits (or exactly, in 16-bit types), sums in fp32 and
    scales: at most (2^-22 + 140 2^-24) sum|q k| scale off, and its exponential another 2^-23 (|s - max| + 4). So
    a weight is off by d = 2^-19 (sum|q k| scale + 1) relative, the weighted mean by 2 d max|v|, plus the sums of the
    products themselves (2^-20 max|v|). 16-bit rows: the weights are rounded to fp16 (2^-11), and the result to
    its type (half a step)."""
    n, heads, dim = q.shape
    g = heads // K.shape[0]
    out, tol = np.zeros(q.shape), np.zeros(q.shape)
    for i in range(n):
        p = length - n + i
        if p < 0:
            continue
        j = np.arange(length)
        see = j <= p
        if window > 0:
            see &= (j > p - window) | (j < sinks)
        if flip:
            see[:] = True
        for h in range(heads):
            k, v = K[h // g][see], V[h // g][see]
            with np.errstate(all="ignore"):
                s = (k @ q[i, h]) * scale
                w = np.exp(s - s.max())
                o = (w @ v) / w.sum()
                a = (np.abs(k) @ np.abs(q[i, h])).max() * abs(scale)
                big = np.abs(v).max()
                t = big * (2 * 2.0 ** -19 * (a + 1) + 2.0 ** -20)
                if kind_bits != F32T:
                    t += big * 2.0 ** -11 + np.abs(o) * HALF_STEP[kind_bits]
                else:
                    t += np.abs(o) * HALF_STEP[F32T]
            out[i, h], tol[i, h] = o, t
    return out, tol
