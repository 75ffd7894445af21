"""Bounds of single precision steps of the rotation, the attention weights and the log probabilities, and the same steps
without what keeps them exact, in numpy: a bound that the lesser step kept as well would notice nothing.
"""
import numpy as np

F = np.float32


# ---- the angle of a rotation ---------------------------------------------------

def angle_cases(n=400, dim=128, seed=0):
    """(positions, frequencies, cosines, sines) in 64-bit mantissas."""
    rng = np.random.default_rng(seed)
    at = np.concatenate([rng.integers(0, 4096, n // 2), rng.integers(0, 1 << 22, n - n // 2)]).astype(np.int64)
    f = (10000.0 ** (-np.arange(dim // 2) / (dim // 2))).astype(F)
    a = at[:, None].astype(np.longdouble) * f.astype(np.longdouble)          # 22 + 24 bits: exact
    return at, f, np.cos(a), np.sin(a)


def angle_bound(value, at, f):
    """Sine and cosine of the rounded angle are good to two steps (2 * 2^-23), what its rounding leaves is added with one
    rounding (2^-24) and its own square forgotten ((2^-25 pi)^2 / 2 < 2^-47). The turns, a product with two more roundings
    of 2^-53 and the constant's, are off by 4 * 2^-53 of themselves, and the angle by 2 pi times that: 4 * 2^-53 of the angle."""
    return 2.5 * 2.0 ** -23 * np.abs(value) + 2.0 ** -47 + 4 * 2.0 ** -53 * np.abs(at[:, None] * f.astype(np.float64))


def angle_rounded(at, f):
    """Cosine and sine of the angle rounded to 32 bits in half turns, themselves exact and rounded once."""
    turns = at[:, None].astype(np.float64) * f.astype(np.float64) * 0.15915494309189535
    h = (2 * (turns - np.rint(turns))).astype(F).astype(np.float64)
    return np.cos(np.pi * h).astype(F), np.sin(np.pi * h).astype(F)


# ---- the weights of equal scores --------------------------------------------------

SCALES = [np.ldexp(1.0 + i / 41.0, 90) for i in range(40)]      # of an 8-bit cache's values: the maximum is near 90
SIZES = [500.0 + i for i in range(10)]                          # of q, over 128 channels of keys of 1


def equal_weights(new, length, group):
    """What every position gets from rows whose scores are all alike."""
    first = length - new
    return np.array([sum(group / (first + i + 1) for i in range(new) if first + i >= j) for j in range(length)])


def weights_bound(want):
    """Relative, up to 16 positions and 16 rows of a group of 8. A weight of the row's sum is an exponential (2^-23), the sum
    of up to 16 equal ones 16 roundings; the norm an exponential, a quotient or a logarithm (3 * 2^-23, and for many rows
    the norm's rounding, below 8: 2^-22); the weight itself an exponential, and 16 additions of those, each 2^-24:
    2 + 16 + 6 + 4 + 2 + 16 = 46 steps of 2^-24."""
    return 46 * 2.0 ** -24 * want


def weight_by_logarithm(score, length):
    """The weight of one of `length` scores, all alike (to the base 2), by the logarithm of the row's sum, which is of the
    scores' size, and rounded so."""
    m = F(score)
    shift = F(m - F(7))
    total = F(F(length) * F(np.exp2(np.float64(m) - np.float64(shift))))
    z = F(shift + F(np.log2(np.float64(total))))
    return np.exp2(np.float64(m) - np.float64(z))


# ---- the entropy beside a token that stands out ------------------------------------

def peaked(rows, vocab, height, seed=0):
    """Logits of one size and one of `height` in each row, and where it is."""
    rng = np.random.default_rng(seed)
    x = rng.standard_normal((rows, vocab)).astype(F)
    at = np.arange(rows) * 31 % vocab
    x[np.arange(rows), at] = height
    return x, at


def peaked_exact(x, at):
    """(entropy, log probability of the token that stands out), by what the others are: log1p and sums of small numbers."""
    d = x.astype(np.float64) - x[np.arange(len(x)), at].astype(np.float64)[:, None]
    e = np.exp(d)
    e[np.arange(len(x)), at] = 0
    rest = e.sum(1)
    return np.log1p(rest) - (e * d).sum(1) / (1 + rest), -np.log1p(rest)


def peaked_bound(x, at):
    """Relative error of both, where no other weight is in the 16 that the large one is added up with. d is the largest
    difference from the maximum. An exponential's argument is a rounded difference times a rounded log2(e), rounded: (2^-24 +
    2^-24 + 2^-26) d, and the exponential 2^-23. A lane's sum is raised to a new maximum at most some 5 times over its steps,
    9 times in the workgroup and 9 where a row is split: the differences are d together, each factor an exponential. 16
    weights are added in 32 bits, the rest in 64. The entropy has a quotient of two such sums, hence twice; the result
    is rounded once."""
    top = x[np.arange(len(x)), at].astype(np.float64)
    d = (top - x.min(1).astype(np.float64))
    one = 2 * d * (2.0 ** -23 + 2.0 ** -26) + 24 * 2.0 ** -23 + 16 * 2.0 ** -24
    return 2 * one + 2.0 ** -24


def peaked_among_16(x, at):
    """What the weights that are added up with the large one in 32 bits lose beside it, absolutely: 15 additions to a sum
    from 1 on round by half a step of it, 2^-24 each, and none by more than what is added, so that it is no more than the
    15 largest of the others either. The sum is off by that, its logarithm as much, and the entropy by (1 + its mean
    difference from the maximum) times that."""
    d = x.astype(np.float64) - x[np.arange(len(x)), at].astype(np.float64)[:, None]
    e = np.exp(d)
    e[np.arange(len(x)), at] = 0
    lost = np.minimum(15 * 2.0 ** -24, np.sort(e, 1)[:, -15:].sum(1))
    return lost * (1 + np.abs((e * d).sum(1))), lost


def peaked_in_32_bits(x, at):
    """Both with sums in 32 bits: 256 lanes, then their join two by two; all else exact."""
    d = (x - x[np.arange(len(x)), at][:, None]).astype(np.float64)
    w = np.exp(d).astype(F)
    t = (w.astype(np.float64) * d).astype(F)
    sums = []
    for y in (w, t):
        y = np.pad(y, ((0, 0), (0, -y.shape[1] % 256))).reshape(len(y), -1, 256)
        a = np.zeros((len(y), 256), F)
        for i in range(y.shape[1]):
            a = a + y[:, i]
        while a.shape[1] > 1:
            a = a[:, ::2] + a[:, 1::2]
        sums.append(a[:, 0].astype(np.float64))
    return (np.log(sums[0]) - sums[1] / sums[0]).astype(F), (-np.log(sums[0])).astype(F)
