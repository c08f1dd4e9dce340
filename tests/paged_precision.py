"""How far FP32 rows' attention may be off in the mean, and what fewer parts of q or of the
weights would give.

Errors are counted in half steps of FP32, u = 2^-24, and as root mean squares: a rounding to
the nearest is u / sqrt(3) of what it rounds, one that cuts off 2 u / sqrt(3), so u stands for
either.  A matrix instruction adds 16 products or more to a sum and rounds it once.  A
score, scale * q . k, whose partial sums are about ||q k|| (2-norm of the products) large and
which takes dim / 16 instructions for each of q's parts, loses sqrt(parts dim / 16) u ||q k||;
the scale, log2 e and the subtraction of the maximum 2 u |score| together; the exponential and
the weight's parts (22 bits or more, 4 u / sqrt(3)) 3 u.  An error e_i of score i moves output d
by w_i (v_id - o_d) e_i, and errors of different i add by squares.  The sums of n weighted values
and of n weights, and 64 rescalings and joined parts, lose sqrt(n / 16 + 64) u of the size of
what they sum, sqrt(sum w^2 v^2) and o.  One and a half times the root mean square of all
that bounds a call's: the half is for q and k whose products add up more evenly than at random.
"""
import numpy as np

U = 2.0 ** -24
MARGIN = 1.5
PARTS = {"F16": 2, "BF16": 3}  # of FP32 rows over a cache of that type


def row(q, k, v, scale, cache):
    """(o, E): a row's output and its expected error per column, all float64."""
    s = scale * (k @ q)
    w = np.exp(s - s.max())
    w /= w.sum()
    o = w @ v
    e = U * (np.sqrt(PARTS[cache] * len(q) / 16) * scale * np.linalg.norm(k * q, axis=1) + 2 * np.abs(s) + 3)
    moved = (w * e)[:, None] * (v - o)
    return o, np.sqrt((moved ** 2).sum(0) + U * U * (len(s) / 16 + 64) * (o ** 2 + (w ** 2) @ (v ** 2)))


def ratio(off, expected):
    """A call's error over what is allowed."""
    return np.sqrt(np.mean(np.square(off))) / (MARGIN * np.sqrt(np.mean(np.square(expected))))


def rounded(x, cache):
    """x rounded to F16 or BF16."""
    if cache == "F16":
        return x.astype(np.float16).astype(np.float32)
    bits = x.astype(np.float32).view(np.uint32)
    return ((bits + 0x7FFF + ((bits >> 16) & 1)) & 0xFFFF0000).astype(np.uint32).view(np.float32)


def parts(x, cache, n):
    """The sum of the first n parts of x, exact in float64."""
    rest, total = x.astype(np.float32), np.zeros(x.shape)
    for _ in range(n):
        h = rounded(rest, cache)
        total += h
        rest = rest - h
    return total


def simulated(q, k, v, scale, cache, q_parts, w_parts):
    """A row by FP32 sums over tiles of 64 keys, q and weights in so many parts."""
    f = np.float32
    up = f(2.0 ** (14 - np.floor(np.log2(np.abs(q).max())))) if cache == "F16" else f(1)
    qq = parts(q.astype(f) * up, cache, q_parts)
    s = np.zeros(len(k), f)
    for d in range(0, len(q), 16):
        s = (s + k[:, d:d + 16] @ qq[d:d + 16]).astype(f)
    c = f(scale) * f(1.4426950408889634) / up
    bias = f(12) if cache == "F16" else f(-15)
    m = f((s * c).max())
    w = np.exp2((s.astype(np.float64) * c - (m - bias)).astype(f)).astype(f)
    ww, o, l = parts(w, cache, w_parts), np.zeros(v.shape[1], f), f(0)
    for t in range(0, len(k), 64):
        for i in range(t, min(t + 64, len(k)), 16):
            o = (o + ww[i:i + 16] @ v[i:i + 16]).astype(f)
        l = f(l + w[t:t + 64].astype(np.float64).sum())
    return (o * (f(1) / l)).astype(f)
