"""Paged-cache operators in plain 64-bit numpy: what the GPU kernels are compared with."""
import math

import numpy as np

NONE = 0xFFFFFFFF
EPS = {"F32": 2.0 ** -23, "F16": 2.0 ** -10, "BF16": 2.0 ** -7}


def plan(page, pages, max_tokens, lens, new, release, table, stack, count):
    """(status bits, outputs by name) of a plan, one token at a time."""
    lens, new, table, stack = [int(x) for x in lens], [int(x) for x in new], table.copy(), stack.copy()
    n, width = len(lens), table.shape[1]
    keep = dict(table=table.copy(), stack=stack.copy(), count=count, lens=list(lens),
                start=[0] * (n + 1), positions=[0] * max_tokens, slots=[NONE] * max_tokens,
                owner=[NONE] * max_tokens, status=[0, 0, 0, 0])
    bits, returned = 0, []
    if any(x > width * page for x in lens):
        bits |= 8
    for r in range(n):
        if release is not None and release[r]:
            if lens[r] <= width * page:
                returned += [int(e) for e in table[r, :-(-lens[r] // page)] if e < pages]
            lens[r] = 0
    if count > pages or count + len(returned) > pages:
        bits |= 8
    if any(x > max_tokens for x in new) or sum(new) > max_tokens:
        bits |= 4
    grow = [a + b if a <= width * page else 0 for a, b in zip(lens, new) if b <= max_tokens]
    if any(x > width * page for x in grow):
        bits |= 2
    need = sum(-(-(a + b) // page) - -(-a // page) for a, b in zip(lens, new))
    if not bits and need > count + len(returned):
        bits |= 1
    if bits:
        keep["status"][0] = bits
        return bits, keep
    for e in returned:
        stack[count] = e
        count += 1
    start, positions, slots, owner = [0], [], [], []
    for r in range(n):
        for p in range(lens[r], lens[r] + new[r]):
            if p % page == 0:
                count -= 1
                table[r, p // page] = stack[count]
            e = int(table[r, p // page])
            positions.append(p)
            slots.append(e * page + p % page if e < pages else NONE)
            owner.append(r)
        start.append(len(positions))
    pad = max_tokens - len(positions)
    return 0, dict(table=table, stack=stack, count=count, lens=[a + b for a, b in zip(lens, new)],
                   start=start, positions=positions + [0] * pad, slots=slots + [NONE] * pad,
                   owner=owner + [NONE] * pad, status=[0, len(positions), need, len(returned)])


def heads(x, weight, eps, positions, axis, theta, rotary):
    """Rows x [tokens, heads, dim] normed (weight None: not) and rotated."""
    x = np.asarray(x, np.float64)
    if weight is not None:
        x = x / np.sqrt(np.mean(x * x, -1, keepdims=True) + eps) * np.asarray(weight, np.float64)
    out, half = x.copy(), rotary // 2
    for i in range(half):
        angle = positions[axis[i]].astype(np.float64) * theta ** (-2.0 * i / rotary)
        c, s = np.cos(angle)[:, None], np.sin(angle)[:, None]
        out[..., i] = x[..., i] * c - x[..., i + half] * s
        out[..., i + half] = x[..., i + half] * c + x[..., i] * s
    return out


def attention(q, k, v, table, start, lens, page, scale, window, sinks):
    """Rows q [tokens, heads, dim] over k, v [pages, page, kv_heads, dim] (all float64):
    (out, bound): bound[t, h] = (scale * max sum |q k|, max |v|, keys seen), for tolerances.
    Rows of no request are NaN."""
    tokens, h, dim = q.shape
    pages, kvh = k.shape[0], k.shape[2]
    out, bound = np.full(q.shape, np.nan), np.zeros((tokens, h, 3))
    for r in range(len(lens)):
        n, new = int(lens[r]), int(start[r + 1]) - int(start[r])
        for j in range(new):
            t, p = int(start[r]) + j, n - new + j
            i = np.arange(min(p + 1, table.shape[1] * page))
            seen = (i + window > p) | (i < sinks) if window else np.ones(len(i), bool)
            i = i[seen & (table[r, i // page] < pages)]
            at = table[r, i // page].astype(np.int64), i % page
            for a in range(h):
                out[t, a] = 0.0
                if not len(i):
                    continue
                kk, vv = k[at[0], at[1], a // (h // kvh)], v[at[0], at[1], a // (h // kvh)]
                s = scale * (kk @ q[t, a])
                w = np.exp(s - s.max())
                out[t, a] = (w / w.sum()) @ vv
                bound[t, a] = scale * np.abs(kk * q[t, a]).sum(-1).max(), np.abs(vv).max(), len(i)
    return out, bound


def attention_tolerance(out, bound, dim, gtype, cache):
    """Per element.  Scores: a dot of dim products in FP32 loses at most (dim + 8) half steps
    of FP32 of the sum of its terms' sizes (8: the parts of q, the scale, the subtraction of
    the maximum); an error e of every score moves a weighted mean by at most 2 e max|v|, and
    the exponential's own error (4 half steps) as much again.  Sums of n weights and values
    lose n + 64 half steps (64: rescaling between tiles and joining of parts).  16-bit types
    round the weights once and the output once, half a step each; F32 over BF16 keeps three
    parts of the weights, F32 over F16 two with 2^-24 of the largest lost."""
    half = EPS["F32"] / 2
    score, vmax, n = bound[..., 0:1], bound[..., 1:2], bound[..., 2:3]
    tol = vmax * (2 * (score * (dim + 8) + 4) + n + 64) * half
    if gtype != "F32":
        tol = tol + vmax * EPS[cache] / 2 + np.abs(out) * EPS[gtype] / 2
    return tol + 1e-30 if gtype != "F16" else tol + 2.0 ** -25  # F16: subnormal outputs


def ragged(rng, requests, longest, new_most):
    lens = [max(1, int(math.exp(rng.uniform(0, math.log(longest + 1))))) for _ in range(requests)]
    lens = [min(longest, n) for n in lens]
    new = [min(n, int(rng.integers(0, new_most + 1))) for n in lens]
    return lens, new
