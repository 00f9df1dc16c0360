"""The paged-cache operators' definitions in 64 bits, as plain loops over
sequences (numpy), and how far fp32 kernels may be from them."""
from __future__ import annotations

import math

import numpy as np

U = 2.0 ** -24  # half a step of fp32
# half a step of a cache type, relative, and of its smallest values, absolute
STEP = {"f32": (2.0 ** -24, 2.0 ** -150), "f16": (2.0 ** -11, 2.0 ** -25),
        "bf16": (2.0 ** -8, 2.0 ** -134)}


def plan(lengths, n_new, table, stack, n_free, page, n_pages, max_rows):
    """(status, lengths, table, stack, n_free, row_start, positions, slots) after a step."""
    n, max_pages = table.shape
    same = (lengths.copy(), table.copy(), stack.copy(), n_free, np.zeros(n + 1, np.int32),
            np.full(max_rows, -1, np.int32), np.full(max_rows, -1, np.int64))
    held = [-(-int(x) // page) for x in lengths]
    freed = sum(h for h, a in zip(held, n_new) if a < 0 and h > 0)
    if any(a < -1 or l < 0 or int(l) + max(int(a), 0) > max_pages * page
           for a, l in zip(n_new, lengths)) or n_free < 0 or n_free + freed > n_pages:
        return (1, *same)
    if sum(max(int(a), 0) for a in n_new) > max_rows:
        return (2, *same)
    need = sum(-(-(int(l) + int(a)) // page) - h for l, a, h in zip(lengths, n_new, held) if a > 0)
    if need > n_free + freed:
        return (3, *same)
    lengths, table, stack, top, start, positions, slots = same
    for i in range(n):
        if n_new[i] < 0:
            for j in range(held[i]):
                stack[top] = table[i, j]
                top += 1
            lengths[i] = 0
    r = 0
    for i in range(n):
        start[i] = r
        for _ in range(max(int(n_new[i]), 0)):
            p = int(lengths[i])
            if p % page == 0:
                top -= 1
                table[i, p // page] = stack[top]
            positions[r] = p
            slots[r] = int(table[i, p // page]) * page + p % page
            lengths[i] += 1
            r += 1
    start[n] = r
    return 0, lengths, table, stack, top, start, positions, slots


def turn(x, w, eps, positions, freqs, magnitude, rot, neox):
    """(y, bound) of heads x [rows, heads, hd]."""
    x = np.asarray(x, np.float64)
    size = np.abs(x)
    if w is not None:
        w = np.asarray(w, np.float64)
        inv = 1.0 / np.sqrt((x * x).mean(-1, keepdims=True) + eps)
        x = x * w * inv
        # the squares' sum: a product, three adds in a lane, six over lanes, all of one sign (10 u,
        # halved by the root); eps, division, root, reciprocal (4 u); two products (2 u)
        size = np.abs(x) * 11 * U
    else:
        size = np.zeros_like(x)
    y, bound = x.copy(), size.copy()
    half = rot // 2
    i = np.arange(half)
    a, b = (i, i + half) if neox else (2 * i, 2 * i + 1)
    t = np.asarray(positions, np.float64)[:, None] * freqs
    c, s = (magnitude * f(t)[:, None] for f in (np.cos, np.sin))
    xa, xb = x[..., a], x[..., b]
    y[..., a], y[..., b] = xa * c - xb * s, xb * c + xa * s
    # cos and sin: the quarter turn's remainder (u / 2 of pi / 2), the function (4 u), the magnitude
    # (2 u with its own rounding); two products and a sum (3 u)
    m = abs(magnitude) * (10 * U * (np.abs(xa) + np.abs(xb)) + size[..., a] + size[..., b])
    bound[..., a] = m
    bound[..., b] = m
    return y, bound + 2.0 ** -140


def stored(y, bound, kind):
    """The bound of y rounded to a cache type."""
    rel, small = STEP[kind]
    return bound + (np.abs(y) + bound) * rel + small


def in_range(y, kind):
    """y as a cache type can hold it: fp16's last finite value is 65504, and
    65520, halfway to 65536, and all beyond round to infinity."""
    return np.where(np.abs(y) >= 65520, np.copysign(np.inf, y), y) if kind == "f16" else y


def gather(pool, table, length):
    """[kv, length, hd] of a sequence: pool [pages, kv, page, hd]."""
    page = pool.shape[2]
    ids = table[:-(-length // page)]
    return np.concatenate([pool[j] for j in ids], axis=1)[:, :length] if length else \
        np.zeros((pool.shape[1], 0, pool.shape[3]))


# fp16 matrix products: a sum is aligned by the exponent fields of its factors
# and keeps 24 bits from its largest term. A subnormal's field is that of 2^-14,
# the smallest normal number, so a product with one is off by up to 2^-24 2^-14
# of the other factor, whatever its own size; with two parts of that factor
# twice that. (The stored value itself is off by up to 2^-25.)
SUBNORMAL = 2.0 ** -37


def attention(q, k, v, pos, scale, softcap=0.0, window=0, slopes=None, kind=None):
    """(out, bound) [heads, hd] of one row q [heads, hd] at pos over k and v
    [kv, keys, hd] (keys 0 .. pos), for a cache of `kind`."""
    heads, hd = q.shape
    kv = k.shape[0]
    q = np.asarray(q, np.float64)
    out, bound = np.zeros((heads, hd)), np.zeros((heads, hd))
    first = max(0, pos + 1 - window) if window else 0
    n = pos + 1 - first
    if n <= 0:
        return out, bound
    for h in range(heads):
        kk = np.asarray(k[h * kv // heads, first:pos + 1], np.float64)
        vv = np.asarray(v[h * kv // heads, first:pos + 1], np.float64)
        s = kk @ q[h] * scale
        # hd products summed in any order, q in parts of 22 bits and more (4 u), scale (2 u)
        err = (hd + 8) * U * (np.abs(kk) @ np.abs(q[h])) * abs(scale)
        if kind == "f16":
            err = err + SUBNORMAL * np.abs(q[h]).sum() * abs(scale)
        if softcap:
            s = softcap * np.tanh(s / softcap)
            err = err + 6 * U * np.abs(s)  # division, tanh (3 u), product (derivative at most 1)
        if slopes is not None:
            bias = float(slopes[h]) * (np.arange(first, pos + 1) - pos)
            s = s + bias
            err = err + 2 * U * (np.abs(bias) + np.abs(s))
        top = s.max()
        p = np.exp(s - top)
        p /= p.sum()
        # the exponent's own roundings: difference, log2 e, exp2, once a tile for the running maximum's
        # steps (their arguments add up to the same difference)
        err = err + 4 * U * np.abs(s - top) + 8 * U
        mean = p @ err
        # the weights' sum and the output's: at most n roundings each; weights in parts of 22 bits
        out[h] = p @ vv
        bound[h] = (p * (err + mean + (2 * n + 24) * U)) @ np.abs(vv)
        # fp16 parts hold a weight down to 2^-39 of the largest
        bound[h] += n * 2.0 ** -39 * np.abs(vv).max() + 2.0 ** -140
        if kind == "f16":  # (the weights add up to 1)
            bound[h] += SUBNORMAL
    return out, bound


def rope_parts(theta, rot, factor, original, fast, slow):
    """Frequencies by parts, straight from their description."""
    def index(turns):
        return rot * math.log(original / (turns * 2 * math.pi)) / (2 * math.log(theta))
    low, high = max(math.floor(index(fast)), 0), min(math.ceil(index(slow)), rot - 1)
    f = np.array([theta ** (-2 * i / rot) for i in range(rot // 2)])
    ramp = np.clip((np.arange(rot // 2) - low) / max(high - low, 1e-3), 0, 1)
    return f / factor * ramp + f * (1 - ramp)
