"""Rows of a paged cache of 4 or 8 bits as include/mlq.h defines them (numpy;
d and m in the fp32 operations of the definition, codes in 64 bits)."""
from __future__ import annotations

import numpy as np

#: levels, middle, bytes of a unit of two elements
KINDS = {"q4": (15, 8, 1), "q8": (255, 128, 2)}


def blocks(hd):
    return 2 if hd <= 64 else 4 if hd <= 128 else 8


def row_bytes(hd, kind):
    return blocks(hd) * (16 * KINDS[kind][2] + 4)


def quantise(x, kind):
    """uint8 [..., row_bytes] of heads x [..., hd] (float32)."""
    levels, middle, unit = KINDS[kind]
    x = np.asarray(x, np.float32)
    hd, nb, lead = x.shape[-1], blocks(x.shape[-1]), x.shape[:-1]
    codes = np.full(lead + (nb, 32), middle, np.int64)
    scales = np.zeros(lead + (nb, 2), np.float16)
    with np.errstate(all="ignore"):
        for b in range(nb):
            e = x[..., 32 * b:32 * b + 32]
            if e.shape[-1] == 0:
                continue
            fine = np.isfinite(e).all(-1)
            lo, hi = e.min(-1), e.max(-1)
            d = ((hi - lo) / np.float32(levels)).astype(np.float16)
            m = (lo + np.float32(middle) * d.astype(np.float32)).astype(np.float16)
            fine &= np.isfinite(d) & np.isfinite(m)
            d, m = np.where(fine, d, np.float16(np.nan)), np.where(fine, m, np.float16(np.nan))
            d64, m64 = d.astype(np.float64)[..., None], m.astype(np.float64)[..., None]
            # (64 bits hold the borders, not the quotient of an element that is tiny next to m)
            e64 = e.astype(np.float64)
            c = np.floor((e64 - m64) / d64 + 0.5)
            c = c + (e64 >= (c + 0.5) * d64 + m64) - (e64 < (c - 0.5) * d64 + m64) + middle
            codes[..., b, :e.shape[-1]] = np.where(d64 > 0, np.clip(c, 0, levels), middle)
            scales[..., b, 0], scales[..., b, 1] = d, m
    pairs = np.moveaxis(codes.reshape(lead + (nb, 16, 2)), -3, -2)
    packed = (pairs[..., 0] | pairs[..., 1] << 4)[..., None] if unit == 1 else pairs
    return np.concatenate([packed.reshape(lead + (-1,)).astype(np.uint8),
                           scales.reshape(lead + (-1,)).view(np.uint8)], -1)


def values(rows, kind, hd):
    """float64 [..., hd], exact: d (c - middle) has at most 19 bits, and the
    exponents of fp16 leave the sum within 53."""
    levels, middle, unit = KINDS[kind]
    nb, lead = blocks(hd), rows.shape[:-1]
    codes, scales = rows[..., :16 * nb * unit], np.ascontiguousarray(rows[..., 16 * nb * unit:]).view(np.float16)
    pairs = np.stack([codes & 15, codes >> 4], -1) if unit == 1 else codes
    c = np.moveaxis(pairs.reshape(lead + (16, nb, 2)), -3, -2).reshape(lead + (nb, 32)).astype(np.float64) - middle
    s = scales.reshape(lead + (nb, 2)).astype(np.float64)
    return (s[..., :1] * c + s[..., 1:]).reshape(lead + (-1,))[..., :hd]


def same_rows(a, b, hd, kind):
    """Row bytes alike: NaN scales by being NaN, everything else by its bits."""
    at = 16 * blocks(hd) * KINDS[kind][2]
    x, y = (np.ascontiguousarray(r[..., at:]).view(np.float16) for r in (a, b))
    return np.array_equal(a[..., :at], b[..., :at]) and np.array_equal(np.isnan(x), np.isnan(y)) and \
        np.array_equal(x[~np.isnan(x)].view(np.uint16), y[~np.isnan(y)].view(np.uint16))


def heads(r, rows, kv, hd):
    """N(0, 1) heads with blocks in them that quantising has to be right for."""
    x = r.standard_normal((rows, kv, hd)).astype(np.float32)
    flat = x.reshape(-1, hd)
    special = [lambda e: 0.0, lambda e: -3.25, lambda e: e * 1e-6, lambda e: e * 1e-9, lambda e: e * 1e4,
               lambda e: e * 60000, lambda e: 1000 + e * 1e-3, lambda e: np.where(np.arange(e.size) == 5, np.nan, e),
               lambda e: np.where(np.arange(e.size) == 0, np.inf, e), lambda e: np.where(np.arange(e.size) == 7, -np.inf, e),
               lambda e: e * 1e38, lambda e: np.where(e > 0, 0.0, -0.0), lambda e: np.round(e * 4) / 8,
               # every element halfway between two codes, but for the ends
               lambda e: np.where(np.arange(e.size) == 0, -8.0, np.where(np.arange(e.size) == 1, 7.0, np.floor(e * 2) + 0.5)),
               lambda e: np.where(np.arange(e.size) < 2, np.arange(e.size) * 255 - 128.0, np.floor(e * 40) + 0.5),
               lambda e: np.full(e.size, 65519.0), lambda e: np.full(e.size, 65520.0), lambda e: np.abs(e) * 5e-8]
    for i, f in enumerate(special):
        if i < len(flat):
            b = 32 * int(r.integers((hd + 31) // 32))
            with np.errstate(all="ignore"):
                flat[i, b:b + 32] = f(flat[i, b:b + 32].copy())
    return x


# ---- attention over such rows ------------------------------------------------------
U = 2.0 ** -24  # half a step of fp32


def sizes(rows, kind, hd):
    """d |c - middle| + |m|: what an element's terms add up to without their signs."""
    levels, middle, unit = KINDS[kind]
    nb = blocks(hd)
    at = 16 * nb * unit
    s = np.abs(np.ascontiguousarray(rows[..., at:]).view(np.float16).astype(np.float64)).reshape(rows.shape[:-1] + (nb, 2))
    flat = rows.copy()
    flat[..., at:] = np.stack([s[..., 0], np.zeros_like(s[..., 1])], -1).astype(np.float16).reshape(rows.shape[:-1] + (-1,)).view(np.uint8)
    return np.abs(values(flat, kind, hd)) + np.repeat(s[..., 1], 32, -1)[..., :hd]


def steps(rows, kind, hd):
    """The largest d of each row; one that is not finite counts as 2^17, past the
    largest that is."""
    nb = blocks(hd)
    at = 16 * nb * KINDS[kind][2]
    d = np.ascontiguousarray(rows[..., at:]).view(np.float16).astype(np.float64).reshape(rows.shape[:-1] + (nb, 2))[..., 0]
    return np.where(np.isfinite(d), d, 2.0 ** 17).max(-1)


def attention(q, k, v, pos, scale, softcap=0.0, window=0, slopes=None, kind="q4"):
    """(out, bound) [heads, hd] of one row q [heads, hd] at pos over the row
    bytes k and v [kv, keys, bytes] (keys 0 .. pos)."""
    heads, hd = q.shape
    kv = k.shape[0]
    q = np.asarray(q, np.float64)
    out, bound = np.zeros((heads, hd)), np.zeros((heads, hd))
    first = max(0, pos + 1 - window) if window else 0
    n = pos + 1 - first
    if n <= 0:
        return out, bound
    parts = {}
    for h in range(heads):
        g = h * kv // heads
        if g not in parts:
            kr, vr = k[g, first:pos + 1], v[g, first:pos + 1]
            parts[g] = values(kr, kind, hd), sizes(kr, kind, hd), values(vr, kind, hd), sizes(vr, kind, hd), steps(vr, kind, hd).max()
        kk, ks, vv, vs, step = parts[g]
        s = kk @ q[h] * scale
        # a block's 32 products and 32 elements of q summed in any order, or the head's products at once;
        # two roundings a block for d and m; q, and elements, in parts of 22 bits, the parts of a product
        # below 2^-24 left out, the value's own rounding, scale
        err = (max(hd, 64) + 2 * blocks(hd) + 20) * U * (ks @ np.abs(q[h])) * abs(scale)
        # (parts hold 2^-39 of the head's largest |q| and of the row's largest element)
        err = err + 2.0 ** -38 * (np.abs(q[h]).max() * ks.sum(-1) + np.abs(q[h]).sum() * ks.max(-1)) * abs(scale)
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
        # (the exponent's own roundings, as for the other types)
        err = err + 4 * U * np.abs(s - top) + 8 * U
        mean = p @ err
        out[h] = p @ vv
        # the weights' sum and the output's: at most n roundings each; d, m, and parts of 22 bits
        bound[h] = (p * (err + mean + (2 * n + 40) * U)) @ vs
        # parts hold a weight times d down to 2^-39 of the largest weight times the largest d (2^-14 at
        # least), each with a code of up to `middle`; an element down to 2^-39 of its row's largest
        bound[h] += n * 2.0 ** -38 * (KINDS[kind][1] * max(step, 2.0 ** -14) + np.nanmax(vs, initial=0.0)) + 2.0 ** -140
    return out, bound
