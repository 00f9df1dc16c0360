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
            c = np.floor((e.astype(np.float64) - m64) / d64 + 0.5) + middle
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
