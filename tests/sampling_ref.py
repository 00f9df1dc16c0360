"""Sampling as include/mlq.h defines it, a row at a time in 64 bits (numpy)."""
from __future__ import annotations

import numpy as np

BIG = float(np.finfo(np.float32).max)


def token(x, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """(token, margin): how far, relative to the sum, the nearest border that
    the token hangs on lies from where u or top_p points."""
    x = np.asarray(x, np.float32).astype(np.float64)
    order = np.flatnonzero(~np.isnan(x) & (x != -np.inf))
    if not len(order):
        return -1, 1.0
    x = np.minimum(x[order], BIG)
    s = np.lexsort((order, -x))
    order, x = order[s], x[s]
    t, p, least, u = (float(np.float32(v)) for v in (temperature, top_p, min_p, u))
    if not t > 0:
        return int(order[0]), 1.0
    if top_k > 0:
        order, x = order[:top_k], x[:top_k]
    with np.errstate(all="ignore"):
        w = np.exp((x - x[0]) * (1.0 / t))
    margin = 1.0
    if p < 1:
        sums = np.cumsum(w)
        target = p * sums[-1]
        n = int((sums < target).sum())
        margin = min(margin, abs(sums[n] - target) / sums[-1], abs(sums[n] - w[n] - target) / sums[-1])
        if w[0] == w[n]:  # (equal weights of 1: nothing is rounded)
            margin = 1.0
        w = w[:n + 1]
    if least > 0:
        n = max(1, int((w >= least).sum()))
        if n > 1 or w[0] >= least:
            margin = min(margin, min((abs(v / least - 1) for v in w if v != 1.0), default=1.0))
        w = w[:n]
    sums = np.cumsum(w)
    target = min(max(u, 0.0) if u == u else 0.0, 1.0) * sums[-1]
    if target >= sums[-1]:
        # the last token that weighs anything (in units of 2^-44, half of one rounded up)
        return int(order[np.flatnonzero(w > 0.5 * 2.0 ** -44)[-1]]), margin
    n = int((sums <= target).sum())
    if w[0] != w[n]:
        margin = min(margin, abs(sums[n] - target) / sums[-1], abs(target - (sums[n] - w[n])) / sums[-1] if n else 1.0)
    return int(order[n]), margin
