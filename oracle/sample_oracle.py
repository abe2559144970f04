"""float64 oracle of the token choice (ops.sample_tokens), row by row, and how
near its decisions are to falling the other way."""

from __future__ import annotations

import math

import numpy as np


def order_of(x):
    """The candidates' indices, largest logit first, equal ones by index."""
    x = np.asarray(x, np.float64)
    at = np.flatnonzero(~np.isnan(x) & (x > -np.inf))
    return at[np.argsort(-x[at], kind="stable")]


def weights(x, top, T):
    with np.errstate(invalid="ignore"):
        d = np.where(x == top, 0.0, (x - top) / T)
    return np.exp(np.where(np.isnan(d), -np.inf, d))     # (an infinite top: the others weigh nothing)


def sample(x, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """-> (token, log-probability, margin): margin is the least distance, relative
    to a total, of a border of the sums from what it is compared with, or of a
    logit from min_p's bar, in temperatures and past what the bar's own float64
    may be off by (inf: no such comparison; logits equal to the largest need
    none, the bar is never above it)."""
    x = np.asarray(x, np.float64)
    order = order_of(x)
    if len(order) == 0:
        return 0, math.nan, math.inf
    top = x[order[0]]
    if not temperature > 0:
        return int(order[0]), 0.0, math.inf
    margin = math.inf
    if top_k > 0:
        order = order[:top_k]
    if top_p < 1:
        w = weights(x[order], top, temperature)
        upto = np.cumsum(w)
        before = upto - w
        goal = max(top_p, 0.0) * upto[-1]
        n = max(int((before < goal).sum()), 1)
        if n < len(order) or n > 1:
            margin = min(margin, float(np.abs(before[1:] - goal).min(initial=math.inf) / upto[-1]))
        order = order[:n]
    if min_p > 0:
        bar = top + temperature * math.log(min_p)
        rest = x[order[1:]]
        with np.errstate(invalid="ignore"):
            if math.isfinite(bar) and min_p != 1:     # (ln 1 = 0: the bar is the top, exactly)
                off = (abs(top) + temperature * abs(math.log(min_p))) * 2.0 ** -51
                far = np.abs(rest[rest != top] - bar).min(initial=math.inf)
                margin = min(margin, max(float(far - off), 0.0) / temperature)
            order = order[:1 + int((rest >= bar).sum())]
    order = np.sort(order)
    w = weights(x[order], top, temperature)
    upto = np.cumsum(w)
    total = upto[-1]
    u = 0.0 if math.isnan(u) else max(float(u), 0.0)
    if u < 1:
        margin = min(margin, float(np.abs(upto[:-1] - u * total).min(initial=math.inf) / total))
        # (a border that is as far below the number as the smallest weights are)
        at = min(int(np.searchsorted(upto, u * total, side="right")), len(order) - 1)
    else:
        at = int(np.flatnonzero(w > 0)[-1])
    return int(order[at]), math.log(w[at] / total) if w[at] > 0 else -math.inf, margin
