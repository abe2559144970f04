"""Float64 numpy oracle of the 8-bit key/value cache: e4m3 codes with one
power-of-two scale per block of 64 tokens, head and tensor.

A cache is a dict of `k`, `v` [B, Hkv, cap, D] (the codes' values, tokens in
order, NaN where nothing was written) and `ke`, `ve` [B, Hkv, cap / 64] (the
scales' exponents)."""

from __future__ import annotations

import numpy as np

BLOCK = 64
E_MIN, E_MAX = -117, 120


def round_e4m3(x):
    """|x| <= 448 to the nearest e4m3 value, ties to even; NaN and infinities
    give NaN."""
    x = np.asarray(x, np.float64)
    fine = np.isfinite(x)
    y = np.where(fine, x, 0.0)
    assert np.abs(y).max(initial=0.0) <= 448.0
    _, e = np.frexp(y)                                   # |y| in [2^(e-1), 2^e)
    step = np.ldexp(1.0, np.maximum(e - 1, -6) - 3)
    return np.where(fine, np.rint(y / step) * step, np.nan)


def block_exponent(x):
    """The smallest e in [E_MIN, E_MAX] with |x| <= 448 * 2^e over the finite x."""
    a = np.abs(x[np.isfinite(x)]).max(initial=0.0)
    e = E_MIN
    while a > np.ldexp(448.0, e) and e < E_MAX:
        e += 1
    return e


def new_cache(B, Hkv, cap, D):
    assert cap % BLOCK == 0
    z = np.full((B, Hkv, cap, D), np.nan)
    e = np.full((B, Hkv, cap // BLOCK), E_MIN)
    return dict(k=z, v=z.copy(), ke=e, ve=e.copy())


def write(cache, k, v, pos, counts=None):
    """k/v [B, S, Hkv, D] behind row pos[b] of each sequence, counts[b] tokens
    of it; in place. A sequence whose rows do not fit is left as it is."""
    B, S, Hkv, _ = k.shape
    cap = cache["k"].shape[2]
    for b in range(B):
        p = int(pos[b])
        c = S if counts is None else min(max(int(counts[b]), 0), S)
        if p < 0 or p + c > cap:
            continue
        for blk in range(p // BLOCK, -(-(p + c) // BLOCK) if c else 0):
            r0, r1 = max(p, blk * BLOCK), min(p + c, (blk + 1) * BLOCK)
            for h in range(Hkv):
                for name, ename, x in (("k", "ke", k), ("v", "ve", v)):
                    new = x[b, r0 - p:r1 - p, h]
                    e = block_exponent(new)
                    if r0 > blk * BLOCK:
                        was = int(cache[ename][b, h, blk])
                        e = max(e, was)
                        old = cache[name][b, h, blk * BLOCK:r0]
                        cache[name][b, h, blk * BLOCK:r0] = round_e4m3(old * 2.0 ** (was - e))
                    cache[name][b, h, r0:r1] = round_e4m3(new / 2.0 ** e)
                    cache[ename][b, h, blk] = e


def values(cache, start=0, n=None):
    """Rows start .. of k and v as values."""
    cap = cache["k"].shape[2]
    n = cap - start if n is None else n
    at = np.arange(start, start + n)
    f = lambda c, e: c[:, :, at] * np.exp2(e[:, :, at // BLOCK].astype(np.float64))[..., None]
    return f(cache["k"], cache["ke"]), f(cache["v"], cache["ve"])


def rows(q, k, v, n_keys, window, sink, sm_scale):
    """q [B, H, s, D] at the end of each sequence of k/v [B, Hkv, cap, D] values
    -> (out [B, H, s, D], spread): spread holds, per output value, the weighted
    mean of |v| and, per row, the largest sum of |q k| sm_scale over its keys
    (what rounding errors are measured by)."""
    B, H, s, D = q.shape
    G = H // k.shape[1]
    out = np.zeros((B, H, s, D))
    mean_v = np.zeros_like(out)
    mags = np.zeros((B, H, s, 1))
    for b in range(B):
        n = min(max(int(n_keys[b]), 0), k.shape[2])
        for i in range(s):
            r = n - s + i
            if r < 0:
                continue
            j = np.arange(r + 1)
            if window > 0:
                j = j[(j < sink) | (j > r - window)]
            for h in range(H):
                kk, vv = k[b, h // G, j], v[b, h // G, j]
                x = kk @ q[b, h, i] * sm_scale
                w = np.exp(x - x.max())
                w /= w.sum()
                out[b, h, i] = w @ vv
                mean_v[b, h, i] = w @ np.abs(vv)
                mags[b, h, i] = (np.abs(kk) @ np.abs(q[b, h, i])).max() * abs(sm_scale)
    return out, dict(mean_v=mean_v, mags=mags)
