"""Shared by the 8-bit cache's tests: between the cache's tensors and the
oracle's, and the tolerance of its attention rows."""

import numpy as np
import torch

from oracle import kv8_oracle as K8


def place():
    """place[i]: where token i of a block stands among its values."""
    at = {}
    for t in range(4):
        for g in range(4):
            for r in range(4):
                at[16 * t + 4 * g + r] = 16 * g + 4 * t + r
    return np.array([at[i] for i in range(64)])


def to_oracle(c):
    """An ops.KV8 as the oracle's dict (the codes' values, token order)."""
    B, Hkv, cap, D = c.k.shape
    k = c.k.float().cpu().numpy().astype(np.float64)
    v = c.v.float().cpu().numpy().astype(np.float64)
    v = v[..., place()].transpose(0, 1, 2, 4, 3).reshape(B, Hkv, cap, D)
    e = [np.log2(s.double().cpu().numpy()) for s in (c.k_scale, c.v_scale)]
    assert all((x == np.rint(x)).all() for x in e), "scales are powers of two"
    return dict(k=k, v=v, ke=e[0].astype(int), ve=e[1].astype(int))


def same(a, b):
    return np.array_equal(a, b, equal_nan=True)


def tolerance(ref, spread, D, n, dtype, add=None):
    """How far a row may be from the float64 one. Relative to the weighted mean
    of |v|: each probability is rounded to fp16 (2^-12) and its exponent is off
    by what D fp32 products and sums, the scale and the reference leave (2^-24
    each of the score's magnitude, and as much again for exp2's own and the
    sums' rounding); both count twice, in the row and in its weight. fp16 ends
    2^-32 below a row's largest weight, which every key may lose. Then the
    result's rounding, and the addend's sum's."""
    u = torch.finfo(dtype).eps / 2
    eps = 2 * (2.0 ** -12 + (D + 8) * 2.0 ** -24 * (spread["mags"] + 1) + (n / 16 + 64) * 2.0 ** -24)
    vmax = spread["mean_v"].max(initial=0.0) + np.abs(ref).max(initial=0.0)
    tol = eps * spread["mean_v"] + n * 2.0 ** -32 * vmax + u * np.abs(ref) * (1 + eps)
    if add is not None:
        tol = tol + u * (np.abs(ref + add) + tol)
    # below the type's normal range a step is fixed
    return tol * 1.0001 + float(torch.finfo(dtype).smallest_normal) * 2 * u
