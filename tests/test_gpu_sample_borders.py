"""GPU parity of ops.sample_tokens where a filter's border is hard to compare:
min_p at the ends of float32, and nuclei of nearly everything, whose border lies
among weights smaller than a sum's error. Every call states how many rows it
compares, or what holds of every row."""

import math

import numpy as np
import pytest
import torch

from oracle import sample_oracle as S
from test_gpu_sample_tokens import DT, check, logits, off, uniform

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("B,V", [(5, 20000), (64, 20000), (3, 3000)])
@pytest.mark.parametrize("scale,T", [(3.4e38, 1e38), (3.4e38, 1e36), (1.0, 0.1), (1e-38, 3e-39), (1e-41, 1e-41), (1e-30, 1e-30)])
def test_min_p_at_the_ends_of_float32(gpu, B, V, scale, T):
    x, u = logits(B, V, "fp32", 80, sigma=1.0), uniform(B, 81)
    y = ((x / x.abs().amax(1, keepdim=True)).double() * scale).float()
    for s in (dict(min_p=0.3), dict(min_p=0.9), dict(top_p=0.9, min_p=0.3), dict(top_k=300, min_p=0.5), dict(min_p=1e-30)):
        compared = check(y, u, sure=False, temperature=torch.tensor([T]).cuda(), **s)
        assert compared >= 0.9 * B, (s, compared)


def nearly(x, u, token, logprob, T, p):
    """A border of top_p that may fall to either side within the sums' error: the
    token is in the nucleus that the error allows, and its stretch meets u."""
    d = 4 * off(len(x))
    order = S.order_of(x)
    w = S.weights(x, x[order[0]], T)
    upto = np.cumsum(w[order])
    W, before = upto[-1], upto - w[order]
    may = order[:max(int((before < (p + d) * W).sum()), 1)]
    sure = np.zeros(len(x), bool)
    sure[order[:max(int((before < (p - d) * W).sum()), 1)]] = True
    assert token in may, token
    kept = w[sure].sum()
    loose = w[may].sum() - kept
    s = np.cumsum(np.where(sure, w, 0))[token]
    assert s + loose + d * W >= u * kept
    assert s - (w[token] if sure[token] else 0) - d * W <= u * (kept + loose)
    slack = 2.0 ** -24 * 1.001 * abs(logprob) + 2 * off(len(x))
    assert math.log(w[token] / (kept + loose)) - slack <= logprob <= math.log(w[token] / kept) + slack


@pytest.mark.parametrize("offset", [0.0, -300.0, 1000.0])
@pytest.mark.parametrize("dtype,V,B", [("fp32", 30011, 6), ("bf16", 30011, 6), ("fp16", 34001, 80), ("fp32", 20000, 64),
                                       ("bf16", 40000, 170)])
def test_nuclei_of_nearly_everything(gpu, dtype, V, B, offset):
    from delta_attention import ops
    for sigma in (0.05, 6.0):
        x = (logits(B, V, dtype, 50, sigma=sigma).float() + offset).to(DT[dtype])
        u = uniform(B, 51)
        X, U = x.double().cpu().numpy(), u.double().cpu().numpy()
        for k in (24, 20, 16):
            p = 1 - 2.0 ** -k
            t, lp = ops.sample_tokens(x, u, top_p=p)
            for b in range(B):
                nearly(X[b], U[b], int(t[b]), float(lp[b]), 1.0, p)
