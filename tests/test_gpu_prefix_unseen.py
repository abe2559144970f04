"""ops.prefix_attention: what stands at places that a row does not see reaches it
in no way, whatever the row tiles.

The rows that see an infinite or NaN value have it in its column; every other
column, and every row that does not see it, has the bits of the same call
without it (a probability does not depend on a value)."""

import math

import pytest
import torch

from test_gpu_prefix import DT, close, expect, make

pytestmark = pytest.mark.gpu


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("Np,cap", [(70, 60), (70, 100), (1150, 700)], ids=["one_launch", "two_tiles", "split"])
@pytest.mark.parametrize("G,s,D", [(64, 2, 64), (71, 3, 128), (128, 2, 32), (128, 3, 256), (64, 4, 128)])
def test_row_tiles_of_one_row(gpu, G, s, D, Np, cap, dtype):
    """64 query heads a kv head and more: a row tile holds the heads of one row,
    and a tile of keys more than that row sees."""
    from delta_attention import ops
    B, P, Hkv = 4, 2, 1
    ts = make(B, P, G, Hkv, s, D, Np, cap, dtype, G + s)
    nps, nks = [Np, 33], [10, cap, s, cap - 3]
    kw = dict(n_prefix=i32(nps), n_keys=i32(nks), sm_scale=D ** -0.5)
    want = ops.prefix_attention(*ts, **kw)
    close(want, expect(*ts, nps, nks, D ** -0.5), dtype)
    # the last row's own place, and what lies behind the counts
    for key in (False, True):
        k, v = ts[3].clone(), ts[4].clone()
        for b in range(B):
            v[b, :, nks[b]:] = math.nan
            k[b, :, nks[b]:] = math.inf
            v[b, :, nks[b] - 1, 0] = math.inf
            v[b, :, nks[b] - 1, 1] = -math.inf
            v[b, :, nks[b] - 1, 2] = math.nan
            if key:
                k[b, :, nks[b] - 1] = math.nan
        got = ops.prefix_attention(*ts[:3], k, v, **kw)
        assert torch.equal(got[:, :, :s - 1], want[:, :, :s - 1])
        if key:
            assert torch.isnan(got[:, :, s - 1]).all()
            continue
        assert (got[:, :, s - 1, 0] == math.inf).all() and (got[:, :, s - 1, 1] == -math.inf).all()
        assert torch.isnan(got[:, :, s - 1, 2]).all()
        assert torch.equal(got[:, :, s - 1, 3:], want[:, :, s - 1, 3:])
    # every place but the first row's
    v = ts[4].clone()
    for b in range(B):
        v[b, :, nks[b] - s + 1:] = math.nan
    got = ops.prefix_attention(*ts[:4], v, **kw)
    assert torch.equal(got[:, :, 0], want[:, :, 0]) and torch.isnan(got[:, :, 1:]).all()
