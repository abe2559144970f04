"""ops.prefix_attention: what stands at places that a row does not see reaches it
in no way, whatever the row tiles and the keys' strides.

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


def same(a, b):
    return a.shape == b.shape and bool(((a == b) | (a.isnan() & b.isnan())).all())


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


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("D", [32, 64, 128, 256])
@pytest.mark.parametrize("Np,cap", [(1, 1), (1, 130), (130, 1), (1, 1300), (1300, 1)])
def test_infinities_of_a_single_key(gpu, Np, cap, D, dtype):
    """A key set of one place, whose value is infinite: its rows are."""
    from delta_attention import ops
    B, P, H, Hkv, s = 4, 2, 8, 2, 1
    ts = make(B, P, H, Hkv, s, D, Np, cap, dtype, Np + cap + D)
    want = ops.prefix_attention(*ts, sm_scale=0.1)
    close(want, expect(*ts, [Np] * P, [cap] * B, 0.1), dtype)
    for i in (2, 4):
        if ts[i].shape[2] > 1:
            continue
        v = ts[i].clone()
        v[..., 0], v[..., 5], v[..., 9] = math.inf, -math.inf, math.nan
        got = ops.prefix_attention(*ts[:i], v, *ts[i + 1:], sm_scale=0.1)
        assert (got[..., 0] == math.inf).all() and (got[..., 5] == -math.inf).all() and torch.isnan(got[..., 9]).all()
        rest = [c for c in range(D) if c not in (0, 5, 9)]
        assert torch.equal(got[..., rest], want[..., rest])


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("D", [32, 64, 128, 256])
@pytest.mark.parametrize("Np,cap,s", [(100, 30, 1), (30, 70, 3), (1001, 900, 1), (900, 1001, 5)])
def test_keys_that_share_their_places(gpu, Np, cap, s, D, dtype):
    """One key read as many (a stride of 0), and keys that overlap (a stride below
    head_dim): the same as of copies, infinite values among them."""
    from delta_attention import ops
    B, P, H, Hkv = 4, 2, 6, 2
    ts = make(B, P, H, Hkv, s, D, Np, cap, dtype, Np + s)
    g = torch.Generator().manual_seed(D)

    def overlapping(n, heads):
        base = torch.randn(heads, 8 * (n - 1) + D, generator=g).to(DT[dtype]).cuda()
        return base, base.as_strided((heads, n, D), (base.stride(0), 8, 1))

    def check(views, **kw):
        got = ops.prefix_attention(ts[0], *views, sm_scale=0.1, **kw)
        copies = [torch.empty(t.shape, device="cuda", dtype=t.dtype).copy_(t) for t in views]
        assert same(got, ops.prefix_attention(ts[0], *copies, sm_scale=0.1, **kw))
        return got

    for kw in (dict(), dict(n_prefix=i32([Np - 7, 1]), n_keys=i32([cap, s, 65 if cap > 65 else cap - 1, cap - 2]))):
        one = [t[:, :, :1].clone() for t in ts[1:]]
        for x in (math.inf, -math.inf):
            one[1][..., 3], one[3][..., 4] = x, x
            got = check([t.expand(-1, -1, n, -1) for t, n in zip(one, (Np, Np, cap, cap))], **kw)
            assert (got[..., 3:5] == x).all() and not torch.isnan(got).any()
        over = [overlapping(Np, P * Hkv), overlapping(Np, P * Hkv), overlapping(cap, B * Hkv), overlapping(cap, B * Hkv)]
        views = [v.view(-1, Hkv, *v.shape[1:]) for _, v in over]
        assert not torch.isnan(check(views, **kw)).any()
        # the first columns of the key past the last one, which are later columns of the last ones
        if not kw:
            for base, _ in (over[1], over[3]):
                base[:, -D + 8:-D + 12] = math.inf
            got = check(views)
            assert torch.isfinite(got[..., :8]).all() and (got[..., 8:12] == math.inf).all()
