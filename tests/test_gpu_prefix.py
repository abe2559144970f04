"""GPU parity of ops.prefix_attention with a float64 computation of the same
rows.

Tolerance, relative to the probability-weighted mean of |v|: a probability is
rounded to the inputs' type (half a step u) and its exponent is off by what D
fp32 products and sums, the scale and the reference leave (2^-24 each of the
score's magnitude), as much again for exp2 and the sums; both count twice, in
the row and in its weight. fp16 probabilities end 2^-32 below a row's largest,
which every key may lose. Then the result's rounding."""

import math

import numpy as np
import pytest
import torch

from helpers import np64

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "fp16": torch.float16}


def make(B, P, H, Hkv, s, D, Np, cap, dtype, seed, std=1.0):
    """q [B,H,s,D] and the four key / value tensors as views of the projections' layout."""
    g = torch.Generator().manual_seed(seed)

    def t(b, n, h):
        return (torch.randn(b, n, h, D, generator=g) * std).to(DT[dtype]).cuda().transpose(1, 2)

    return t(B, s, H), t(P, Np, Hkv), t(P, Np, Hkv), t(B, cap, Hkv), t(B, cap, Hkv)


def expect(q, kp, vp, k, v, n_prefix, n_keys, scale):
    """float64 rows -> (out, mean |v|, largest score magnitude, keys)."""
    q, kp, vp, k, v = (np64(t) for t in (q, kp, vp, k, v))
    B, H, s, D = q.shape
    P, Hkv = kp.shape[:2]
    out, mean_v, mags = np.zeros_like(q), np.zeros((B, H, s, 1)), np.zeros((B, H, s, 1))
    for b in range(B):
        p, n = b // (B // P), n_keys[b]
        for h in range(H):
            hk = h // (H // Hkv)
            for i in range(s):
                m = max(min(n - s + i + 1, n), 0)
                kk = np.concatenate([kp[p, hk, :n_prefix[p]], k[b, hk, :m]])
                vv = np.concatenate([vp[p, hk, :n_prefix[p]], v[b, hk, :m]])
                if not len(kk):
                    continue
                x = kk @ q[b, h, i] * scale
                w = np.exp(x - x.max())
                w /= w.sum()
                out[b, h, i] = w @ vv
                mean_v[b, h, i] = (w @ np.abs(vv)).max()
                mags[b, h, i] = (np.abs(kk) @ np.abs(q[b, h, i])).max() * abs(scale)
    return out, mean_v, mags, max(n_prefix, default=0) + max(n_keys, default=0)


def close(got, want, dtype):
    out, mean_v, mags, n = want
    D = out.shape[-1]
    t = torch.finfo(DT[dtype])
    u = t.eps / 2
    eps = 2 * (u + (D + 8) * 2.0 ** -24 * (mags + 1) + (n / 16 + 64) * 2.0 ** -24)
    tol = eps * mean_v + n * 2.0 ** -32 * mean_v.max(initial=0.0) + u * np.abs(out) * (1 + eps)
    tol = tol * 1.0001 + t.smallest_normal * 2 * u
    err = np.abs(np64(got) - out)
    assert (err <= tol).all(), (float((err / tol).max()), np.argwhere(~(err <= tol))[:4])


def run(case, dtype, n_prefix=None, n_keys=None, seed=0, scale=None, device=False):
    from delta_attention import ops
    B, P, H, Hkv, s, D, Np, cap = case
    ts = make(*case, dtype, seed)
    scale = D ** -0.5 if scale is None else scale
    nps = [Np] * P if n_prefix is None else n_prefix
    nks = [cap] * B if n_keys is None else n_keys
    kw = {}
    if n_prefix is not None:
        kw["n_prefix"] = torch.tensor(nps, dtype=torch.int32, device="cuda")
    if n_keys is not None:
        kw["n_keys"] = torch.tensor(nks, dtype=torch.int32, device="cuda")
    got = ops.prefix_attention(*ts, sm_scale=scale, **kw)
    assert got.shape == ts[0].shape and got.dtype == DT[dtype] and got.stride() == ts[0].stride()
    clamp = [min(max(x, 0), Np) for x in nps], [min(max(x, 0), cap) for x in nks]
    close(got, expect(*ts, *clamp, scale), dtype)
    return got, ts


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("case", [
    # B, P, H, Hkv, s, D, Np, cap
    (1, 1, 1, 1, 1, 32, 1, 1), (2, 1, 2, 1, 1, 64, 63, 2), (3, 3, 4, 2, 1, 128, 64, 65),
    (4, 2, 10, 2, 1, 128, 65, 64), (5, 1, 8, 8, 1, 256, 129, 30), (16, 1, 8, 2, 1, 128, 1000, 100),
    (33, 1, 16, 2, 1, 64, 777, 5), (8, 2, 24, 4, 1, 32, 515, 300), (40, 2, 8, 1, 1, 128, 300, 7),
    (2, 1, 4, 2, 3, 128, 200, 3), (4, 2, 6, 2, 17, 64, 333, 130), (1, 1, 8, 2, 70, 128, 100, 200),
    (3, 1, 4, 4, 5, 256, 90, 64), (6, 1, 5, 1, 40, 32, 150, 41),
], ids=str)
def test_rows(gpu, case, dtype):
    run(case, dtype, seed=sum(case))


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_counts_on_the_device(gpu, dtype):
    """Prefixes and own keys of every length up to the capacity and outside it:
    none, one, fewer than the rows, a tile's borders."""
    run((8, 4, 4, 2, 1, 128, 200, 140), dtype, [200, 0, 1, 64], [140, 0, 0, 1, 64, 65, 63, 128], 1)
    run((6, 2, 4, 2, 5, 64, 130, 70), dtype, [0, 129], [0, 1, 4, 5, 70, 66], 2)
    run((4, 2, 2, 2, 3, 32, 90, 50), dtype, [-7, 500], [-1, 3, 99, 50], 3)
    got, _ = run((4, 2, 2, 2, 3, 256, 90, 50), dtype, [0, 0], [0, 1, 2, 3], 4)
    assert not got[0].any() and not got[1, :, :2].any() and not got[2, :, :1].any()


def test_one_count_for_all(gpu):
    from delta_attention import ops
    ts = make(4, 2, 4, 2, 1, 128, 100, 50, "bf16", 5)
    one = ops.prefix_attention(*ts, n_prefix=torch.tensor([70], dtype=torch.int32, device="cuda"),
                               n_keys=torch.tensor([33], dtype=torch.int32, device="cuda"), sm_scale=0.1)
    host = ops.prefix_attention(*ts, n_prefix=70, n_keys=33, sm_scale=0.1)
    each = ops.prefix_attention(*ts, n_prefix=torch.tensor([70] * 2, dtype=torch.int32, device="cuda"),
                                n_keys=torch.tensor([33] * 4, dtype=torch.int32, device="cuda"), sm_scale=0.1)
    assert torch.equal(one, host) and torch.equal(one, each)
    close(one, expect(*ts, [70] * 2, [33] * 4, 0.1), "bf16")


@pytest.mark.parametrize("case", [(3, 1, 4, 2, 2, 64, 0, 30), (3, 1, 4, 2, 2, 64, 30, 0), (2, 2, 4, 2, 1, 128, 0, 0),
                                  (0, 1, 4, 2, 1, 64, 10, 10), (2, 1, 4, 2, 0, 64, 10, 10)], ids=str)
def test_nothing_on_one_side(gpu, case):
    run(case, "bf16")


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("D", [32, 64, 128, 256])
def test_hidden_places_may_hold_anything(gpu, D, dtype):
    """NaN and infinities behind the counts, and among a sequence's later keys
    and values, leave the rows that do not see them as they were."""
    from delta_attention import ops
    B, P, H, Hkv, s, Np, cap = 4, 2, 4, 2, 6, 150, 100
    ts = make(B, P, H, Hkv, s, D, Np, cap, dtype, 6)
    nps, nks = [130, 64], [90, 67, 6, 64]
    kw = dict(n_prefix=torch.tensor(nps, dtype=torch.int32, device="cuda"),
              n_keys=torch.tensor(nks, dtype=torch.int32, device="cuda"), sm_scale=D ** -0.5)
    want = ops.prefix_attention(*ts, **kw)
    close(want, expect(*ts, nps, nks, D ** -0.5), dtype)
    q, kp, vp, k, v = (t.clone() for t in ts)
    for p in range(P):
        kp[p, :, nps[p]:] = math.nan
        vp[p, :, nps[p]:] = math.inf
    for b in range(B):
        k[b, :, nks[b]:] = math.inf
        v[b, :, nks[b]:] = math.nan
        # the own places of rows 4 and 5
        k[b, :, nks[b] - 2] = math.nan
        v[b, :, nks[b] - 2, ::3] = -math.inf
        v[b, :, nks[b] - 1] = math.nan
    got = ops.prefix_attention(q, kp, vp, k, v, **kw)
    assert torch.equal(got[:, :, :4], want[:, :, :4])
    assert torch.isnan(got[:, :, 4:]).all()
    # values alone: those who see an infinity have it, with its sign
    v = ts[4].clone()
    for b in range(B):
        v[b, :, nks[b] - 2, 0] = math.inf
        v[b, :, nks[b] - 2, 1] = -math.inf
        v[b, :, nks[b] - 1, 0] = -math.inf
        v[b, :, nks[b] - 1, 2] = math.nan
    got = ops.prefix_attention(*ts[:4], v, **kw)
    assert torch.equal(got[:, :, :4], want[:, :, :4])
    assert (got[:, :, 4, 0] == math.inf).all() and (got[:, :, 4, 1] == -math.inf).all()
    assert torch.isnan(got[:, :, 5, 0]).all() and (got[:, :, 5, 1] == -math.inf).all() and torch.isnan(got[:, :, 5, 2]).all()
    assert torch.equal(got[:, :, 4, 2:], want[:, :, 4, 2:]) and torch.equal(got[:, :, 5, 3:], want[:, :, 5, 3:])


def test_scales(gpu):
    for scale in (0.0, -0.3, 2.0):
        run((4, 2, 4, 2, 2, 64, 100, 40), "bf16", seed=7, scale=scale)


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_references_that_move_late(gpu, dtype):
    """Keys whose scores grow along the sets: the references move tile by tile;
    then a set whose largest score lies far below the other's."""
    from delta_attention import ops
    case = (4, 1, 4, 2, 2, 64, 700, 300)
    for rise in (1, -1):
        ts = make(*case, dtype, 8)
        grow = torch.linspace(0.1, 6, 700, device="cuda")
        kp = (ts[1].float() * (grow if rise > 0 else grow.flip(0))[:, None]).to(DT[dtype])
        k = (ts[3].float() * 0.05).to(DT[dtype])
        got = ops.prefix_attention(ts[0], kp, ts[2], k, ts[4], sm_scale=0.3)
        close(got, expect(ts[0], kp, ts[2], k, ts[4], [700], [300] * 4, 0.3), dtype)


def test_rows_without_a_softmax(gpu):
    """A row whose every score is -inf is NaN, one that sees no key zero."""
    from delta_attention import ops
    ts = make(2, 1, 2, 1, 1, 32, 5, 3, "bf16", 9)
    q = ts[0].abs()
    kp, k = torch.full_like(ts[1], -math.inf), torch.full_like(ts[3], -math.inf)
    n = torch.tensor([3, 0], dtype=torch.int32, device="cuda")
    assert torch.isnan(ops.prefix_attention(q, kp, ts[2], k, ts[4], n_keys=n, sm_scale=1.0)).all()
    got = ops.prefix_attention(q, kp, ts[2], k, ts[4], n_prefix=0, n_keys=n, sm_scale=1.0)
    assert torch.isnan(got[0]).all() and not got[1].any()


def test_layouts(gpu):
    from delta_attention import ops
    B, P, H, Hkv, s, D, Np, cap = case = (4, 2, 4, 2, 3, 64, 100, 40)
    ts = make(*case, "bf16", 10)
    want = ops.prefix_attention(*ts, sm_scale=0.2)
    close(want, expect(*ts, [Np] * P, [cap] * B, 0.2), "bf16")
    packed = [t.contiguous() for t in ts]
    assert torch.equal(ops.prefix_attention(*packed, sm_scale=0.2), want)
    # rows 8 bytes off, and elements apart: copied
    wide = [torch.zeros(*t.shape[:3], 2 * D + 4, device="cuda", dtype=t.dtype) for t in ts]
    for skip, step in ((4, 1), (0, 2)):
        views = [w[..., skip:skip + D * step:step] for w in wide]
        for to, t in zip(views, ts):
            to.copy_(t)
        assert torch.equal(ops.prefix_attention(*views, sm_scale=0.2), want)
    # one prefix and one set of own keys, read as several
    ep = [t[:1].expand(P, -1, -1, -1) for t in ts[1:3]]
    ek = [t[:1].expand(B, -1, -1, -1) for t in ts[3:]]
    got = ops.prefix_attention(ts[0], *ep, *ek, sm_scale=0.2)
    assert torch.equal(got, ops.prefix_attention(ts[0], *(t.contiguous() for t in (*ep, *ek)), sm_scale=0.2))
    # a given result, inside a larger tensor that keeps the rest
    room = torch.full((B, s, H + 1, D), 7.0, device="cuda", dtype=torch.bfloat16)
    out = room[:, :, :H].transpose(1, 2)
    assert ops.prefix_attention(*ts, sm_scale=0.2, out=out) is out
    assert torch.equal(out, want) and (room[:, :, H] == 7).all()


def test_far_offsets(gpu):
    """A prefix of more than 4 GiB a tensor: the keys that count lie past it."""
    from delta_attention import ops
    Hkv, D, Np = 8, 256, 1150007
    kp = torch.zeros(1, Np, Hkv, D, device="cuda", dtype=torch.bfloat16)
    vp = torch.zeros_like(kp)
    kp[0, Np - 3] = 1.0
    vp[0, Np - 3] = torch.arange(Hkv, device="cuda")[:, None].to(torch.bfloat16) + 1
    q = torch.ones(2, Hkv, 1, D, device="cuda", dtype=torch.bfloat16)
    k = torch.zeros(2, Hkv, 3, D, device="cuda", dtype=torch.bfloat16)
    out = ops.prefix_attention(q, kp.transpose(1, 2), vp.transpose(1, 2), k, k, sm_scale=1.0)
    assert torch.equal(out, (torch.arange(Hkv, device="cuda") + 1).to(torch.bfloat16)[None, :, None, None].expand_as(out))


def test_repeats_itself_and_leaves_its_inputs(gpu):
    from delta_attention import ops
    ts = make(16, 1, 8, 2, 1, 128, 5000, 200, "bf16", 11)
    kept = [t.clone() for t in ts]
    a = ops.prefix_attention(*ts, sm_scale=0.1)
    assert all(torch.equal(ops.prefix_attention(*ts, sm_scale=0.1), a) for _ in range(5))
    assert all(torch.equal(x, y) for x, y in zip(ts, kept))


def test_recorded_and_on_other_streams(gpu):
    """One recorded call serves every length; two recorded calls of different
    sizes replayed in turn, between eager ones."""
    from delta_attention import ops
    sets = [make(8, 2, 8, 2, 1, 128, 900, 200, "bf16", 12), make(6, 1, 4, 2, 4, 64, 300, 64, "fp16", 13)]
    counts = [(torch.tensor([900, 100], dtype=torch.int32, device="cuda"), torch.full((8,), 200, dtype=torch.int32, device="cuda")),
              (torch.tensor([300], dtype=torch.int32, device="cuda"), torch.full((6,), 64, dtype=torch.int32, device="cuda"))]

    def call(i):
        return ops.prefix_attention(*sets[i], n_prefix=counts[i][0], n_keys=counts[i][1], sm_scale=0.1)

    call(0), call(1)
    torch.cuda.synchronize()
    graphs = []
    for i in (0, 1):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = call(i)
        graphs.append((g, out))
    side = torch.cuda.Stream()
    for r in range(5):
        for i in (0, 1):
            counts[i][0].copy_(torch.randint(0, sets[i][1].shape[2] + 1, counts[i][0].shape,
                                             generator=torch.Generator().manual_seed(r)).int())
            counts[i][1].copy_(torch.randint(0, sets[i][3].shape[2] + 1, counts[i][1].shape,
                                             generator=torch.Generator().manual_seed(9 + r)).int())
            sets[i][0].mul_(-1)
        want = [call(i).clone() for i in (0, 1)]
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            there = [call(i) for i in (0, 1)]
        torch.cuda.synchronize()
        for g, _ in graphs:
            g.replay()
        torch.cuda.synchronize()
        for i in (0, 1):
            assert torch.equal(graphs[i][1], want[i]) and torch.equal(there[i], want[i]), (r, i)
            close(want[i], expect(*sets[i], counts[i][0].tolist(), counts[i][1].tolist(), 0.1), ("bf16", "fp16")[i])


def test_agrees_with_a_cache_that_holds_both(gpu):
    """The rows of ops.decode_attention over each sequence's prefix and own keys
    in one cache, to the two kernels' roundings."""
    from delta_attention import ops
    B, P, H, Hkv, s, D, Np, cap = 6, 2, 8, 2, 1, 128, 700, 90
    ts = make(B, P, H, Hkv, s, D, Np, cap, "bf16", 14)
    got = ops.prefix_attention(*ts, sm_scale=D ** -0.5)
    kk, vv = (torch.cat([ts[i].repeat_interleave(B // P, 0), ts[i + 2]], 2) for i in (1, 2))
    ref = ops.decode_attention(ts[0], kk, vv, window=0, sink=0, sm_scale=D ** -0.5)
    assert (got.float() - ref.float()).abs().max().item() <= 6 * 2.0 ** -9 * vv.abs().max().item()


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("case", [
    # B, P, H, Hkv, s, D, Np, cap: keys that count, of larger capacities
    (1, 1, 1, 1, 1, 32, 1, 1), (2, 1, 2, 1, 1, 64, 63, 2), (3, 3, 4, 2, 1, 128, 64, 65),
    (4, 2, 10, 2, 1, 128, 65, 64), (5, 1, 8, 8, 1, 256, 129, 30), (40, 2, 8, 1, 1, 128, 300, 7),
    (2, 1, 4, 2, 3, 128, 200, 3), (4, 2, 6, 2, 17, 64, 333, 130), (1, 1, 8, 2, 70, 128, 100, 200),
    (3, 1, 4, 4, 5, 256, 90, 64), (6, 1, 5, 1, 40, 32, 150, 41), (24, 1, 8, 1, 2, 256, 70, 9),
], ids=str)
def test_short_keys_in_large_caches(gpu, case, dtype):
    """Few keys of many places: split, where caches of their size are not."""
    B, P, H, Hkv, s, D, Np, cap = case
    run((B, P, H, Hkv, s, D, Np + 1300, cap + 900), dtype, [Np] * P, [cap] * B, seed=sum(case))
    run((B, P, H, Hkv, s, D, Np + 1300, cap), dtype, [Np] * P, [cap] * B, seed=sum(case) + 1)
    run((B, P, H, Hkv, s, D, Np, cap + 1300), dtype, [Np] * P, [cap] * B, seed=sum(case) + 2)


def test_counts_in_large_caches(gpu):
    for dtype in DT:
        run((8, 4, 4, 2, 1, 128, 1200, 840), dtype, [1200, 0, 1, 64], [840, 0, 0, 1, 64, 65, 63, 128], 21)
        run((6, 2, 4, 2, 5, 64, 1130, 70), dtype, [0, 129], [0, 1, 4, 5, 70, 66], 22)
        run((4, 2, 2, 2, 3, 32, 990, 50), dtype, [-7, 1500], [-1, 3, 99, 50], 23)
        got, _ = run((4, 2, 2, 2, 3, 256, 990, 50), dtype, [0, 0], [0, 1, 2, 3], 24)
        assert not got[0].any() and not got[1, :, :2].any() and not got[2, :, :1].any()


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("D,s,H", [(32, 6, 4), (64, 6, 4), (128, 6, 4), (256, 6, 4), (64, 40, 8)])
def test_hidden_places_of_large_caches(gpu, D, s, H, dtype):
    from delta_attention import ops
    B, P, Hkv, Np, cap = 4, 2, 2, 1150, 700
    ts = make(B, P, H, Hkv, s, D, Np, cap, dtype, 26)
    nps, nks = [130, 64], [490, 67, s, 64]
    kw = dict(n_prefix=torch.tensor(nps, dtype=torch.int32, device="cuda"),
              n_keys=torch.tensor(nks, dtype=torch.int32, device="cuda"), sm_scale=D ** -0.5)
    want = ops.prefix_attention(*ts, **kw)
    close(want, expect(*ts, nps, nks, D ** -0.5), dtype)
    q, kp, vp, k, v = (t.clone() for t in ts)
    for p in range(P):
        kp[p, :, nps[p]:] = math.nan
        vp[p, :, nps[p]:] = math.inf
    for b in range(B):
        k[b, :, nks[b]:] = math.inf
        v[b, :, nks[b]:] = math.nan
        v[b, :, nks[b] - 1, ::3] = -math.inf     # the last row's own place
        v[b, :, nks[b] - 1, 1] = math.nan
    got = ops.prefix_attention(q, kp, vp, k, v, **kw)
    assert torch.equal(got[:, :, :s - 1], want[:, :, :s - 1])
    assert (got[:, :, s - 1, ::3] == -math.inf).all() and torch.isnan(got[:, :, s - 1, 1]).all()
    assert torch.equal(got[:, :, s - 1, 2::3], want[:, :, s - 1, 2::3])


@pytest.mark.parametrize("D", [64, 128, 256])
def test_lengths_around_the_split(gpu, D):
    """Capacities from one tile past the longest that one launch takes, batches
    with few sums and with many, the references moving in either set."""
    from delta_attention import ops
    for B, H, s in ((2, 2, 1), (64, 16, 1), (4, 8, 9)):
        for tiles in (1, 2, 3, 4, 6, 7, 8, 12, 13, 14, 15):
            own = min(64 * (tiles // 2) + s, 64 * tiles)
            run((B, 2, H, 2, s, D, 64 * tiles - own + 1, own), "bf16", seed=tiles + B)
    ts = make(4, 2, 4, 2, 2, D, 120, 100, "fp16", 28)
    for i in (1, 3):
        kk = list(ts)
        kk[i] = (kk[i].float() * torch.linspace(0.1, 8, kk[i].shape[2], device="cuda")[:, None]).half()
        got = ops.prefix_attention(*kk, sm_scale=0.3)
        close(got, expect(*kk, [120] * 2, [100] * 4, 0.3), "fp16")
