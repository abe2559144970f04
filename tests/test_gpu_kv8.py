"""GPU parity of the 8-bit key/value cache (ops.kv8_write / kv8_read /
kv8_attention) with the float64 oracle: codes and scales bit for bit, read rows
bit for bit, attention rows within the bound of kv8_helpers.tolerance."""

import numpy as np
import pytest
import torch

from helpers import np64
from kv8_helpers import place, same, to_oracle, tolerance
from oracle import kv8_oracle as K8

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "fp16": torch.float16}


def tokens(B, S, Hkv, D, dtype, seed, spread=True):
    """Tokens whose magnitude varies over heads and rows (so do the scales)."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(B, S, Hkv, D, generator=g)
    if spread:
        x = x * torch.exp2(torch.randint(-6, 7, (B, S, Hkv, 1), generator=g).float())
    return x.to(dtype).cuda()


def garbage(c, seed):
    """Every byte and scale of a new cache set to noise, NaN codes among them."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    for t in (c.k, c.v):
        t.view(torch.uint8).random_(0, 256, generator=g)
    for t in (c.k_scale, c.v_scale):
        t.copy_(torch.exp2(torch.randint(-100, 100, t.shape, device="cuda", generator=g).float()))
    return c


def check_cache(c, ref, live):
    """Codes and scales of the first live[b] rows equal the oracle's."""
    got = to_oracle(c)
    for b, n in enumerate(live):
        nb = -(-n // 64)
        for x in ("k", "v"):
            assert same(got[x][b, :, :n], ref[x][b, :, :n]), (b, x)
        for x in ("ke", "ve"):
            assert np.array_equal(got[x][b, :, :nb], ref[x][b, :, :nb]), (b, x)


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("B,Hkv,D,cap,pos,S", [
    (1, 1, 128, 64, 0, 64),        # one whole block
    (1, 2, 128, 128, 0, 1),        # the first token
    (2, 3, 64, 256, 0, 130),       # whole blocks and a part
    (1, 2, 32, 320, 5, 200),       # from inside a block
    (2, 2, 256, 192, 63, 66),      # the last row of a block, one of the next but one
    (1, 8, 128, 1024, 127, 777),
])
def test_write_codes_and_scales(gpu, B, Hkv, D, cap, pos, S, dtype):
    from delta_attention import ops
    c = garbage(ops.kv8_empty(B, Hkv, cap, D), 1)
    ref = K8.new_cache(B, Hkv, cap, D)
    if pos:
        k0, v0 = (tokens(B, pos, Hkv, D, DT[dtype], s) for s in (2, 3))
        ops.kv8_write(c, k0, v0, 0)
        K8.write(ref, np64(k0), np64(v0), [0] * B)
    k, v = (tokens(B, S, Hkv, D, DT[dtype], s) for s in (4, 5))
    before = to_oracle_bytes(c)
    ops.kv8_write(c, k, v, pos)
    torch.cuda.synchronize()
    K8.write(ref, np64(k), np64(v), [pos] * B)
    check_cache(c, ref, [pos + S] * B)
    # rows behind the last one keep their bytes, blocks behind it their scales
    after = to_oracle_bytes(c)
    end = pos + S
    assert np.array_equal(after[0][:, :, end:], before[0][:, :, end:])
    assert np.array_equal(after[1][:, :, end:], before[1][:, :, end:])
    nb = -(-end // 64)
    for x, y in zip(after[2:], before[2:]):
        assert np.array_equal(x[:, :, nb:], y[:, :, nb:])


def to_oracle_bytes(c):
    """Raw bytes in token order, and the scales."""
    B, Hkv, cap, D = c.k.shape
    v = c.v.view(torch.uint8).cpu().numpy()[..., place()].transpose(0, 1, 2, 4, 3).reshape(B, Hkv, cap, D)
    return c.k.view(torch.uint8).cpu().numpy(), v, c.k_scale.cpu().numpy(), c.v_scale.cpu().numpy()


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("D", [32, 64, 128, 256])
def test_write_few_tokens(gpu, D, dtype):
    """A few tokens behind others, from two to more than the calls for few
    tokens take: inside a block, across two, at a block's first and last row,
    right-padded (to none in one sequence), with larger scales than the block's
    and with infinities and NaN."""
    from delta_attention import ops
    B, Hkv, cap, at_once = 5, 3, 192, 512 // D
    for S in (2, 3, at_once, at_once + 1, 2 * at_once, 2 * at_once + 1, 3 * at_once + 2, 64):
        c, ref = garbage(ops.kv8_empty(B, Hkv, cap, D), S), K8.new_cache(B, Hkv, cap, D)
        pos = [7, 64 - S // 2, 64, 127, 128 - S]
        k0, v0 = (tokens(B, 128, Hkv, D, DT[dtype], 50 + S + s) * 0.25 for s in (0, 1))
        counts = torch.tensor(pos, dtype=torch.int32, device="cuda")
        ops.kv8_write(c, k0, v0, 0, counts=counts)
        K8.write(ref, np64(k0), np64(v0), [0] * B, pos)
        for ragged, new in ((False, [S] * B), (True, [S, S - 1, 1, 0, S // 2 + 1])):
            k, v = (tokens(B, S, Hkv, D, DT[dtype], 70 + S + s) for s in (0, 1))
            k[0, S // 2, 1, 3], v[1, 0, 2, 5], v[2, 0, 0, 1] = float("inf"), float("nan"), 300.0
            given = torch.tensor(new, dtype=torch.int32, device="cuda") if ragged else None
            was = to_oracle_bytes(c)[:2]
            ops.kv8_write(c, k, v, torch.tensor(pos, device="cuda"), counts=given)
            K8.write(ref, np64(k), np64(v), pos, new)
            check_cache(c, ref, [a + n for a, n in zip(pos, new)])
            now = to_oracle_bytes(c)[:2]
            for b, (a, n) in enumerate(zip(pos, new)):     # rows behind keep their bytes
                assert all(same(x[b, :, a + n:], y[b, :, a + n:]) for x, y in zip(was, now)), (S, b)


@pytest.mark.parametrize("D", [32, 64, 128, 256])
def test_write_token_by_token(gpu, D):
    """Tokens appended one at a time, each larger than the last by up to 2^12:
    a block's earlier codes move to its larger scales, into the subnormals."""
    from delta_attention import ops
    B, Hkv, cap = 2, 2, 128
    c, ref = garbage(ops.kv8_empty(B, Hkv, cap, D), 7), K8.new_cache(B, Hkv, cap, D)
    for i in range(70):
        k, v = (tokens(B, 1, Hkv, D, torch.bfloat16, 100 + 2 * i + s, False) * 2.0 ** ((i * 5) % 13) for s in (0, 1))
        pos = torch.tensor([i, i + 3], device="cuda") if i else torch.zeros(2, dtype=torch.int64, device="cuda")
        if i == 1:    # the second sequence stands three rows further from here on
            k3, v3 = (tokens(1, 3, Hkv, D, torch.bfloat16, s) for s in (8, 9))
            ops.kv8_write(ops.KV8(*(t[1:] for t in c)), k3, v3, 1)
            one = {x: y[1:] for x, y in ref.items()}
            K8.write(one, np64(k3), np64(v3), [1])
        ops.kv8_write(c, k, v, pos)
        K8.write(ref, np64(k), np64(v), pos.tolist())
    check_cache(c, ref, [70, 73])


def test_write_special_values(gpu):
    """Zeros, the type's extremes and subnormals, infinities and NaN: the scale
    comes from the finite values, what has no code becomes NaN, and no other
    block or value is touched by it."""
    from delta_attention import ops
    for dtype in (torch.bfloat16, torch.float16):
        fi = torch.finfo(dtype)
        x = torch.zeros(1, 64 * 8, 1, 128, dtype=dtype)
        x[0, 64:128] = fi.max                                            # the largest
        x[0, 128:192] = fi.tiny * fi.eps                                 # the smallest subnormal
        x[0, 192:256] = torch.randn(64, 1, 128) * fi.tiny                # around the normal range's end
        x[0, 256:320] = torch.randn(64, 1, 128)
        x[0, 256, 0, :5] = torch.tensor([float("inf"), -float("inf"), float("nan"), -0.0, 447.9])
        x[0, 320:384] = float("inf")                                     # nothing finite
        x[0, 384:448] = torch.linspace(-448, 448, 64 * 128).view(64, 1, 128)
        x[0, 448:] = 2.0 ** (torch.arange(64 * 128) % 30 - 20).float().view(64, 1, 128)
        x = x.cuda()
        c, ref = ops.kv8_empty(1, 1, 512, 128), K8.new_cache(1, 1, 512, 128)
        ops.kv8_write(c, x, -x, 0)
        K8.write(ref, np64(x), np64(-x), [0])
        check_cache(c, ref, [512])
        # one more inside a block of moderate values: only the finite ones move the scale
        y = torch.full((1, 1, 1, 128), float("nan"), dtype=dtype, device="cuda")
        y[..., 3] = 1e4
        ops.kv8_write(c, y, y, 300)
        K8.write(ref, np64(y), np64(y), [300])
        check_cache(c, ref, [301])


def test_write_padded_and_refused_rows(gpu):
    """Counts per sequence (clamped to [0, S]); device positions whose rows do
    not fit leave their sequence unchanged."""
    from delta_attention import ops
    B, Hkv, D, cap, S = 6, 2, 64, 256, 90
    c = garbage(ops.kv8_empty(B, Hkv, cap, D), 3)
    before = [t.clone() for t in c]
    k, v = (tokens(B, S, Hkv, D, torch.float16, s) for s in (1, 2))
    pos = torch.tensor([0, 64, 0, 192, -1, 166], device="cuda")
    counts = torch.tensor([90, 33, -5, 70, 4, 1000], dtype=torch.int32, device="cuda")
    ops.kv8_write(c, k, v, pos, counts=counts)
    ref = K8.new_cache(B, Hkv, cap, D)
    K8.write(ref, np64(k), np64(v), pos.tolist(), counts.tolist())
    got = to_oracle(c)
    for b, (a, n) in enumerate(((0, 90), (64, 33), (166, 90))):
        b = (0, 1, 5)[b]
        if b == 5:     # its first block already held rows: their (noise) scale may stay the larger
            continue
        for x in ("k", "v"):
            assert same(got[x][b, :, a:a + n], ref[x][b, :, a:a + n])
    for b in (2, 3, 4):
        for t, u in zip(c, before):
            assert torch.equal(t[b].view(torch.uint8), u[b].view(torch.uint8)), b
    # one position and one count for all
    c2, c3 = ops.kv8_empty(B, Hkv, cap, D), ops.kv8_empty(B, Hkv, cap, D)
    ops.kv8_write(c2, k, v, torch.tensor([7], device="cuda"), counts=torch.tensor([50], dtype=torch.int32, device="cuda"))
    ops.kv8_write(c3, k[:, :50], v[:, :50], 7)
    for x in ("k", "v"):
        assert same(to_oracle(c2)[x][:, :, 7:57], to_oracle(c3)[x][:, :, 7:57])


def test_write_strides(gpu):
    """Strided tokens (views of one fused projection), and a cache that is a
    slice of a larger one over sequences and heads."""
    from delta_attention import ops
    B, S, Hkv, D = 2, 100, 2, 64
    big = tokens(B, S, 7, D, torch.bfloat16, 4)
    k, v = big[:, :, 2:4], big[:, :, 4:6]
    whole = garbage(ops.kv8_empty(5, 6, 128, D), 5)
    keep = [t.clone() for t in whole]
    part = ops.KV8(*(t[1:5:2, 3:5] for t in whole))
    ops.kv8_write(part, k, v, 9)
    kk, vv = ops.kv8_read(part, 64, 45)                      # a block written whole: no noise in its scale
    o = K8.new_cache(B, Hkv, 128, D)
    K8.write(o, np64(k), np64(v), [9] * B)
    ok, ov = K8.values(o, 64, 45)
    assert same(np64(kk), ok) and same(np64(vv), ov)
    for t, u in zip(whole, keep):
        for b in range(5):
            for h in range(6):
                if b not in (1, 3) or h not in (3, 4):
                    assert torch.equal(t[b, h].view(torch.uint8), u[b, h].view(torch.uint8))


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("B,Hkv,D,cap,start,n", [
    (1, 1, 128, 64, 0, 64), (1, 2, 64, 192, 1, 1), (2, 2, 32, 256, 63, 130), (1, 3, 256, 320, 100, 217),
    (1, 8, 128, 2048, 5, 2043),
])
def test_read(gpu, B, Hkv, D, cap, start, n, dtype):
    from delta_attention import ops
    c, ref = ops.kv8_empty(B, Hkv, cap, D), K8.new_cache(B, Hkv, cap, D)
    k, v = (tokens(B, cap, Hkv, D, torch.bfloat16, s) for s in (1, 2))
    k[0, min(70, cap - 1), 0, 3] = float("nan")
    k[:, : cap // 2] *= 2.0 ** 10                     # past float16's largest for some
    v[:, : cap // 2] *= 2.0 ** -14                    # into float16's subnormals
    ops.kv8_write(c, k, v, 0)
    K8.write(ref, np64(k), np64(v), [0] * B)
    want = []
    for x in K8.values(ref, start, n):
        top = float(torch.finfo(DT[dtype]).max)
        want.append(torch.from_numpy(np.clip(x, -top, top)).to(DT[dtype]))
    got = ops.kv8_read(c, start, n, dtype=DT[dtype])
    for x, y in zip(got, want):
        assert x.shape == (B, Hkv, n, D) and same(np64(x), np64(y))
    # rows behind each sequence's end are zero; strided outputs keep their other rows
    live = torch.tensor([start + n // 2 + b for b in range(B)], dtype=torch.int32, device="cuda")
    buf = torch.full((2, B, n + 3, Hkv, D), 7.0, dtype=DT[dtype], device="cuda")
    out = tuple(buf[i, :, 2:n + 2].transpose(1, 2) for i in (0, 1))
    ops.kv8_read(c, start, n, n_keys=live, out=out)
    for x, y in zip(out, want):
        y = np64(y)
        for b in range(B):
            y[b, :, max(int(live[b]) - start, 0):] = 0
        assert same(np64(x), y)
    assert (buf[:, :, :2] == 7).all() and (buf[:, :, n + 2:] == 7).all()


@pytest.mark.parametrize("D", [32, 64, 128, 256])
def test_write_and_read_many_blocks(gpu, D):
    """More workgroups than some rounds of the XCDs take, the last one not whole:
    every block of a padded batch is written and read once."""
    from delta_attention import ops
    B, Hkv, cap, S = 3, 3, 3200, 3111
    c, ref = garbage(ops.kv8_empty(B, Hkv, cap, D), D), K8.new_cache(B, Hkv, cap, D)
    k0, v0 = (tokens(B, 5, Hkv, D, torch.bfloat16, s) for s in (1, 2))
    k, v = (tokens(B, S, Hkv, D, torch.bfloat16, s) for s in (3, 4))
    new = [S, 2990, 64]
    ops.kv8_write(c, k0, v0, 0)
    ops.kv8_write(c, k, v, 5, counts=torch.tensor(new, dtype=torch.int32, device="cuda"))
    K8.write(ref, np64(k0), np64(v0), [0] * B)
    K8.write(ref, np64(k), np64(v), [5] * B, new)
    check_cache(c, ref, [5 + n for n in new])
    live = torch.tensor([5 + n for n in new], dtype=torch.int32, device="cuda")
    for start, n in ((0, cap), (61, 2999)):
        for x, y in zip(ops.kv8_read(c, start, n, n_keys=live), K8.values(ref, start, n)):
            for b, m in enumerate(new):
                y[b, :, max(5 + m - start, 0):] = 0
            assert same(np64(x), y), (start, n)


def filled(B, Hkv, cap, D, n, dtype, seed, scale=1.0):
    """A cache of noise with n[b] tokens of N(0, 1) times a varying factor."""
    from delta_attention import ops
    c, ref = garbage(ops.kv8_empty(B, Hkv, cap, D), seed), K8.new_cache(B, Hkv, cap, D)
    g = torch.Generator().manual_seed(seed + 1)
    k, v = ((torch.randn(B, max(max(n), 1), Hkv, D, generator=g)
             * torch.exp2(torch.randint(-1, 2, (B, 1, Hkv, 1), generator=g).float()) * scale).to(dtype).cuda() for _ in (0, 1))
    counts = torch.tensor(n, dtype=torch.int32, device="cuda")
    ops.kv8_write(c, k, v, 0, counts=counts)
    K8.write(ref, np64(k), np64(v), [0] * B, n)
    return c, ref, counts


def check_rows(got, q, ref, n, window, sink, scale, add=None, what=""):
    kk, vv = K8.values(ref)
    want, spread = K8.rows(np64(q), kk, vv, n, window, sink, scale)
    a = None if add is None else np64(add)
    tol = tolerance(want, spread, q.shape[3], max(max(n), 1), q.dtype, a)
    if a is not None:
        want = want + a
    d = np.abs(np64(got) - want)
    worst = float((d / tol).max())
    print(f"{what}: worst {worst:.3f} of the bound", flush=True)
    assert np.isfinite(np64(got)).all() and worst <= 1.0, (what, worst)


ROWS = [
    # B, Hkv, G, D, cap, n, s, window, sink
    (1, 1, 1, 128, 64, [1], 1, 0, 0),
    (1, 2, 4, 128, 64, [64], 1, 0, 0),
    (1, 2, 4, 128, 128, [65], 1, 0, 0),
    (2, 2, 4, 64, 1024, [1000, 3], 1, 0, 0),
    (3, 1, 5, 128, 2048, [0, 1, 2047], 1, 0, 0),              # an empty sequence
    (1, 2, 4, 128, 4096, [4001], 1, 512, 64),                 # sinks and a window
    (2, 2, 2, 32, 1024, [1021, 300], 1, 100, 7),
    (1, 1, 8, 256, 1024, [999], 1, 0, 0),
    (1, 2, 1, 256, 1024, [999], 1, 333, 20),
    (2, 2, 4, 128, 512, [500, 2], 6, 0, 0),                   # more rows than keys in one
    (1, 2, 4, 64, 2048, [2000], 5, 200, 33),
    (1, 1, 8, 128, 512, [400], 4, 0, 0),                      # 32 rows
    (1, 1, 12, 64, 512, [400], 5, 130, 3),                    # 60 rows
    (1, 2, 4, 256, 512, [300], 7, 0, 0),                      # 28 rows, head_dim 256
    (1, 1, 4, 128, 512, [290], 100, 0, 0),                    # 400 rows: several row tiles
    (1, 1, 8, 256, 256, [200], 9, 64, 10),                    # 72 rows, head_dim 256
    (70, 1, 2, 32, 128, [(i * 37) % 129 for i in range(70)], 1, 0, 0),   # more sequences than lanes
    (1, 1, 4, 128, 20480, [20001], 1, 0, 0),                  # a long one: many splits
    (2, 1, 20, 128, 8192, [8192, 100], 1, 1000, 5000),        # sinks past the window's start
    (300, 1, 1, 32, 192, [(i * 53) % 193 for i in range(300)], 1, 0, 0),  # more than are kept in registers
    (3, 2, 8, 64, 1024, [1000, 0, 513], 40, 100, 70),         # several row tiles, ragged, windows
    (1, 1, 1, 128, 131072, [70], 1, 0, 0),                    # a few keys of a large capacity
    (2, 1, 16, 32, 256, [256, 3], 4, 0, 0),                   # 64 rows, more rows than keys
    (70, 1, 2, 32, 4224, [4200 if i % 23 == 5 else (i * 37) % 300 for i in range(70)], 1, 0, 0),    # as above, split
    (260, 1, 1, 32, 4160, [4160 if i in (3, 258) else (i * 53) % 400 for i in range(260)], 1, 0, 0),
    (66, 1, 3, 64, 4224, [(i * 997) % 4225 for i in range(66)], 2, 4100, 100),                      # and with a window
    (5, 2, 4, 128, 640, [640, 0, 1, 333, 577], 1, 0, 0),      # the longest lists that stay whole,
    (5, 2, 4, 128, 704, [704, 0, 1, 333, 577], 1, 0, 0),      # and one block more
    (24, 4, 2, 64, 1536, [(i * 611) % 1537 for i in range(24)], 5, 0, 0),       # whole for their number
    (40, 8, 1, 128, 3008, [(i * 733) % 2561 for i in range(40)], 1, 2300, 150), # whole by their windows
]


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("B,Hkv,G,D,cap,n,s,window,sink", ROWS)
def test_rows(gpu, B, Hkv, G, D, cap, n, s, window, sink, dtype):
    from delta_attention import ops
    c, ref, counts = filled(B, Hkv, cap, D, n, DT[dtype], 17 * B + cap + s)
    q = tokens(B, s, Hkv * G, D, DT[dtype], 5, False).transpose(1, 2)
    scale = D ** -0.5
    got = ops.kv8_attention(q, c, n_keys=counts, window=window, sink=sink, sm_scale=scale)
    assert got.shape == q.shape and got.dtype == q.dtype
    what = f"B{B} H{Hkv * G}/{Hkv} D{D} n{n[:3]} s{s} w{window} k{sink} {dtype}"
    check_rows(got, q, ref, n, window, sink, scale, what=what)
    add = tokens(B, s, Hkv * G, D, DT[dtype], 6, False).transpose(1, 2)
    got = ops.kv8_attention(q, c, n_keys=counts, window=window, sink=sink, sm_scale=scale, add=add)
    check_rows(got, q, ref, n, window, sink, scale, add, what=what + " add")
    if len(set(n)) == 1:     # the host's count
        got = ops.kv8_attention(q, c, n_keys=n[0], window=window, sink=sink, sm_scale=scale)
        check_rows(got, q, ref, n, window, sink, scale, what=what + " host count")


@pytest.mark.parametrize("seed", range(24))
def test_random_runs(gpu, seed):
    """Random shapes, types and lengths: a padded prompt, a chunk and tokens into
    a cache of noise, then rows over it and a stretch read back."""
    import random
    from delta_attention import ops
    r = random.Random(1000 + seed)
    B, Hkv, G, D = r.choice([1, 1, 2, 3, 5]), r.choice([1, 2, 3]), r.choice([1, 2, 3, 4, 7, 9]), r.choice([32, 64, 128, 256])
    dtype = DT[r.choice(["bf16", "fp16"])]
    cap = 64 * r.randint(1, 9)
    c, ref = garbage(ops.kv8_empty(B, Hkv, cap, D), seed), K8.new_cache(B, Hkv, cap, D)
    n = [0] * B
    print(f"seed {seed}: B{B} H{Hkv * G}/{Hkv} D{D} cap {cap} {dtype}", flush=True)
    for step in range(r.randint(1, 4)):
        S = min(r.choice([1, 1, r.randint(1, 40), r.randint(1, cap)]), cap - max(n))
        if S < 1:
            break
        cnt = [S] * B if r.random() < 0.5 else [r.randint(0, S) for _ in range(B)]
        k, v = (tokens(B, S, Hkv, D, dtype, seed * 50 + 2 * step + i) for i in (0, 1))
        ops.kv8_write(c, k, v, torch.tensor(n, device="cuda"), counts=torch.tensor(cnt, dtype=torch.int32, device="cuda"))
        K8.write(ref, np64(k), np64(v), n, cnt)
        n = [a + b for a, b in zip(n, cnt)]
    check_cache(c, ref, n)
    s = r.choice([1, 1, 2, r.randint(1, 12), 33])
    window = r.choice([0, 0, r.randint(1, cap), 2 ** 31 - 1])
    sink = r.choice([0, r.randint(0, 130)])
    scale = r.choice([D ** -0.5, 0.3, -0.05])
    q = tokens(B, s, Hkv * G, D, dtype, seed, False).transpose(1, 2)
    live = {x: np.nan_to_num(y) if x in ("k", "v") else y for x, y in ref.items()}   # (no key past n is looked at)
    got = ops.kv8_attention(q, c, n_keys=torch.tensor(n, dtype=torch.int32, device="cuda"), window=window, sink=sink,
                            sm_scale=scale)
    check_rows(got, q, live, n, window, sink, scale, what=f"seed {seed} n{n} s{s} w{window} k{sink} scale {scale:.3f}")
    a = r.randint(0, cap - 1)
    m = r.randint(1, cap - a)
    kk, vv = ops.kv8_read(c, a, m, n_keys=torch.tensor(n, dtype=torch.int32, device="cuda"), dtype=dtype)
    for x, y in zip((kk, vv), K8.values(live, a, m)):
        for b in range(B):
            y[b, :, max(n[b] - a, 0):] = 0
        assert same(np64(x), np64(torch.from_numpy(y).to(dtype)))


@pytest.mark.parametrize("seed", range(16))
def test_random_split_rows(gpu, seed):
    """Random shapes at capacities whose lists are split or just not: the count
    given by the host, by one device entry and by one per sequence, and a
    recorded call of the last two that serves other lengths."""
    import random
    from delta_attention import ops
    r = random.Random(7000 + seed)
    B, Hkv, G, D = r.choice([1, 1, 2, 3, 6, 67]), r.choice([1, 2, 4]), r.choice([1, 2, 4, 9]), r.choice([32, 64, 128, 256])
    dtype, s = DT[r.choice(["bf16", "fp16"])], r.choice([1, 1, 2, 5, 12])
    most = max(4, min(90, 2 ** 21 // (64 * B * Hkv * D)))
    cap = 64 * r.randint(most // 2, most)
    window = r.choice([0, 0, r.randint(1, cap)])
    sink, scale = r.choice([0, r.randint(0, 200)]), r.choice([D ** -0.5, -0.05])
    c, ref, _ = filled(B, Hkv, cap, D, [cap] * B, dtype, 90 + seed)
    q = tokens(B, s, Hkv * G, D, dtype, 91 + seed, False).transpose(1, 2)
    what = f"seed {seed}: B{B} H{Hkv * G}/{Hkv} D{D} cap {cap} s{s} w{window} k{sink}"

    def rows(n_keys):
        return ops.kv8_attention(q, c, n_keys=n_keys, window=window, sink=sink, sm_scale=scale)

    n = r.randint(1, cap)
    check_rows(rows(n), q, ref, [n] * B, window, sink, scale, what=what + " host")
    for form in ("one", "each"):
        now = torch.zeros(1 if form == "one" else B, dtype=torch.int32, device="cuda")
        rows(now)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = rows(now)
        for n in (cap, r.randint(1, cap), 0, 1, r.randint(cap // 2, cap)):
            lens = [n] * B if form == "one" else [r.randint(0, n) if b else n for b in range(B)]
            now.copy_(torch.tensor(lens[:now.numel()], dtype=torch.int32))
            graph.replay()
            assert torch.equal(out, rows(now)), (what, form, lens[:4])
            check_rows(out, q, ref, lens, window, sink, scale, what=f"{what} {form} {lens[:3]}")


def test_offsets_past_32_bits(gpu):
    """Sequences of 16M tokens at head_dim 256: codes 4 GiB into a head, the
    second sequence past them; tokens at both ends, a window's rows, a read."""
    from delta_attention import ops
    cap, D = 1 << 24, 256
    c = ops.kv8_empty(2, 1, cap, D)
    head = [tokens(2, 70, 1, D, torch.bfloat16, x, False) for x in (1, 2)]
    tail = [tokens(2, 203, 1, D, torch.bfloat16, x, False) for x in (3, 4)]
    ops.kv8_write(c, *head, 0)
    at = cap - 204
    ops.kv8_write(c, *tail, torch.tensor([at, at], device="cuda"))
    one = [tokens(2, 1, 1, D, torch.bfloat16, x, False) for x in (5, 6)]
    ops.kv8_write(c, *one, cap - 1)
    # the same tokens in a short cache whose blocks lie alike: 70 at the start, 204 to the end
    short = ops.kv8_empty(2, 1, 384, D)
    ops.kv8_write(short, *head, 0)
    ops.kv8_write(short, *tail, 384 - 204)
    ops.kv8_write(short, *one, 383)
    for x, y in zip(ops.kv8_read(c, at, 204), ops.kv8_read(short, 180, 204)):
        assert torch.equal(x, y)
    q = tokens(2, 2, 4, D, torch.bfloat16, 7, False).transpose(1, 2)
    kw = dict(window=150, sink=70, sm_scale=0.06)
    assert torch.equal(ops.kv8_attention(q, c, n_keys=cap, **kw), ops.kv8_attention(q, short, n_keys=384, **kw))


def test_rows_large_scores(gpu):
    """Scores from -300 to 300 with the largest late: the running reference
    moves up many times, and rows end with one key's value."""
    from delta_attention import ops
    B, Hkv, G, D, n = 1, 1, 4, 128, 1500
    c, ref, counts = filled(B, Hkv, 1536, D, [n], torch.float16, 3, scale=3.0)
    q = tokens(B, 1, G, D, torch.float16, 5, False).transpose(1, 2) * 8
    got = ops.kv8_attention(q, c, n_keys=counts, sm_scale=1.0)
    check_rows(got, q, ref, [n], 0, 0, 1.0, what="large scores")


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_rows_other_scales(gpu, dtype):
    """A negative scale, and zero (every key weighs alike)."""
    from delta_attention import ops
    n = [700, 64]
    c, ref, counts = filled(2, 2, 1024, 64, n, DT[dtype], 40)
    q = tokens(2, 2, 6, 64, DT[dtype], 41, False).transpose(1, 2)
    for scale in (-0.2, 0.0, 1e-30):
        got = ops.kv8_attention(q, c, n_keys=counts, window=200, sink=3, sm_scale=scale)
        check_rows(got, q, ref, n, 200, 3, scale, what=f"scale {scale}")
    for bad in (float("nan"), float("inf"), 1e39):
        with pytest.raises(AssertionError):
            ops.kv8_attention(q, c, n_keys=counts, sm_scale=bad)


def test_rows_huge_scores_and_infinite_queries(gpu):
    """Scores near float32's ends (finite bf16 inputs) pick the largest; a query
    with an infinity or NaN gives its own row NaN and no other."""
    from delta_attention import ops
    D, n = 64, 130
    k = torch.zeros(1, n, 1, D, dtype=torch.bfloat16, device="cuda")
    k[0, :, 0, 0] = torch.linspace(-1, 1, n)
    v = tokens(1, n, 1, D, torch.bfloat16, 2, False)
    c = ops.kv8_empty(1, 1, 192, D)
    ops.kv8_write(c, k, v, 0)
    q = torch.zeros(1, 4, 1, D, dtype=torch.bfloat16, device="cuda")
    q[0, 0, 0, 0], q[0, 1, 0, 0] = 1e38, -1e38
    q[0, 2, 0, 0] = float("inf")
    q[0, 3, 0, 1] = 1.0
    got = ops.kv8_attention(q, c, n_keys=n, sm_scale=1.0)
    kk, vv = ops.kv8_read(c, 0, n)
    for h, at in ((0, kk[0, 0, :, 0].argmax()), (1, kk[0, 0, :, 0].argmin())):
        same_k = kk[0, 0, :, 0] == kk[0, 0, at, 0]            # (codes tie: the row is their mean)
        want = vv[0, 0, same_k].float().mean(0)
        assert (got[0, h, 0].float() - want).abs().max() <= 2.0 ** -7 * max(1.0, want.abs().max().item())
    assert got[0, 2].isnan().all()
    want = vv[0, 0].float().mean(0)
    assert (got[0, 3, 0].float() - want).abs().max() <= 2.0 ** -8
    low = ops.kv8_attention(-q[:, :1].abs() * 3, c, n_keys=1, sm_scale=1.0)   # one key, its score +3e38
    assert torch.equal(low[0, 0, 0], vv[0, 0, 0])


@pytest.mark.parametrize("early,late,scale", [(-3e38, -9e37, 2e-38), (-3e38, 3e38, 1.2e-38), (3e38, -3e38, 1.2e-38)])
def test_rows_scores_of_floats_ends(gpu, early, late, scale):
    """Scores near float32's ends under a scale near its smallest: a wave's
    first blocks, which such a scale leaves within reach of a row without keys,
    still count when later blocks move the row's reference, and so do keys
    further from the largest score than float32 reaches."""
    from delta_attention import ops
    B, Hkv, n, D = 64, 16, 1024, 32                   # one item per head, four blocks a wave
    k = torch.zeros(B, n, Hkv, D, dtype=torch.bfloat16, device="cuda")
    k[..., 0] = early / 2e19
    k[:, -64:, :, 0] = late / 2e19
    v = tokens(B, n, Hkv, D, torch.bfloat16, 3, False)
    c = ops.kv8_empty(B, Hkv, n, D)
    ops.kv8_write(c, k, v, 0)
    q = torch.zeros(B, Hkv, 1, D, dtype=torch.bfloat16, device="cuda")
    q[..., 0] = 2e19
    got = ops.kv8_attention(q, c, n_keys=n, sm_scale=scale)
    check_rows(got, q, to_oracle(c), [n] * B, 0, 0, float(np.float32(scale)), what=f"scores {early} then {late}")


def test_rows_shared_prefix_and_refused_writes(gpu):
    """One sequence's cache expanded over a batch serves its rows (a shared
    prompt); writing through the expansion is refused."""
    from delta_attention import ops
    c, ref, _ = filled(1, 2, 512, 64, [400], torch.bfloat16, 12)
    many = ops.KV8(*(t.expand(5, *t.shape[1:]) for t in c))
    q = tokens(5, 2, 6, 64, torch.bfloat16, 13, False).transpose(1, 2)
    got = ops.kv8_attention(q, many, n_keys=torch.tensor([400], dtype=torch.int32, device="cuda"), sm_scale=0.125)
    check_rows(got, q, {x: np.repeat(y, 5, 0) for x, y in ref.items()}, [400] * 5, 0, 0, 0.125, what="shared")
    with pytest.raises(AssertionError, match="invalid"):
        ops.kv8_write(many, tokens(5, 1, 2, 64, torch.bfloat16, 1), tokens(5, 1, 2, 64, torch.bfloat16, 2), 400)


def test_gpu_refusals(gpu):
    """Arguments that only fail with GPU tensors: counts and positions of the
    wrong type, size or device; keys past the capacity; results unlike q."""
    from delta_attention import ops
    c = ops.kv8_empty(2, 2, 128, 64)
    k = tokens(2, 3, 2, 64, torch.bfloat16, 1)
    q = tokens(2, 1, 4, 64, torch.bfloat16, 2).transpose(1, 2)
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")
    for bad in (i32(0, 1), torch.tensor([0, 1, 2], device="cuda"), torch.tensor([0, 1]), torch.tensor([[0, 1]], device="cuda"),
                torch.arange(4, device="cuda")[::2], -1, 126):
        with pytest.raises(AssertionError):
            ops.kv8_write(c, k, k, bad)
    with pytest.raises(AssertionError):
        ops.kv8_write(c, k, k, 0, counts=torch.tensor([1, 2], device="cuda"))
    with pytest.raises(AssertionError):
        ops.kv8_write(c, k.cpu(), k, 0)
    for bad in (129, -1, i32(1, 2, 3), torch.tensor([1, 2], device="cuda")):
        with pytest.raises(AssertionError):
            ops.kv8_attention(q, c, n_keys=bad, sm_scale=1.0)
    with pytest.raises(AssertionError):
        ops.kv8_attention(q, c, n_keys=1, sm_scale=1.0, out=torch.empty(2, 4, 1, 64, dtype=torch.float16, device="cuda"))
    with pytest.raises(AssertionError):
        ops.kv8_attention(q, c, n_keys=1, sm_scale=1.0, add=q[:, :2])
    with pytest.raises(AssertionError):
        ops.kv8_read(c, 0, 5, dtype=torch.float32)
    # nothing to do is no error
    assert ops.kv8_attention(q[:, :, :0], c, n_keys=1, sm_scale=1.0).shape == (2, 4, 0, 64)
    assert ops.kv8_read(c, 7, 0)[0].shape == (2, 2, 0, 64)
    ops.kv8_write(c, k[:, :0], k[:, :0], 128)


def test_rows_in_place_and_unaligned(gpu):
    """The result written over q; q and the tokens at addresses and strides that
    are not 16-byte aligned."""
    from delta_attention import ops
    c, ref, counts = filled(2, 1, 1024, 64, [1000, 70], torch.bfloat16, 14)
    q = tokens(2, 2, 4, 64, torch.bfloat16, 15, False).transpose(1, 2)
    want = ops.kv8_attention(q, c, n_keys=counts, sm_scale=0.1)
    raw = torch.empty(q.numel() + 1, dtype=q.dtype, device="cuda")[1:]
    odd = raw.view(2, 4, 2, 64).copy_(q)
    assert odd.data_ptr() % 16 and torch.equal(ops.kv8_attention(odd, c, n_keys=counts, sm_scale=0.1), want)
    k = tokens(2, 5, 1, 64, torch.bfloat16, 16)
    wide = torch.zeros(2, 5, 1, 67, dtype=k.dtype, device="cuda")
    wide[..., 2:66] = k
    c2 = ops.KV8(*(t.clone() for t in c))
    ops.kv8_write(c, k, k, 1000)
    ops.kv8_write(c2, wide[..., 2:66], wide[..., 2:66], 1000)
    for a, b in zip(c, c2):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
    # (the write moved the earlier codes of its block to a larger scale)
    want = ops.kv8_attention(q, c, n_keys=counts, sm_scale=0.1)
    qq = q.clone()
    ops.kv8_attention(qq, c, n_keys=counts, sm_scale=0.1, out=qq)
    assert torch.equal(qq, want)


def test_rows_nan_in_masked_places(gpu):
    """NaN keys and values that a row does not see (behind the last key, before
    its window, of later rows) do not reach it; the rows that see one are NaN
    in its columns."""
    from delta_attention import ops
    B, Hkv, G, D, cap, n, s, window, sink = 1, 1, 2, 64, 512, 300, 4, 70, 5
    for at, tensor in ((298, "v"), (229, "v"), (100, "v"), (3, "v"), (6, "v"), (298, "k"), (150, "k")):
        k, v = (tokens(B, n, Hkv, D, torch.bfloat16, x, False) for x in (1, 2))
        (k if tensor == "k" else v)[0, at, 0, 9] = float("nan")
        c = garbage(ops.kv8_empty(B, Hkv, cap, D), at)
        ops.kv8_write(c, k, v, 0)
        q = tokens(B, s, G, D, torch.bfloat16, 3, False).transpose(1, 2)
        got = np64(ops.kv8_attention(q, c, n_keys=n, window=window, sink=sink, sm_scale=0.125))
        for i in range(s):
            r = n - s + i
            sees = at <= r and (at < sink or at > r - window)
            bad = np.isnan(got[0, :, i])
            want = np.zeros_like(bad)
            if sees and tensor == "k":
                want[:] = True
            elif sees:
                want[:, 9] = True
            assert np.array_equal(bad, want), (at, tensor, i)


def test_rows_strides_and_outputs(gpu):
    """Strided queries and outputs (other rows kept), a sliced cache."""
    from delta_attention import ops
    B, Hkv, G, D, n = 2, 2, 3, 64, [200, 131]
    c, ref, counts = filled(B, Hkv, 256, D, n, torch.bfloat16, 8)
    big = tokens(B, 3, 2 * Hkv * G, D, torch.bfloat16, 9, False)
    q = big[:, 1:3, Hkv * G:].transpose(1, 2)
    buf = torch.full((B, 4, Hkv * G, D), 7.0, dtype=torch.bfloat16, device="cuda")
    out = buf[:, 1:3].transpose(1, 2)
    got = ops.kv8_attention(q, c, n_keys=counts, sm_scale=0.1, out=out)
    assert got is out
    check_rows(out, q, ref, n, 0, 0, 0.1, what="strided")
    assert (buf[:, 0] == 7).all() and (buf[:, 3] == 7).all()
    part = ops.KV8(*(t[:, 1:] for t in c))
    one = ops.kv8_attention(q[:, G:], part, n_keys=counts, sm_scale=0.1)
    check_rows(one, q[:, G:], {x: y[:, 1:] for x, y in ref.items()}, n, 0, 0, 0.1, what="one head's cache")


def test_rows_repeat_and_streams(gpu):
    """The same call twice, on another stream and beside another call gives the
    same bits."""
    from delta_attention import ops
    c, ref, counts = filled(2, 2, 4096, 128, [4001, 977], torch.bfloat16, 21)
    q = tokens(2, 1, 8, 128, torch.bfloat16, 22, False).transpose(1, 2)
    call = lambda: ops.kv8_attention(q, c, n_keys=counts, sm_scale=0.09)
    a = call()
    torch.cuda.synchronize()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    with torch.cuda.stream(s1):
        b = [call() for _ in range(3)]
    with torch.cuda.stream(s2):
        d = [call() for _ in range(3)]
    torch.cuda.synchronize()
    assert all(torch.equal(a, x) for x in b + d)


def test_append_and_rows_in_a_graph(gpu):
    """A decode step (append one token per sequence, attend) recorded once and
    replayed while positions and counts advance on the device, against the
    same steps run eagerly on a second cache: every replay's bits."""
    from delta_attention import ops
    B, Hkv, G, D, cap = 2, 2, 4, 128, 320
    n0 = [62, 130]
    caches = [filled(B, Hkv, cap, D, n0, torch.bfloat16, 31)[0] for _ in (0, 1)]
    src = [tokens(B, 80, Hkv, D, torch.bfloat16, s) for s in (1, 2)]
    qs = tokens(B, 80, Hkv * G, D, torch.bfloat16, 3, False)
    k, v = (torch.empty(B, 1, Hkv, D, dtype=torch.bfloat16, device="cuda") for _ in (0, 1))
    q = torch.empty(B, Hkv * G, 1, D, dtype=torch.bfloat16, device="cuda")
    out = torch.empty_like(q)

    def step(c, pos, counts):
        ops.kv8_write(c, k, v, pos)
        ops.kv8_attention(q, c, n_keys=counts, window=100, sink=9, sm_scale=0.09, out=out)
        pos.add_(1)
        counts.add_(1)

    def load(i):
        k.copy_(src[0][:, i:i + 1])
        v.copy_(src[1][:, i:i + 1])
        q.copy_(qs[:, i:i + 1].transpose(1, 2))

    pos = [torch.tensor(n0, device="cuda") for _ in (0, 1)]
    cnt = [(p + 1).to(torch.int32) for p in pos]
    load(0)
    for j in (0, 1):
        step(caches[j], pos[j], cnt[j])
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        step(caches[0], pos[0], cnt[0])
    for i in range(1, 80):
        load(i)
        g.replay()
        got = out.clone()
        step(caches[1], pos[1], cnt[1])
        assert torch.equal(got, out), i
    # both sequences' last rows against the rows recomputed from the whole history
    for a, b in zip(to_oracle(caches[0]).values(), to_oracle(caches[1]).values()):
        assert same(a, b)


def test_prompt_chunk_token_run(gpu):
    """Used together: a padded prompt, a chunk behind it, tokens one by one, rows
    after each; the read-back through the framework's rows kernel agrees with the
    cache's own rows."""
    from delta_attention import ops
    from delta_attention.delta_kernel import attention as rows_attention
    B, Hkv, G, D, cap = 2, 2, 4, 128, 512
    c, ref = ops.kv8_empty(B, Hkv, cap, D), K8.new_cache(B, Hkv, cap, D)
    n = [0, 0]
    scale = D ** -0.5
    for step, (S, cnt) in enumerate([(200, [200, 151]), (70, [70, 70]), (1, [1, 1]), (1, [1, 1])]):
        k, v = (tokens(B, S, Hkv, D, torch.bfloat16, 50 + 2 * step + s, False) for s in (0, 1))
        ops.kv8_write(c, k, v, torch.tensor(n, device="cuda"),
                      counts=torch.tensor(cnt, dtype=torch.int32, device="cuda"))
        K8.write(ref, np64(k), np64(v), n, cnt)
        n = [a + b for a, b in zip(n, cnt)]
        check_cache(c, ref, n)
        q = tokens(B, 3, Hkv * G, D, torch.bfloat16, 60 + step, False).transpose(1, 2)
        got = ops.kv8_attention(q, c, n_keys=torch.tensor(n, dtype=torch.int32, device="cuda"), sm_scale=scale)
        check_rows(got, q, ref, n, 0, 0, scale, what=f"step {step}")
    for b in range(B):
        one = ops.KV8(*(t[b:b + 1] for t in c))
        kk, vv = ops.kv8_read(one, 0, n[b])
        mask = torch.arange(n[b] - 3, n[b], device="cuda")[None]
        rows = rows_attention(q[b:b + 1].contiguous(), kk, vv, mask, scale)
        assert (rows.float() - got[b:b + 1].float()).abs().max().item() < 2e-2
