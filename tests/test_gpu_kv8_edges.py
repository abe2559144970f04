"""The 8-bit key/value cache at the ends of what its calls allow: what they
refuse on a GPU, the largest keys, scores of infinity, lengths past the
capacity."""

import numpy as np
import pytest
import torch

from helpers import np64
from kv8_helpers import to_oracle, tolerance
from oracle import kv8_oracle as K8

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "fp16": torch.float16}


def test_results_that_share_their_place_are_refused(gpu):
    """A result expanded over sequences, heads or rows; one of a single entry
    there may have any stride."""
    from delta_attention import ops
    c = ops.kv8_empty(2, 2, 128, 64)
    k = torch.randn(2, 100, 2, 64, device="cuda").bfloat16()
    ops.kv8_write(c, k, k, 0)
    q = torch.randn(2, 4, 3, 64, device="cuda").bfloat16()
    for i in range(3):
        one = [1 if j == i else x for j, x in enumerate((2, 4, 3))]
        with pytest.raises(AssertionError, match="invalid"):
            ops.kv8_attention(q, c, n_keys=100, sm_scale=0.1, out=torch.empty(*one, 64, device="cuda").bfloat16().expand(2, 4, 3, 64))
        one = [1 if j == i else x for j, x in enumerate((2, 2, 5))]
        out = [torch.empty(*s, 64, device="cuda").bfloat16().expand(2, 2, 5, 64) for s in (one, (2, 2, 5))]
        for pair in (out, out[::-1]):
            with pytest.raises(AssertionError, match="invalid"):
                ops.kv8_read(c, 0, 5, out=pair)
    want = ops.kv8_attention(q[:1, :, :1], ops.KV8(*(t[:1] for t in c)), n_keys=100, sm_scale=0.1)
    out = torch.empty(4, 64, device="cuda").bfloat16().as_strided((1, 4, 1, 64), (0, 64, 0, 1))
    ops.kv8_attention(q[:1, :, :1], ops.KV8(*(t[:1] for t in c)), n_keys=100, sm_scale=0.1, out=out)
    assert torch.equal(out, want)


def test_out_of_memory_is_torchs(gpu):
    """Results past the card's memory raise torch's own error: a long cache
    expanded over sequences asks for 2 TB."""
    from delta_attention import ops
    c = ops.KV8(*(t.expand(1 << 28, *t.shape[1:]) for t in ops.kv8_empty(1, 1, 64, 32)))
    with pytest.raises(torch.OutOfMemoryError):
        ops.kv8_read(c, 0, 64)


def test_write_padded_past_the_capacity(gpu):
    """A padded length past the capacity, up to the largest int32, with counts
    that fit: the counts' tokens are written, and nothing else."""
    from delta_attention import ops
    B, Hkv, D, cap = 2, 2, 64, 256
    for S in (300, 2 ** 31 - 1):
        k, v = (torch.randn(B, 1, Hkv, D, device="cuda").bfloat16() for _ in (0, 1))
        c, ref = ops.kv8_empty(B, Hkv, cap, D), K8.new_cache(B, Hkv, cap, D)
        for t in c[:2]:
            t.view(torch.uint8).fill_(0x55)
        counts, pos = [90, 7], [100, 249]
        first = torch.randn(B, 256, Hkv, D, device="cuda").bfloat16()
        ops.kv8_write(c, first, first, 0, counts=torch.tensor(pos, dtype=torch.int32, device="cuda"))
        K8.write(ref, np64(first), np64(first), [0, 0], pos)
        ops.kv8_write(c, k.expand(B, S, Hkv, D), v.expand(B, S, Hkv, D), torch.tensor(pos, device="cuda"),
                      counts=torch.tensor(counts, dtype=torch.int32, device="cuda"))
        K8.write(ref, *(np64(x.expand(B, 90, Hkv, D)) for x in (k, v)), pos, counts)
        got = to_oracle(c)
        for b in range(B):
            n = pos[b] + counts[b]
            for x in ("k", "v"):
                assert np.array_equal(got[x][b, :, :n], ref[x][b, :, :n]), (S, b, x)
                assert (got[x][b, :, n:] == 13.0).all()            # (0x55)
            for x in ("ke", "ve"):
                assert np.array_equal(got[x][b, :, :-(-n // 64)], ref[x][b, :, :-(-n // 64)]), (S, b, x)


@pytest.mark.parametrize("D,G,s,n", [
    (32, 1, 1, 100), (64, 4, 1, 4000), (128, 4, 1, 100), (128, 4, 1, 20001), (256, 2, 1, 3000),   # one row tile a wave
    (64, 4, 6, 2000), (128, 8, 4, 500), (256, 8, 4, 500),                                         # two
    (32, 8, 8, 700), (128, 8, 8, 700), (128, 4, 40, 500),                                         # four, and several
])
def test_rows_of_the_largest_keys(gpu, D, G, s, n):
    """Keys up to bfloat16's largest: their codes reach 256 * 2^120, which no
    bfloat16 and no float32 holds, though their scores are ordinary."""
    from delta_attention import ops
    g = torch.Generator().manual_seed(D + n)
    top = torch.finfo(torch.bfloat16).max
    k = torch.randn(1, n, 2, D, generator=g) * 2.0 ** 126
    k[0, ::7, :, 3] = float(top)
    k[0, 5::11, 1, 0] = -float(top)
    k = k.clamp(-float(top), float(top)).to(torch.bfloat16)
    k[0, n // 2:n // 2 + 70] *= 2.0 ** -8                # (and a block or two of a smaller scale)
    v = torch.randn(1, n, 2, D, generator=g).to(torch.bfloat16)
    q = (1 + torch.rand(1, 2 * G, s, D, generator=g)) * 2.0 ** -125
    q = (q * (torch.randint(0, 2, q.shape, generator=g) * 2 - 1)).to(torch.bfloat16)
    c, ref = ops.kv8_empty(1, 2, n, D), K8.new_cache(1, 2, -(-n // 64) * 64, D)
    for t in c[:2]:
        t.view(torch.uint8).fill_(0x7f)
    ops.kv8_write(c, k.cuda(), v.cuda(), 0)
    K8.write(ref, np64(k), np64(v), [0])
    assert ref["ke"].max() == 120 and np.nanmax(np.abs(ref["k"])) >= 256
    kk, vv = K8.values(ref)
    for scale in (D ** -0.5, -0.02):
        got = ops.kv8_attention(q.cuda(), c, n_keys=n, sm_scale=scale)
        want, spread = K8.rows(np64(q), kk, vv, [n], 0, 0, scale)
        tol = tolerance(want, spread, D, n, torch.bfloat16)
        d = np.abs(np64(got) - want)
        assert np.isfinite(np64(got)).all() and (d <= tol).all(), float((d / tol).max())


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("D,cap,n,s,window", [(128, 128, 70, 3, 0), (64, 8192, 8000, 2, 0), (128, 8192, 8000, 9, 700),
                                              (256, 4096, 4001, 1, 0), (32, 256, 2, 4, 0)])
def test_rows_whose_every_score_is_minus_infinity(gpu, D, cap, n, s, window, dtype):
    """They have no softmax: NaN. Zeros are for rows without keys alone."""
    from delta_attention import ops
    g = torch.Generator().manual_seed(n)
    k = torch.randn(1, n, 1, D, generator=g)
    k[..., 5] = 1 + torch.rand(1, n, 1, generator=g)
    c = ops.kv8_empty(1, 1, cap, D)
    ops.kv8_write(c, k.to(DT[dtype]).cuda(), k.to(DT[dtype]).cuda(), 0)
    q = torch.randn(1, 4, s, D, generator=g).to(DT[dtype]).cuda()
    count = torch.tensor([n], dtype=torch.int32, device="cuda")
    for keys in (n, count):
        usual = ops.kv8_attention(q, c, n_keys=keys, window=window, sm_scale=0.1)
        bad = q.clone()
        bad[0, 2, :, 5] = -float("inf")
        got = ops.kv8_attention(bad, c, n_keys=keys, window=window, sm_scale=0.1)
        empty = max(s - n, 0)                             # rows before the sequence's start
        assert (got[:, :, :empty] == 0).all() and got[0, 2, empty:].isnan().all()
        for h in (0, 1, 3):
            assert torch.equal(got[0, h], usual[0, h])
    # sequences of different lengths, the count of each on the device
    two = ops.KV8(*(t.expand(3, *t.shape[1:]) for t in c))
    lens = torch.tensor([n, 1, 0], dtype=torch.int32, device="cuda")
    got = ops.kv8_attention(bad.expand(3, 4, s, D), two, n_keys=lens, window=window, sm_scale=0.1)
    for b, m in enumerate((n, 1, 0)):
        empty = max(s - m, 0)
        assert (got[b, :, :empty] == 0).all() and got[b, 2, empty:].isnan().all()
        assert got[b, [0, 1, 3]].isfinite().all()


@pytest.mark.parametrize("D,S", [(64, 1), (256, 1), (64, 3), (256, 2), (64, 16), (256, 4), (128, 90), (32, 200), (256, 64)])
def test_write_clamps_counts(gpu, D, S):
    """Counts above S write S tokens, those below zero none, by every kernel of
    the write: behind rows that were written before, up to the capacity's end,
    and the rows behind keep their bytes."""
    from delta_attention import ops
    B, Hkv, cap = 4, 2, 512
    c, ref = ops.kv8_empty(B, Hkv, cap, D), K8.new_cache(B, Hkv, cap, D)
    for t in c[:2]:
        t.view(torch.uint8).fill_(0x55)                            # 13
    pos = [0, 64, 37, cap - S]
    g = torch.Generator().manual_seed(S)
    first, k, v = (torch.randn(B, n, Hkv, D, generator=g).bfloat16().cuda() for n in (cap, S, S))
    ops.kv8_write(c, first, -first, 0, counts=torch.tensor(pos, dtype=torch.int32, device="cuda"))
    K8.write(ref, np64(first), np64(-first), [0] * B, pos)
    at = torch.tensor(pos, device="cuda")
    before = [t.clone() for t in c]
    for low in (torch.tensor([-5, -1, -2 ** 31, 0], dtype=torch.int32, device="cuda"),
                torch.tensor([-3], dtype=torch.int32, device="cuda")):
        ops.kv8_write(c, k, v, at, counts=low)
        for t, u in zip(c, before):
            assert torch.equal(t.view(torch.uint8), u.view(torch.uint8))
    ops.kv8_write(c, k, v, at, counts=torch.tensor([1000, S + 1, 2 ** 31 - 1, S + 7], dtype=torch.int32, device="cuda"))
    K8.write(ref, np64(k), np64(v), pos, [S] * B)
    got = to_oracle(c)
    for b in range(B):
        n = pos[b] + S
        for x in ("k", "v"):
            assert np.array_equal(got[x][b, :, :n], ref[x][b, :, :n]), (b, x)
            assert (got[x][b, :, n:] == 13.0).all(), (b, x)
        for x in ("ke", "ve"):
            nb = -(-n // 64)
            assert np.array_equal(got[x][b, :, :nb], ref[x][b, :, :nb]), (b, x)
            assert (got[x][b, :, nb:] == K8.E_MIN).all()


def test_rows_hold_sums_of_large_values(gpu):
    """Values up to n |v| < 2^114, with keys whose weights run up to 2^14 times
    what they count: the first blocks of each wave set its reference, and every
    later score lies 5.9 (log2) above it."""
    from delta_attention import ops
    n, D = 2500, 32
    g = torch.Generator().manual_seed(1)
    k = torch.zeros(1, n, 1, D)
    k[0, 256:, 0, 0] = 4.0
    v = (1 + torch.rand(1, n, 1, D, generator=g) * 0.875) * 2.0 ** 101
    k, v = k.to(torch.bfloat16), v.to(torch.bfloat16)
    assert n * float(v.max()) < 2.0 ** 114
    q = torch.zeros(1, 2, 1, D, dtype=torch.bfloat16)
    q[..., 0] = 1
    scale = 5.9 * float(np.log(2.0)) / 4
    c, ref = ops.kv8_empty(1, 1, n, D), K8.new_cache(1, 1, 2560, D)
    ops.kv8_write(c, k.cuda(), v.cuda(), 0)
    K8.write(ref, np64(k), np64(v), [0])
    kk, vv = K8.values(ref)
    want, spread = K8.rows(np64(q), kk, vv, [n], 0, 0, scale)
    got = np64(ops.kv8_attention(q.cuda(), c, n_keys=n, sm_scale=scale))
    tol = tolerance(want, spread, D, n, torch.bfloat16)
    assert np.isfinite(got).all() and (np.abs(got - want) <= tol).all(), float((np.abs(got - want) / tol).max())


def test_read_results_are_independent(gpu):
    """Changing one result in place leaves the other as autograd saved it, and
    neither keeps the other's memory."""
    from delta_attention import ops
    c = ops.kv8_empty(1, 2, 128, 64)
    x = torch.randn(1, 100, 2, 64, device="cuda").bfloat16()
    ops.kv8_write(c, x, x, 0)
    k, v = ops.kv8_read(c, 0, 100)
    p = torch.rand(1, 2, 3, 100, device="cuda", requires_grad=True)
    y = (p.unsqueeze(-1) * v.float().unsqueeze(2)).sum()
    w = torch.ones_like(v, requires_grad=True)
    z = (w * v).sum()                                   # (saves v itself)
    k.mul_(2)
    (y + z).backward()
    assert torch.equal(w.grad, v) and not k._is_view() and not v._is_view()
    for t in (k, v):
        assert t.untyped_storage().nbytes() == t.numel() * 2
