"""GPU parity of ops.sample_tokens with the float64 oracle: the same token where
no border of the oracle's sums is next to what it is compared with, and its
log-probability.

The kernel's weights are integers in units of 2^-bits of the largest (bits = 45
up to 2^17 tokens), each off by half a unit and 2^-50 of itself: a sum over a
row is off by V * 2^-(bits + 1) + 2^-50 of it at most, which is 2^-29 for 2^17
tokens if every error has one sign. Tokens are compared where the oracle's
margin is above four times that (one sum's and one total's error, in each of a
filter's and the draw's comparison); log-probabilities are off by twice it and
float32's rounding."""

import math

import numpy as np
import pytest
import torch

from oracle import sample_oracle as S

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def off(V):
    bits = min(45, 62 - max(V - 1, 0).bit_length())
    return V * 2.0 ** -(bits + 1) + 2.0 ** -50


def logits(B, V, dtype, seed, sigma=2.5):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(B, V, generator=g) * sigma
    x += (torch.rand(B, V, generator=g) < max(1 / 2000, 2 / V)) * (4 + 6 * torch.rand(B, V, generator=g))
    return x.to(DT[dtype]).cuda()


def uniform(B, seed):
    return torch.rand(B, generator=torch.Generator().manual_seed(seed)).cuda()


def check(x, u, got=None, sure=True, **settings):
    """sure: every row's margin is wide enough (else such rows are passed over)."""
    from delta_attention import ops
    tok, lp = got if got is not None else ops.sample_tokens(x, u, **settings)
    assert tok.dtype == torch.int64 and lp.dtype == torch.float32 and tok.shape == lp.shape == (x.shape[0],)
    X, U, tok, lp = x.float().cpu().numpy(), u.cpu().numpy(), tok.cpu().numpy(), lp.double().cpu().numpy()
    V, compared = X.shape[1], 0

    def entry(v, b):
        return v[b if v.numel() > 1 else 0].item() if isinstance(v, torch.Tensor) else (
            v if isinstance(v, int) else float(np.float32(v)))

    for b in range(len(X)):
        s = {k: entry(v, b) for k, v in settings.items()}
        want, wlp, margin = S.sample(X[b], U[b], **s)
        if margin <= 4 * off(V):
            assert not sure, (b, margin, s)
            continue
        compared += 1
        assert tok[b] == want, (b, int(tok[b]), want, margin, s)
        if math.isnan(wlp):
            assert math.isnan(lp[b])
        else:
            assert abs(lp[b] - wlp) <= abs(wlp) * 2.0 ** -24 * 1.001 + 2 * off(V), (b, lp[b], wlp)
    return compared


SETTINGS = [dict(), dict(temperature=0.7, top_p=0.9), dict(top_k=50), dict(top_k=50, top_p=0.8, min_p=0.05),
            dict(temperature=1.7, min_p=0.1), dict(temperature=0.3, top_k=1000, top_p=0.99), dict(temperature=0.0),
            dict(top_k=1), dict(top_p=0.0), dict(min_p=1.0), dict(temperature=8.0, top_p=0.999)]


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("V", [1, 2, 63, 64, 65, 513, 2047, 2049, 8191, 50021])
def test_rows_of_every_length(gpu, V, dtype):
    B = 7
    x, u = logits(B, V, dtype, V), uniform(B, V + 1)
    for s in SETTINGS:
        check(x, u, sure=V < 60000 and s.get("temperature", 1) < 8, **s)


@pytest.mark.parametrize("B,V,dtype,s", [
    (1, 128256, "bf16", dict(temperature=0.7, top_p=0.9)), (2, 131072, "fp16", dict(top_p=0.98)),
    (1, 131073, "fp32", dict()), (3, 151936, "bf16", dict(top_k=5000, top_p=0.95)),
    (300, 1000, "bf16", dict(temperature=0.8, top_k=40, min_p=0.02)), (1, 1 << 20, "fp16", dict(top_p=0.9)),
    (40, 32000, "fp32", dict(temperature=1.2, top_p=0.9, min_p=0.001)),
    (160, 20011, "bf16", dict(top_k=50, top_p=0.9)), (161, 9999, "fp32", dict(temperature=1.4, top_p=0.97)),
    (200, 12345, "fp16", dict(temperature=0.6)), (170, 30000, "bf16", dict(min_p=0.03)),
    (165, 9000, "fp16", dict(top_k=4000, top_p=0.9)), (159, 9000, "fp16", dict(top_k=4000, top_p=0.9)),
])
def test_long_rows_and_wide_batches(gpu, B, V, dtype, s):
    x, u = logits(B, V, dtype, V + B), uniform(B, V)
    compared = check(x, u, sure=False, **s)
    assert compared >= 0.9 * B, compared


def test_settings_of_the_rows(gpu):
    from delta_attention import ops
    B, V = 96, 4999
    g = torch.Generator().manual_seed(3)

    def choice(vals, dtype):
        return torch.tensor(vals, dtype=dtype)[torch.randint(0, len(vals), (B,), generator=g)].cuda()

    x, u = logits(B, V, "bf16", 4), uniform(B, 5)
    s = dict(temperature=choice([0.0, -1.0, math.nan, 0.3, 1.0, 2.0], torch.float32),
             top_k=choice([-5, 0, 1, 7, 300, 4998, 4999, 2 ** 31 - 1], torch.int32),
             top_p=choice([-1.0, 0.0, 0.5, 0.9, 1.0, 2.0], torch.float32),
             min_p=choice([-1.0, 0.0, 0.05, 1.0, 3.0], torch.float32))
    check(x, u, **s)
    # one entry for all, and beside settings of the host's
    one = dict(temperature=torch.tensor([0.8]).cuda(), top_k=torch.tensor([30], dtype=torch.int32).cuda(), top_p=0.9)
    check(x, u, **one)
    a = ops.sample_tokens(x, u, **one)
    b = ops.sample_tokens(x, u, temperature=0.8, top_k=30, top_p=0.9)
    assert all(torch.equal(p, q) for p, q in zip(a, b))
    # no number as top_p: off; as min_p: off
    nan = torch.full((1,), math.nan).cuda()
    a, b = ops.sample_tokens(x, u, top_p=nan, min_p=nan), ops.sample_tokens(x, u)
    assert all(torch.equal(p, q) for p, q in zip(a, b))
    # an infinite temperature weighs every candidate alike
    inf = torch.full((1,), math.inf).cuda()
    t, lp = ops.sample_tokens(x[:, :4096], u, temperature=inf)
    assert torch.equal(t, (u.double() * 4096).floor().long())
    assert (lp + math.log(4096)).abs().max().item() <= math.log(4096) * 2.0 ** -24 * 1.001


def test_rows_that_a_mask_leaves_little_of(gpu):
    from delta_attention import ops
    V, inf, nan = 3001, math.inf, math.nan
    for dtype in ("bf16", "fp16", "fp32"):
        low = torch.finfo(DT[dtype]).min
        x = logits(9, V, dtype, 6)
        x[0] = -inf
        x[1] = nan
        x[2] = -inf
        x[2, 2999] = -5.0                        # one candidate
        x[3, :3000] = low                        # the type's lowest value is a candidate
        x[4] = low
        x[5, 7] = inf
        x[5, 100] = inf
        x[6, ::2] = nan
        x[7, 1:] = -inf
        x[7, 0] = low
        x[8] = inf
        u = torch.tensor([0.3, 0.4, 0.9, 0.99, 0.5, 0.7, 0.2, 0.6, 0.25], device="cuda")
        for s in (dict(), dict(top_k=5), dict(top_p=0.7), dict(top_k=3, top_p=0.9, min_p=0.5), dict(temperature=0.0)):
            check(x, u, sure=False, **s)
            t, lp = ops.sample_tokens(x, u, **s)
            assert t[:2].tolist() == [0, 0] and torch.isnan(lp[:2]).all()
            assert t[2].item() == 2999 and t[3].item() == 3000 and t[7].item() == 0
            assert t[5].item() in (7, 100) and not torch.isnan(lp[2:]).any()
        t, lp = ops.sample_tokens(x, u)
        assert t[4].item() == int(0.5 * V) and t[5].item() == 100
        assert t[8].item() == int(0.25 * V)


def test_equal_logits_are_taken_by_index(gpu):
    from delta_attention import ops
    V = 4096
    x = torch.zeros(V, V, device="cuda", dtype=torch.bfloat16)
    x[:, ::2] = -0.0                             # (equal to 0)
    u = torch.arange(V, device="cuda").float() / V
    t, _ = ops.sample_tokens(x, u)               # exact borders: the token at which the sum passes u
    assert torch.equal(t, torch.arange(V, device="cuda"))
    t, _ = ops.sample_tokens(x, u, top_k=1024)
    assert torch.equal(t, torch.arange(V, device="cuda") // 4)
    t, _ = ops.sample_tokens(x, u, top_p=0.5)
    assert torch.equal(t, torch.arange(V, device="cuda") // 2)
    t, _ = ops.sample_tokens(x, u, top_k=2048, top_p=0.25, min_p=1.0)
    assert torch.equal(t, torch.arange(V, device="cuda") // 8)
    assert not ops.sample_tokens(x, u, temperature=0.0)[0].any()
    # two levels: the second one's first by index
    x[:, 1000:1010] = 1.0
    t, _ = ops.sample_tokens(x, torch.full_like(u, 0.9999), top_k=13)
    assert (t == 1009).all()
    check(x[:64], uniform(64, 8), sure=False, top_k=13)


@pytest.mark.parametrize("n", [512, 64])
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_long_rows_of_few_values(gpu, dtype, n):
    """More equal logits than a list holds, at the border of top_k, of top_p, of
    both; by index, exactly."""
    from delta_attention import ops
    V = 65536
    x = torch.zeros(1, V, device="cuda", dtype=DT[dtype]).expand(n, V)
    u = (torch.arange(n, device="cuda").float() + 0.5) / n
    at = (torch.arange(n, device="cuda").double() + 0.5) / n
    for kept, s in ((V, dict()), (V, dict(top_k=0, min_p=1.0)), (512, dict(top_k=512)), (16384, dict(top_p=0.25)),
                    (5000, dict(top_k=5000)), (4096, dict(top_k=8192, top_p=0.5)), (300, dict(top_k=600, top_p=0.5))):
        t, lp = ops.sample_tokens(x, u, **s)
        assert torch.equal(t, (at * kept).floor().long()), s
        assert (lp + math.log(kept)).abs().max().item() <= math.log(kept) * 2.0 ** -24 * 1.001 + 2 * off(V)
    # two values, the larger one past the list too
    y = torch.zeros(1, V, device="cuda", dtype=DT[dtype])
    y[:, ::8] = 1.0
    check(y.expand(40, V), uniform(40, 21), sure=False, top_p=0.5)
    check(y.expand(40, V), uniform(40, 22), sure=False, top_k=10000)
    check(y.expand(40, V), uniform(40, 23), sure=False, top_k=10000, top_p=0.9, temperature=0.5)


def test_rows_around_the_list(gpu):
    """Row lengths at which the launches change, and masks that leave fewer
    candidates than top_k or than groups."""
    for V, B in ((3583, 6), (3584, 6), (3585, 6), (4097, 6), (8192, 6), (8193, 6), (9001, 160), (20000, 6)):
        x, u = logits(B, V, "bf16", V), uniform(B, V + 2)
        x[1, 100:] = -math.inf
        x[2, :] = -math.inf
        x[2, V - 1] = 3.0
        x[3, ::2] = math.nan
        x[4, 7:] = torch.finfo(torch.bfloat16).min
        for s in SETTINGS + [dict(top_k=700), dict(top_k=3000, top_p=0.9)]:
            check(x, u, sure=False, **s)


@pytest.mark.parametrize("V", [33, 40000])
def test_the_ends_of_u(gpu, V):
    from delta_attention import ops
    x = logits(1, V, "fp32", 9).expand(8, V)     # (one row, read eight times)
    u = torch.tensor([0.0, 2.0 ** -149, 2.0 ** -24, 1 - 2.0 ** -24, 1.0, 7.0, -3.0, math.nan], device="cuda")
    for s in (dict(), dict(top_k=20), dict(top_p=0.9)):
        t, lp = ops.sample_tokens(x, u, **s)
        kept = sorted(S.order_of(x[0].cpu().numpy())[:20]) if "top_k" in s else None
        if kept:
            assert t[0].item() == kept[0] and t[4].item() == kept[-1]
        assert t[0] == t[1] == t[6] == t[7] and t[4] == t[5]
        assert t[3] <= t[4] and (lp > -math.inf).all() and (lp <= 0).all()
        check(x, u, sure=False, **s)


def test_strides_and_offsets(gpu):
    from delta_attention import ops
    B, V = 5, 777
    for dtype in DT:
        base = logits(B, 2 * V + 3, dtype, 10)
        u = uniform(B, 11)
        for off_ in (0, 1, 3):
            x = base[:, off_:off_ + V]           # rows apart, at any offset
            check(x, u, top_p=0.9)
            assert all(torch.equal(p, q) for p, q in zip(ops.sample_tokens(x, u, top_k=9),
                                                         ops.sample_tokens(x.contiguous(), u, top_k=9)))
        check(base[:, ::2][:, :V], u, top_k=20)  # tokens apart
        check(base.t()[:B * 100:100], uniform(B, 12)) if V * 2 >= B * 100 else None


def test_a_row_does_not_depend_on_its_batch(gpu):
    from delta_attention import ops
    x, u = logits(170, 32000, "bf16", 13), uniform(170, 14)
    for s in (dict(), dict(top_p=0.95), dict(top_k=100, top_p=0.9), dict(top_k=6000), dict(min_p=0.01)):
        t, lp = ops.sample_tokens(x, u, **s)
        again = ops.sample_tokens(x, u, **s)
        assert torch.equal(t, again[0]) and torch.equal(lp, again[1])
        for b in (0, 33, 169):
            one = ops.sample_tokens(x[b:b + 1], u[b:b + 1], **s)
            assert one[0].item() == t[b].item() and one[1].item() == lp[b].item()


def test_frequencies(gpu):
    """Draws over evenly spread numbers have the probabilities' frequencies,
    exactly: u = (i + 1/2) / n meets each token's stretch within one draw."""
    from delta_attention import ops
    n, V = 20000, 300
    x = logits(1, V, "fp32", 15, sigma=1.0)
    u = (torch.arange(n, dtype=torch.float64) + 0.5).div(n).float().cuda()
    t, _ = ops.sample_tokens(x.expand(n, V), u, temperature=1.3)
    p = torch.softmax(x[0].double() / float(np.float32(1.3)), -1).cpu()
    count = torch.bincount(t.cpu(), minlength=V).double()
    # the ends of a stretch each within a draw, and u rounded to float32
    assert (count - n * p).abs().max().item() <= 2 + n * 2.0 ** -24
    assert (t.diff() >= 0).all()


def test_nothing_to_draw(gpu):
    from delta_attention import ops
    t, lp = ops.sample_tokens(torch.empty(0, 50, device="cuda"), torch.empty(0, device="cuda"))
    assert t.shape == lp.shape == (0,)


def test_recorded_and_on_other_streams(gpu):
    from delta_attention import ops
    B, V = 6, 50021
    x, u = logits(B, V, "bf16", 16), uniform(B, 17)
    T, K = torch.full((B,), 0.9, device="cuda"), torch.full((B,), 60, dtype=torch.int32, device="cuda")
    ops.sample_tokens(x, u)
    graphs = []
    for s in (dict(temperature=T, top_k=K, top_p=0.9), dict(temperature=T, top_p=0.9)):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            got = ops.sample_tokens(x, u, **s)
        graphs.append((g, got, s))
    side = torch.cuda.Stream()
    for i in range(5):
        x.copy_(logits(B, V, "bf16", 20 + i))
        u.copy_(uniform(B, 30 + i))
        T.fill_(0.5 + 0.2 * i)
        K.fill_(1 + 400 * i)
        want = [tuple(y.clone() for y in ops.sample_tokens(x, u, **s)) for _, _, s in graphs]
        torch.cuda.synchronize()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            there = ops.sample_tokens(x, u, **graphs[0][2])
        for g, _, _ in graphs:
            g.replay()
        torch.cuda.synchronize()
        for (_, got, s), w in zip(graphs, want):
            assert torch.equal(got[0], w[0]) and torch.equal(got[1], w[1]), (i, s)
            check(x, u, got=got, sure=False, **s)
        assert torch.equal(there[0], want[0][0])


@pytest.mark.parametrize("B,V,dtype", [(5, 50021, "bf16"), (21, 20011, "fp32"), (48, 40000, "fp16"), (70, 34000, "bf16"),
                                       (66, 20000, "fp32"), (161, 33000, "fp16")])
def test_settings_of_long_rows(gpu, B, V, dtype):
    """Rows of one call that end in different ways: greedy ones, lists short and
    long and too long, nuclei, whole rows."""
    g = torch.Generator().manual_seed(B)

    def choice(vals, dtype):
        return torch.tensor(vals, dtype=dtype)[torch.randint(0, len(vals), (B,), generator=g)].cuda()

    x, u = logits(B, V, dtype, 40), uniform(B, 41)
    x[1, 50:] = -math.inf
    x[2] = math.nan
    k = [0, 0, 0, 1, 7, 120, 1000, 1536, 1537, 5000, V - 1, V]
    s = dict(temperature=choice([0.0, 0.3, 0.8, 1.0, 1.5], torch.float32), top_k=choice(k, torch.int32),
             top_p=choice([0.0, 0.5, 0.9, 1.0, 1.0], torch.float32), min_p=choice([0.0, 0.0, 0.05, 1.0, 3.0], torch.float32))
    compared = check(x, u, sure=False, **s)
    assert compared >= 0.9 * B
    # a top_k for all beside temperatures of the rows (greedy ones among them)
    for top_k in (40, 127, 128, 129, 1536, 1537, V):
        check(x, u, sure=False, temperature=s["temperature"], top_k=top_k, top_p=0.9)
    check(x, u, sure=False, temperature=s["temperature"])
    check(x, u, sure=False, temperature=0.0, top_k=5)


@pytest.mark.parametrize("B,V", [(9, 50021), (72, 12000), (162, 40000)])
@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
def test_long_rows_that_a_mask_leaves_little_of(gpu, dtype, B, V):
    inf, nan = math.inf, math.nan
    low = torch.finfo(DT[dtype]).min
    x, u = logits(B, V, dtype, 43), uniform(B, 44)
    x[0] = -inf
    x[1] = nan
    x[2] = -inf
    x[2, V - 3] = -5.0
    x[3, :V - 1] = low
    x[4] = low
    x[5, 7] = inf
    x[5, V - 100] = inf
    x[6, ::2] = nan
    x[7, 1:] = -inf
    x[7, 0] = low
    x[8] = inf
    for s in SETTINGS + [dict(top_p=0.3, temperature=20.0), dict(top_p=0.7, min_p=0.01)]:
        check(x, u, sure=False, **s)


@pytest.mark.parametrize("offset", [0.0, -300.0, 1000.0])
def test_nuclei_of_shifted_and_narrow_rows(gpu, offset):
    """Logits far from zero, or within a few steps of their type: the border's
    bin holds few values, or one, or the first."""
    for dtype, V, B in (("fp32", 30011, 6), ("bf16", 30011, 6), ("fp16", 34001, 80), ("fp32", 20000, 64)):
        for sigma in (1e-3, 0.05, 6.0):
            x = (logits(B, V, dtype, 50, sigma=sigma).float() + offset).to(DT[dtype])
            u = uniform(B, 51)
            for s in (dict(top_p=0.3), dict(top_p=0.97, temperature=0.6), dict(top_p=2.0 ** -30), dict(top_p=1 - 2.0 ** -24),
                      dict(top_p=0.9, min_p=0.2)):
                check(x, u, sure=False, **s)


@pytest.mark.parametrize("B,V", [(5, 20000), (64, 20000), (3, 3000)])
def test_the_ends_of_float32(gpu, B, V):
    """Logits and temperatures near the type's largest and smallest numbers: a
    nucleus's histogram spans more than a float, or less than its smallest step."""
    x, u = logits(B, V, "fp32", 60, sigma=1.0), uniform(B, 61)
    x = x / x.abs().amax(1, keepdim=True)
    for scale, T in ((3.4e38, 1e38), (3.4e38, 3.4e38), (3.4e38, 1e36), (1e-38, 3e-39), (1e-41, 1e-41), (1.0, 1e-45), (1e-30, 1e30)):
        y = (x.double() * scale).float()
        for s in (dict(), dict(top_p=0.6), dict(top_k=300, top_p=0.9), dict(top_p=0.9, min_p=0.3)):
            check(y, u, sure=False, temperature=torch.tensor([T]).cuda(), **s)
        # masked by the type's lowest value
        y[:, ::3] = torch.finfo(torch.float32).min
        for s in (dict(top_p=0.6), dict(top_k=300, top_p=0.9)):
            check(y, u, sure=False, temperature=torch.tensor([T]).cuda(), **s)


def test_calls_at_once(gpu):
    """Calls of two streams beside each other, their parts among each other's."""
    from delta_attention import ops
    sets = [(logits(48, 60000, "bf16", 70), uniform(48, 71)), (logits(70, 40000, "fp32", 72), uniform(70, 73))]
    settings = [dict(top_p=0.9), dict(top_k=700, top_p=0.95), dict(), dict(temperature=1.6, top_p=0.99)]
    want = [[ops.sample_tokens(x, u, **s) for s in settings] for x, u in sets]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    torch.cuda.synchronize()
    for _ in range(6):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i] += [ops.sample_tokens(*sets[i], **s) for s in settings]
    torch.cuda.synchronize()
    for i in (0, 1):
        for j, (t, lp) in enumerate(got[i]):
            w = want[i][j % len(settings)]
            assert torch.equal(t, w[0]) and torch.equal(lp, w[1]), (i, j)
