"""What is measured of sampled generation: the choice of the next tokens, and
the attention of a batch whose sequences share a prompt, each as a user's
program calls it.

  sample   ops.sample_tokens: one token per row of logits [B, V] from a given
           random number in [0, 1) per row. Rows are ordered by logit (largest
           first, equal ones by index) and cut to the first top_k, then to the
           shortest run whose probability reaches top_p, then to the tokens of
           at least min_p times the largest one's probability; the token is the
           one at which the probabilities of the tokens left, summed by index,
           pass the random number. Temperature 0 takes the first in order.
           Returns the tokens and their log-probabilities among the tokens left.
  prefix   ops.prefix_attention: the last s rows of each of B sequences; every
           B / P of them share one of P prefixes, whose keys all rows see, and
           each has keys of its own (row i of n own keys stands at n - s + i
           and sees those up to itself)

Logits are N(0, sigma) with some tokens well above the others, as a language
model's are; queries, keys and values are N(0, 1), so that scores have unit
variance.
"""

from __future__ import annotations

import math
import os
import sys

import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


# ---------------------------------------------------------------------------
# the cases

def listed():
    return [
        # one sequence's decode step, a small vocabulary, temperature alone: latency
        dict(name="sample_one_plain", kind="sample", B=1, V=32000, dtype="fp16", mixed=False,
             temperature=0.8, top_k=0, top_p=1.0, min_p=0.0, masked=0.0),
        # the same of the default model's vocabulary, with a nucleus
        dict(name="sample_one_top_p", kind="sample", B=1, V=128256, dtype="bf16", mixed=False,
             temperature=0.7, top_k=0, top_p=0.9, min_p=0.0, masked=0.0),
        # a few samples of one prompt, logits cast to 32 bits, an odd vocabulary padded with -inf
        dict(name="sample_few_fp32", kind="sample", B=8, V=50021, dtype="fp32", mixed=False,
             temperature=1.0, top_k=50, top_p=0.95, min_p=0.0, masked=0.01),
        # a serving batch, every request with its own settings (greedy ones among them)
        dict(name="sample_batch_mixed", kind="sample", B=64, V=151936, dtype="bf16", mixed=True,
             temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, masked=0.0),
        # many samples, all filters on
        dict(name="sample_wide", kind="sample", B=256, V=128256, dtype="bf16", mixed=False,
             temperature=0.9, top_k=200, top_p=0.9, min_p=0.02, masked=0.0),
        # many samples from nearly flat distributions: few tokens are cut
        dict(name="sample_wide_flat", kind="sample", B=192, V=100003, dtype="fp16", mixed=False,
             temperature=1.5, top_k=0, top_p=0.98, min_p=0.0, masked=0.0),
        # four samples of one short prompt, a few tokens each: a decode step's layer, latency
        dict(name="prefix_short", kind="prefix", P=1, n=4, Hkv=8, G=4, D=128, Np=2711, dev=False,
             cap=256, lo=37, hi=37, s=1, dtype="bf16"),
        # sixteen samples of a long document
        dict(name="prefix_128k", kind="prefix", P=1, n=16, Hkv=8, G=4, D=128, Np=131072, dev=False,
             cap=1024, lo=513, hi=1000, s=1, dtype="bf16"),
        # three prompts of different lengths, five samples each, very different own lengths
        dict(name="prefix_groups_fp16", kind="prefix", P=3, n=5, Hkv=8, G=5, D=128, Np=20011, dev=True,
             cap=3008, lo=1, hi=3001, s=1, dtype="fp16"),
        # the widest heads, an odd prefix
        dict(name="prefix_d256", kind="prefix", P=1, n=8, Hkv=4, G=2, D=256, Np=40009, dev=False,
             cap=512, lo=200, hi=333, s=1, dtype="bf16"),
        # eight questions of 48 tokens about one document, head_dim 64: several rows a sequence
        dict(name="prefix_questions_d64", kind="prefix", P=1, n=8, Hkv=8, G=4, D=64, Np=30011, dev=False,
             cap=64, lo=48, hi=48, s=48, dtype="bf16"),
        # the largest: 128 samples, so many rows that the products bound it
        dict(name="prefix_many", kind="prefix", P=1, n=128, Hkv=8, G=4, D=128, Np=65536, dev=False,
             cap=512, lo=100, hi=500, s=1, dtype="bf16"),
    ]


def draw(rng):
    def log(a, b):
        return int(round(math.exp(rng.uniform(math.log(a), math.log(max(a, b))))))

    if rng.random() < 0.5:
        V = log(100, 200000)
        B = log(1, min(256, 256 * 128256 // V))
        mixed = rng.random() < 0.3
        return dict(kind="sample", B=B, V=V, dtype=rng.choice(["bf16", "fp16", "fp32"]), mixed=mixed,
                    temperature=1.0 if mixed else rng.choice([0.0, 0.3, 0.7, 1.0, 1.5]),
                    top_k=0 if mixed else rng.choice([0, 0, 1, log(2, 2000)]),
                    top_p=1.0 if mixed else rng.choice([1.0, 0.5, 0.9, 0.95, 0.99]),
                    min_p=0.0 if mixed else rng.choice([0.0, 0.0, 0.02, 0.1]),
                    masked=rng.choice([0.0, 0.0, 0.01, 0.5]))
    D, Hkv, G = rng.choice([32, 64, 128, 128, 256]), rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 4, 5, 8])
    P, n, s = rng.choice([1, 1, 2, 3]), log(1, 64), rng.choice([1, 1, 1, log(2, 40)])
    by_bytes = 8 * 131072 * 128 // (P * Hkv * D)
    by_flops = 8 * 512 * 65536 * 128 // (P * Hkv * n * G * s * D)
    Np = log(1, min(by_bytes, by_flops, 150000))
    hi = log(s, max(s, min(3000, 8 * 131072 * 128 // 4 // (P * n * Hkv * D))))
    return dict(kind="prefix", P=P, n=n, Hkv=Hkv, G=G, D=D, Np=Np, dev=rng.random() < 0.4,
                cap=hi + rng.choice([0, rng.randint(0, 300)]), lo=rng.choice([hi, min(1, hi)]), hi=hi, s=s,
                dtype=rng.choice(["bf16", "fp16"]))


def _own_lengths(case):
    """Own keys of each sequence, from `hi` down to `lo` in even steps."""
    B, lo, hi = case["P"] * case["n"], case["lo"], case["hi"]
    return [hi - (hi - lo) * b // max(B - 1, 1) for b in range(B)]


def _prefix_lengths(case):
    """Keys of each prefix: Np, or (held on the device) Np less a fifth for each further one."""
    Np = case["Np"]
    return [max(Np - p * (Np // 5), 1) if case["dev"] else Np for p in range(case["P"])]


def work(case):
    if case["kind"] == "sample":
        e = 4 if case["dtype"] == "fp32" else 2
        return {"bytes": case["B"] * (case["V"] * e + 4 + 12), "flops": 0}
    Hkv, G, D, s, n = case["Hkv"], case["G"], case["D"], case["s"], case["n"]
    own_n, pre_n = _own_lengths(case), _prefix_lengths(case)
    keys = sum(own_n) + sum(pre_n)
    pairs = n * s * sum(pre_n) + sum(max(x - s + i + 1, 0) for x in own_n for i in range(s))
    rows = case["P"] * n * s * Hkv * G
    return {"bytes": Hkv * keys * D * 4 + rows * D * 4, "flops": 4 * Hkv * G * D * pairs}


# ---------------------------------------------------------------------------
# inputs

def _logits(B, V, dtype, masked, g):
    x = torch.randn(B, V, device="cuda", generator=g)
    x *= 1.5 + torch.rand(B, 1, device="cuda", generator=g)
    few = torch.rand(B, V, device="cuda", generator=g) < max(1 / 2000, 2 / V)
    x += few * (4 + 6 * torch.rand(B, V, device="cuda", generator=g))
    if masked:
        x[:, V - max(int(V * masked), 1):] = -math.inf
        x[:, 0] = 0.0
    return x.to(dtype)


def _choice(values, B, dtype, g):
    v = torch.tensor(values, dtype=dtype, device="cuda")
    return v[torch.randint(0, len(values), (B,), device="cuda", generator=g)]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed) * 7919 + 29)
    dtype = DTYPES[case["dtype"]]
    if case["kind"] == "sample":
        B = case["B"]
        st = dict(case=dict(case), logits=_logits(B, case["V"], dtype, case["masked"], g),
                  u=torch.rand(B, device="cuda", generator=g))
        if case["mixed"]:
            st.update(temperature=_choice([0.0, 0.3, 0.7, 1.0, 1.3], B, torch.float32, g),
                      top_k=_choice([0, 0, 1, 20, 50, 1000], B, torch.int32, g),
                      top_p=_choice([0.5, 0.8, 0.9, 0.95, 1.0], B, torch.float32, g),
                      min_p=_choice([0.0, 0.0, 0.02, 0.1], B, torch.float32, g))
        else:
            st.update({x: case[x] for x in ("temperature", "top_k", "top_p", "min_p")})
        return st
    P, n, Hkv, G, D, s = (case[x] for x in ("P", "n", "Hkv", "G", "D", "s"))

    def tensor(*shape):
        x = torch.empty(*shape, device="cuda", dtype=dtype)
        for part in x:
            part.copy_(torch.randn(*shape[1:], device="cuda", generator=g))
        return x.transpose(1, 2)      # [b, heads, tokens, D] views of the projections' layout

    st = dict(case=dict(case), q=tensor(P * n, s, Hkv * G, D),
              k_prefix=tensor(P, case["Np"], Hkv, D), v_prefix=tensor(P, case["Np"], Hkv, D),
              k=tensor(P * n, case["cap"], Hkv, D), v=tensor(P * n, case["cap"], Hkv, D),
              n_keys=torch.tensor(_own_lengths(case), dtype=torch.int32, device="cuda"))
    st["n_prefix"] = (torch.tensor(_prefix_lengths(case), dtype=torch.int32, device="cuda") if case["dev"]
                      else case["Np"])
    return st


# ---------------------------------------------------------------------------
# one pass

def run(st):
    sample = st["case"]["kind"] == "sample"
    if own:
        return (_own_sample if sample else _own_prefix)(st)
    return (_sample if sample else _prefix)(st)


def _ops():
    pkg = os.path.join(os.getcwd(), "delta-attention_amd")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    from delta_attention import ops
    return ops


def _own_sample(st):
    return _ops().sample_tokens(st["logits"], st["u"], temperature=st["temperature"], top_k=st["top_k"],
                                top_p=st["top_p"], min_p=st["min_p"])


def _own_prefix(st):
    return _ops().prefix_attention(st["q"], st["k_prefix"], st["v_prefix"], st["k"], st["v"],
                                   n_prefix=st["n_prefix"], n_keys=st["n_keys"],
                                   sm_scale=st["case"]["D"] ** -0.5)


def _column(x, like):
    """A setting (a number, or one per row) as a 64-bit column, rounded to 32 bits first."""
    if not isinstance(x, torch.Tensor):
        x = torch.full((1,), x, device=like.device, dtype=torch.float32)
    return x.double()[:, None]


def _sample(st):
    # in 64 bits: a border of the cumulative sums must not move past the random number
    x = st["logits"].double()
    B, V = x.shape
    T, k, p, m = (_column(st[c], x) for c in ("temperature", "top_k", "top_p", "min_p"))
    greedy = T <= 0
    T = torch.where(greedy, torch.ones_like(T), T)
    xs, order = torch.sort(x, dim=-1, descending=True, stable=True)
    top = xs[:, :1]
    rank = torch.arange(V, device=x.device)
    ws = torch.exp((xs - top) / T)
    keep = (k <= 0) | (rank < k)
    cut = torch.where(keep, ws, torch.zeros_like(ws))
    upto = cut.cumsum(-1)
    before = upto - cut
    keep = keep & ((p >= 1) | (before < p * upto[:, -1:]))
    keep = keep & (xs >= top + T * torch.log(m))
    keep |= rank == 0
    kept = torch.zeros_like(ws).scatter_(1, order, torch.where(keep, ws, torch.zeros_like(ws)))
    upto = kept.cumsum(-1)
    total = upto[:, -1:]
    token = (upto <= st["u"].double()[:, None] * total).sum(-1, keepdim=True).clamp(max=V - 1)
    token = torch.where(greedy, order[:, :1], token)
    logp = (x.gather(1, token) - top) / T - torch.log(total)
    logp = torch.where(greedy, torch.zeros_like(logp), logp)
    return token[:, 0], logp[:, 0].float()


def _prefix(st):
    case = st["case"]
    P, n, Hkv, G, D, s = (case[x] for x in ("P", "n", "Hkv", "G", "D", "s"))
    B, Np, cap, dev = P * n, case["Np"], case["cap"], st["q"].device
    q = st["q"].float().view(P, n, Hkv, G, s, D).transpose(1, 2)              # [P, Hkv, n, G, s, D]
    x = torch.matmul(q.reshape(P, Hkv, n * G * s, D), st["k_prefix"].float().transpose(-1, -2))
    x = x.view(P, Hkv, n, G * s, Np).mul_(D ** -0.5)
    if case["dev"]:
        past = torch.arange(Np, device=dev) >= st["n_prefix"].view(P, 1, 1, 1, 1)
        x = x.masked_fill_(past, -math.inf)
    qo = q.transpose(1, 2).reshape(B, Hkv, G * s, D)
    y = torch.matmul(qo, st["k"].float().transpose(-1, -2)).view(B, Hkv, G, s, cap) * D ** -0.5
    at = st["n_keys"].view(B, 1, 1, 1, 1) - s + torch.arange(s, device=dev).view(s, 1)
    y = y.masked_fill_(torch.arange(cap, device=dev) > at, -math.inf)
    y = y.view(P, n, Hkv, G * s, cap).transpose(1, 2)                         # [P, Hkv, n, G s, cap]
    top = torch.maximum(x.amax(-1, keepdim=True), y.amax(-1, keepdim=True))
    top = torch.where(top == -math.inf, torch.zeros_like(top), top)
    x = x.sub_(top).exp_()
    y = torch.exp(y - top)
    total = x.sum(-1, keepdim=True) + y.sum(-1, keepdim=True)
    o = torch.matmul(x.view(P, Hkv, n * G * s, Np), st["v_prefix"].float()).view(P, Hkv, n, G * s, D)
    yo = y.transpose(1, 2).reshape(B, Hkv, G * s, cap)
    o = o + torch.matmul(yo, st["v"].float()).view(P, n, Hkv, G * s, D).transpose(1, 2)
    o = o / torch.where(total > 0, total, torch.ones_like(total))
    return o.transpose(1, 2).reshape(B, Hkv * G, s, D).to(st["q"].dtype)


# ---------------------------------------------------------------------------
# the definitions in 64 bits

def _exact_sample(st):
    x = st["logits"].float().cpu().numpy().astype(np.float64)
    u = st["u"].cpu().numpy().astype(np.float64)
    B, V = x.shape

    def entry(c, b):
        v = st[c]
        return float(v[b]) if isinstance(v, torch.Tensor) else float(np.float32(v))

    tokens, logs = [], []
    for b in range(B):
        T, k, p, m = (entry(c, b) for c in ("temperature", "top_k", "top_p", "min_p"))
        order = np.argsort(-x[b], kind="stable")
        first = int(order[0])
        if T <= 0:
            tokens.append(first)
            logs.append(0.0)
            continue
        if k > 0:
            order = order[:int(k)]
        d = (x[b, order] - x[b, first]) / T
        w = np.exp(d)
        if p < 1:
            sums = np.concatenate([[0.0], np.cumsum(w)])
            order = order[:max(int(np.searchsorted(sums[:-1], p * sums[-1], side="left")), 1)]
        if m > 0:
            order = order[:max(int((x[b, order] >= x[b, first] + T * math.log(m)).sum()), 1)]
        order = np.sort(order)
        w = np.exp((x[b, order] - x[b, first]) / T)
        sums = np.cumsum(w)
        at = min(int(np.searchsorted(sums, u[b] * sums[-1], side="right")), len(order) - 1)
        tokens.append(int(order[at]))
        logs.append((x[b, order[at]] - x[b, first]) / T - math.log(math.fsum(w)))
    return torch.tensor(tokens), torch.tensor(logs, dtype=torch.float64)


def _exact_prefix(st):
    case = st["case"]
    P, n, Hkv, G, D, s = (case[x] for x in ("P", "n", "Hkv", "G", "D", "s"))
    pre, mine = _prefix_lengths(case), _own_lengths(case)
    out = torch.zeros(P * n, Hkv * G, s, D, dtype=torch.float64, device="cuda")
    at = torch.arange(s, device="cuda")[:, None]
    for p in range(P):
        for h in range(Hkv):
            kp = st["k_prefix"][p, h, :pre[p]].double()
            vp = st["v_prefix"][p, h, :pre[p]].double()
            for b in range(p * n, (p + 1) * n):
                N = mine[b]
                key = torch.cat([kp, st["k"][b, h, :N].double()])
                value = torch.cat([vp, st["v"][b, h, :N].double()])
                place = torch.arange(key.shape[0], device="cuda") - pre[p]
                hidden = (place >= 0) & (place > N - s + at)                                 # [s, keys]
                scores = st["q"][b, h * G:(h + 1) * G].double().reshape(G * s, D) @ key.T * D ** -0.5
                scores.view(G, s, -1).masked_fill_(hidden, -math.inf)
                out[b, h * G:(h + 1) * G] = (torch.softmax(scores, -1) @ value).view(G, s, D)
    return out


def exact(case, seed):
    st = prepare(case, seed)
    return _exact_sample(st) if case["kind"] == "sample" else _exact_prefix(st)
