"""Sampled generation: ops.sample_tokens and ops.prefix_attention together, as
LlamaForCausalLM.generate_sampled / generate and the text wrapper use them."""

import types

import numpy as np
import pytest
import torch

from helpers import write_checkpoint
from oracle import sample_oracle as S

pytestmark = pytest.mark.gpu


def _small_model(dtype=torch.bfloat16, **kw):
    from delta_attention.model import LlamaConfig, random_llama
    cfg = dict(vocab_size=512, hidden_size=2048, intermediate_size=4096, num_hidden_layers=2,
               num_attention_heads=16, num_key_value_heads=4, head_dim=128, delta_lambda=64, sliding_window=256,
               sink_tokens=16, initializer_range=0.05)
    return random_llama(LlamaConfig(**{**cfg, **kw}), "cuda", dtype, seed=7)


def _ids(s, seed, b=1, vocab=512):
    return torch.randint(0, vocab, (b, s), device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed))


def _u(rows, n, seed):
    return torch.rand(rows, n, device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed))


def _drawn(tokens, logits, u, **settings):
    """Every token is the oracle's draw from its step's logits."""
    for j, lg in enumerate(logits):
        x = lg.cpu().numpy()
        for b in range(x.shape[0]):
            want, _, margin = S.sample(x[b], float(u[b, j]), **settings)
            if margin > 2.0 ** -28:
                assert int(tokens[b, j]) == want, (j, b, margin)


@pytest.mark.parametrize("graph", [False, True])
@pytest.mark.parametrize("b,samples", [(1, 1), (1, 5), (2, 3)])
def test_tokens_are_drawn_from_each_steps_logits(gpu, b, samples, graph):
    m = _small_model()
    n, settings = 12, dict(temperature=float(np.float32(0.8)), top_k=40, top_p=float(np.float32(0.9)))
    ids, u = _ids(700, 1, b), _u(b * samples, n, 2)
    lg, lp = [], []
    toks = m.generate_sampled(ids, n, u, samples=samples, graph=graph, logits_out=lg, logprobs_out=lp, **settings)
    assert toks.shape == (b * samples, n) and len(lg) == len(lp) == n
    _drawn(toks, lg, u, **settings)
    for x, y, t in zip(lg, lp, toks.t()):
        assert y.shape == (b * samples,) and (y <= 0).all()
    # the prompts' own pass: every sample of one prompt starts from the same logits
    for p in range(b):
        assert all(torch.equal(lg[0][p * samples], lg[0][p * samples + i]) for i in range(samples))
    again = m.generate_sampled(ids, n, u, samples=samples, graph=graph, **settings)
    assert torch.equal(again, toks)


@pytest.mark.parametrize("samples", [1, 4])
def test_recorded_steps_repeat_the_static_ones(gpu, samples):
    m = _small_model()
    ids, u = _ids(600, 3, 2), _u(2 * samples, 10, 4)
    a, b, c = [], [], []
    t0 = m.generate_sampled(ids, 10, u, samples=samples, top_p=0.95, graph=True, logits_out=a)
    t1 = m.generate_sampled(ids, 10, u, samples=samples, top_p=0.95, graph=True, record=False, logits_out=b)
    t2 = m.generate_sampled(ids, 10, u, samples=samples, top_p=0.95, logits_out=c)
    assert torch.equal(t0, t1) and all(torch.equal(x, y) for x, y in zip(a, b))
    same = int((t0 == t2).all(0).long().cumprod(0).sum())
    assert same >= 1
    for i in range(same):
        assert (a[i] - c[i]).abs().max().item() <= 2e-2 * max(1.0, c[i].abs().max().item()), i


@pytest.mark.parametrize("kv", ["model", "fp8"])
def test_samples_are_the_sequences_that_one_at_a_time_gives(gpu, kv):
    """Sample i of a prompt has, up to rounding, the logits of the same sequence
    generated by itself (its tokens forced), with the prompt's keys shared or
    (8-bit) copied."""
    m = _small_model(kv_cache=kv)
    samples, n = 4, 8
    ids, u = _ids(500, 5), _u(samples, n, 6)
    lg = []
    toks = m.generate_sampled(ids, n, u, samples=samples, temperature=1.2, logits_out=lg)
    assert len({tuple(t) for t in toks.tolist()}) > 1
    for i in range(samples):
        one = []
        alone = m.generate_sampled(ids, n, u[i:i + 1], temperature=1.2, logits_out=one)
        same = int((alone[0] == toks[i]).long().cumprod(0).sum())
        assert same >= 1
        for j in range(same + (same < n)):       # (the step that differs still has the same past)
            d = (one[j][0] - lg[j][i]).abs().max().item()
            assert d <= 2e-2 * max(1.0, one[j].abs().max().item()), (i, j, d)


def test_temperature_zero_is_greedy(gpu):
    m = _small_model()
    ids = _ids(400, 8, 2)
    greedy = m.generate_greedy(ids, 9)
    assert torch.equal(m.generate_sampled(ids, 9, _u(2, 9, 9), temperature=0.0), greedy)
    several = m.generate_sampled(ids, 9, _u(6, 9, 9), temperature=0.0, samples=3)
    assert torch.equal(several[0::3], several[1::3]) and torch.equal(several[0::3], several[2::3])
    assert torch.equal(several[0::3, 0], greedy[:, 0])       # the prompts' pass


def test_settings_of_the_sequences(gpu):
    """Device settings, one entry per sequence: the greedy ones among them
    follow the argmax of their own logits."""
    m = _small_model()
    ids, u = _ids(300, 10), _u(4, 7, 11)
    T = torch.tensor([0.0, 0.7, 0.0, 1.5], device="cuda")
    K = torch.tensor([0, 5, 9, 0], dtype=torch.int32, device="cuda")
    lg = []
    toks = m.generate_sampled(ids, 7, u, samples=4, temperature=T, top_k=K, graph=True, logits_out=lg)
    for j, x in enumerate(lg):
        assert torch.equal(toks[[0, 2], j], x[[0, 2]].argmax(-1))
        assert (x[1].topk(5).indices == toks[1, j]).any()


def test_generate(gpu):
    m = _small_model()
    ids = _ids(260, 12, 2)

    def draw(**kw):
        g = torch.Generator(device="cuda").manual_seed(5)
        return m.generate(ids, max_new_tokens=6, do_sample=True, generator=g, **kw)

    out = draw(num_return_sequences=3, temperature=1.1, top_p=0.9)
    assert out.shape == (6, 266) and torch.equal(out[:, :260], ids.repeat_interleave(3, 0))
    assert torch.equal(out, draw(num_return_sequences=3, temperature=1.1, top_p=0.9))
    u = torch.rand(6, 6, device="cuda", generator=torch.Generator(device="cuda").manual_seed(5))
    want = m.generate_sampled(ids, 6, u, samples=3, temperature=1.1, top_k=50, top_p=0.9)
    assert torch.equal(out[:, 260:], want)
    # left-padded rows: each over its real tokens, with its own numbers
    mask = torch.ones_like(ids)
    mask[1, :100] = 0
    padded = m.generate(ids, attention_mask=mask, max_new_tokens=6, do_sample=True, num_return_sequences=2,
                        generator=torch.Generator(device="cuda").manual_seed(6))
    u = torch.rand(4, 6, device="cuda", generator=torch.Generator(device="cuda").manual_seed(6))
    assert torch.equal(padded[:2, 260:], m.generate_sampled(ids[:1], 6, u[:2], samples=2, top_k=50))
    assert torch.equal(padded[2:, 260:], m.generate_sampled(ids[1:, 100:], 6, u[2:], samples=2, top_k=50))
    # an eos token ends a sequence, the others go on
    eos = int(out[0, 262])
    cut = draw(num_return_sequences=3, temperature=1.1, top_p=0.9, eos_token_id=eos, pad_token_id=511)
    for a, b in zip(cut, out):
        t = b[260:].tolist()
        end = t.index(eos) + 1 if eos in t else 6
        assert a[260:260 + end].tolist() == t[:end] and (a[260 + end:] == 511).all()
    with pytest.raises(NotImplementedError, match="generator"):
        m.generate(ids, max_new_tokens=2, do_sample=True)
    with pytest.raises(ValueError, match="num_return_sequences"):
        draw(num_return_sequences=0)
    for bad in (_u(5, 6, 1), _u(6, 5, 1), _u(6, 6, 1).double()):
        with pytest.raises(AssertionError, match="u: float32"):
            m.generate_sampled(ids, 6, bad, samples=3)
    m.config.decode_mode = "delta"
    with pytest.raises(NotImplementedError, match="dense decode"):
        m.generate_sampled(ids[:1], 6, _u(2, 6, 1), samples=2)
    m.config.decode_mode = "dense"


def test_the_sparse_decodes_take_sampled_tokens(gpu):
    m = _small_model(decode_mode="delta", gamma_dec=3)
    ids, u = _ids(700, 13), _u(1, 9, 14)
    lg = []
    toks = m.generate_sampled(ids, 9, u, top_k=20, graph=True, logits_out=lg)
    _drawn(toks, lg, u, top_k=20)


def test_wrapper_returns_every_sample(gpu, tmp_path):
    from delta_attention.config import Config
    from delta_attention.model_wrapper import HuggingFaceModel
    write_checkpoint(tmp_path, seed=3)
    w = HuggingFaceModel(Config(model_str=str(tmp_path), delta_lambda=16, sliding_window=128, sink_tokens=16),
                         max_new_tokens=5)
    prompts = [" ".join(f"w{2 + (7 * i + j) % 60}" for j in range(n)) for i, n in enumerate((300, 280))]

    def draw():
        return w.process_batch(prompts, do_sample=True, num_return_sequences=3, temperature=1.5, top_k=0,
                               generator=torch.Generator(device="cuda").manual_seed(1))

    res = draw()
    assert [len(r["text"]) for r in res] == [3, 3] and res == draw()
    assert len(set(res[0]["text"] + res[1]["text"])) > 1
    assert all(len(t.split()) <= 5 for r in res for t in r["text"])


def test_cache_contents(gpu):
    """The shared cache: the prompt's buffers as the prefill wrote them, each
    sequence's own tokens in its rows, by eager, static and several-token
    passes; the delta prefill on it is refused."""
    from delta_attention.model import KVCache
    m = _small_model()
    cfg = m.config
    ids, more = _ids(200, 15, 2), _ids(9, 16, 6)
    with torch.inference_mode():
        base = KVCache(cfg, 2, 200, "cuda", torch.bfloat16)
        m.model(ids, None, base)
        cache = base.for_samples(cfg, 3, 9)
        kept = [k.clone() for k in base.k]
        cfg._attn_implementation = "sdpa_rectangle"
        flat = KVCache(cfg, 6, 209, "cuda", torch.bfloat16)
        for i in range(cfg.num_hidden_layers):
            flat.k[i][:, :200] = base.k[i].repeat_interleave(3, 0)
            flat.v[i][:, :200] = base.v[i].repeat_interleave(3, 0)
        flat.len = list(base.len)
        outs = []
        for c in (cache, flat):
            h = [m.model(more[:, :4], None, c), m.model(more[:, 4:5], None, c)]      # four tokens, one
            c.start_static()
            for j in (5, 6):                                                         # static ones
                h.append(m.model(more[:, j:j + 1], None, c))
                c.advance_static()
            c.stop_static(2)
            h.append(m.model(more[:, 7:], None, c))
            assert c.seq_len() == 209
            outs.append(torch.cat(h, 1).float())
        cfg._attn_implementation = "window"
        assert all(torch.equal(a, b) for a, b in zip(base.k, kept))
        assert (outs[0] - outs[1]).abs().max().item() <= 2e-2 * outs[1].abs().max().item()
        # (layer 0's keys are the projections': the same bits; below, what the layers' roundings leave)
        assert torch.equal(cache.k[0], flat.k[0][:, 200:]) and torch.equal(cache.v[0], flat.v[0][:, 200:])
        d = (cache.k[1].float() - flat.k[1][:, 200:].float()).abs().max().item()
        assert d <= 3e-2 * flat.k[1].float().abs().max().item(), d
        with pytest.raises(NotImplementedError, match="whole prompt"):
            m.model(more[:, :1], None, cache)
        with pytest.raises(AssertionError):
            cfg._attn_implementation = "sdpa_rectangle"
            m.model(more[:, :1], None, cache)    # the cache is full
    cfg._attn_implementation = "window"


def test_float32_layer(gpu):
    """float32 models attend in bf16 over a shared cache too."""
    from delta_attention import ops
    from delta_attention.llama import LlamaAttention, SharedKeys
    cfg = types.SimpleNamespace(hidden_size=256, num_attention_heads=4, num_key_value_heads=2, head_dim=64,
                                attention_bias=False, attention_dropout=0.0, rms_norm_eps=1e-6,
                                _attn_implementation="sdpa_rectangle", decode_mode="dense")
    m = LlamaAttention(cfg, 0).cuda()
    g = torch.Generator().manual_seed(17)
    q, kp, vp, k, v = (torch.randn(*s, generator=g).cuda() for s in ((4, 4, 2, 64), (2, 2, 90, 64), (2, 2, 90, 64),
                                                                     (4, 2, 20, 64), (4, 2, 20, 64)))
    out, _ = m.sdpa_rectangle_forward(m, q, SharedKeys(kp, vp, k, v, 13), None, scaling=0.125)
    assert out.dtype == torch.float32
    h = [t.to(torch.bfloat16) for t in (q, kp, vp, k, v)]
    want = ops.prefix_attention(*h, n_keys=13, sm_scale=0.125)
    assert torch.equal(out, want.transpose(1, 2).float())
