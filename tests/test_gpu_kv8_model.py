"""The 8-bit cache inside the model stack: LlamaAttention's decode and
rectangle passes over a CachedKeys8 against the float64 oracle, the cache's
steps in generation (host lengths, static, recorded), and generation end to
end with config.kv_cache = "fp8"."""

import types

import numpy as np
import pytest
import torch

from helpers import np64, write_checkpoint
from kv8_helpers import same, to_oracle, tolerance
from oracle import kv8_oracle as K8

pytestmark = pytest.mark.gpu


def _module(**kw):
    from delta_attention.llama import LlamaAttention
    base = dict(hidden_size=1024, num_attention_heads=8, num_key_value_heads=2, head_dim=128,
                attention_bias=False, attention_dropout=0.0, rms_norm_eps=1e-6,
                _attn_implementation="sdpa_rectangle", mode="delta", delta_lambda=64,
                sliding_window=512, sink_tokens=64, stride_policy="fixed", log_drift=False,
                decode_mode="dense", gamma_dec=8, refresh_policy="fixed", drift_threshold=0.95,
                drift_k=2.0, gamma_dec_max=128)
    base.update(kw)
    return LlamaAttention(types.SimpleNamespace(**base), 0).cuda().to(torch.bfloat16)


def _cached(n, cap=1280, seed=0, dtype=torch.bfloat16):
    from delta_attention import ops
    from delta_attention.llama import CachedKeys8
    g = torch.Generator().manual_seed(seed)
    k, v = (torch.randn(1, n, 2, 128, generator=g).to(dtype).cuda() for _ in (0, 1))
    c = ops.kv8_empty(1, 2, cap, 128)
    for t in (c.k, c.v):
        t.view(torch.uint8).fill_(0x7f)        # NaN wherever nothing is written
    ops.kv8_write(c, k, v, 0)
    return CachedKeys8(c, n)


def _expect(q, keys, window, sink):
    kk, vv = K8.values(to_oracle(keys.cache))
    return K8.rows(np64(q), kk, vv, [keys.n_keys], window, sink, 128 ** -0.5)


def _near(out, q, want, spread, n):
    got = np64(out).transpose(0, 2, 1, 3)      # [b, s, h, d] -> [b, h, s, d]
    tol = tolerance(want, spread, 128, n, q.dtype)
    assert (np.abs(got - want) <= tol).all(), float((np.abs(got - want) / tol).max())


@pytest.mark.parametrize("mode,window,sink", [("dense", 0, 0), ("sparse", 512, 64)])
def test_decode_rows(gpu, mode, window, sink):
    m, keys = _module(decode_mode=mode), _cached(1100)
    g = torch.Generator().manual_seed(5)
    q = torch.randn(1, 8, 1, 128, generator=g).to(torch.bfloat16).cuda()
    out, _ = m.sdpa_rectangle_forward(m, q, keys, None, scaling=128 ** -0.5)
    _near(out, q, *_expect(q, keys, window, sink), 1100)


def test_rectangle_rows_and_read_back(gpu):
    """Short passes read the codes, longer ones the read-back: both are the
    rows of the cache's values."""
    from delta_attention.llama import DIRECT_ROWS8
    from helpers import assert_close
    m, keys = _module(), _cached(900)
    g = torch.Generator().manual_seed(6)
    for s in (2, 64, 65, 300):
        q = torch.randn(1, 8, s, 128, generator=g).to(torch.bfloat16).cuda()
        out, _ = m.sdpa_rectangle_forward(m, q, keys, None, scaling=128 ** -0.5)
        want, spread = _expect(q, keys, 0, 0)
        if s * 4 <= DIRECT_ROWS8:
            _near(out, q, want, spread, 900)
        else:                      # (the rows kernel's own bound: its probabilities are bf16)
            assert_close(np64(out).transpose(0, 2, 1, 3), want, what=f"read-back {s}")


@pytest.mark.parametrize("policy,log_drift", [("fixed", False), ("drift", True)])
def test_delta_decode(gpu, policy, log_drift):
    """The delta decode's anchors and corrections on 8-bit rows: dense rows at
    anchors, sparse + last correction between."""
    m, keys = _module(decode_mode="delta", gamma_dec=3, refresh_policy=policy, drift_threshold=-2.0,
                      gamma_dec_max=3, log_drift=log_drift), _cached(1000)
    g = torch.Generator().manual_seed(7)
    last = None
    for step in range(7):
        q = torch.randn(1, 8, 1, 128, generator=g).to(torch.bfloat16).cuda()
        out, _ = m.sdpa_rectangle_forward(m, q, keys, None, scaling=128 ** -0.5)
        dense, ds = _expect(q, keys, 0, 0)
        sparse, ss = _expect(q, keys, 512, 64)
        if m._dec_state["steps"] == 0:
            assert step % 3 == 0
            _near(out, q, dense, ds, 1000)
            last = dense - sparse
        else:
            # four bf16 roundings of values near one: the two rows, the difference, the sum
            got = np64(out).transpose(0, 2, 1, 3)
            big = max(np.abs(dense).max(), np.abs(sparse).max(), np.abs(last).max(), np.abs(sparse + last).max())
            assert np.abs(got - (sparse + last)).max() <= 6 * 2.0 ** -8 * big


def _small_model(**kw):
    from delta_attention.model import LlamaConfig, random_llama
    cfg = LlamaConfig(vocab_size=512, hidden_size=2048, intermediate_size=4096, num_hidden_layers=2,
                      num_attention_heads=16, num_key_value_heads=4, head_dim=128,
                      delta_lambda=64, sliding_window=256, sink_tokens=16, kv_cache="fp8", **kw)
    return random_llama(cfg, "cuda", torch.bfloat16, seed=7)


def _ids(s, seed, b=1):
    return torch.randint(0, 512, (b, s), device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed))


@pytest.mark.parametrize("mode,gamma_dec", [("dense", 1), ("sparse", 1), ("delta", 3)])
def test_graph_decode_replays(gpu, mode, gamma_dec):
    """Recorded decode steps over the 8-bit cache: the same logits, bit for bit,
    as the static steps run eagerly; the host-length steps' to rounding."""
    m = _small_model(decode_mode=mode, gamma_dec=gamma_dec)
    assert m.graph_decodable()
    ids = _ids(700, 11)
    lg_graph, lg_static, lg_eager = [], [], []
    a = m.generate_greedy(ids, 10, graph=True, logits_out=lg_graph)
    b = m.generate_greedy(ids, 10, graph=True, record=False, logits_out=lg_static)
    c = m.generate_greedy(ids, 10, logits_out=lg_eager)
    assert a.shape == (1, 10) and torch.equal(a, b)
    for x, y in zip(lg_graph, lg_static):
        assert torch.equal(x, y)
    assert torch.equal(lg_graph[0], lg_eager[0])        # the prompt's own pass
    n_same = int((a == c).long().cumprod(1).sum())
    assert n_same >= 2
    for i in range(n_same):
        d = (lg_graph[i] - lg_eager[i]).abs().max().item()
        assert d <= 2e-2 * max(1.0, lg_eager[i].abs().max().item()), (i, d)


def test_generation_is_near_the_16_bit_cache(gpu):
    """The prompt's pass is the same; a decode step's logits move by what the
    codes' rounding (2^-4 of a value at most) makes of the attention output."""
    m = _small_model()
    ids = _ids(600, 12, b=2)
    lg8, lg16 = [], []
    t8 = m.generate_greedy(ids, 4, logits_out=lg8)
    m.config.kv_cache = "model"
    t16 = m.generate_greedy(ids, 4, logits_out=lg16)
    assert torch.equal(lg8[0], lg16[0]) and torch.equal(t8[:, 0], t16[:, 0])
    d = (lg8[1] - lg16[1]).abs().max().item()
    assert 0 < d <= 2.0 ** -4 * lg16[1].abs().max().item(), d
    m.config.kv_cache = "int4"
    with pytest.raises(ValueError, match="kv_cache"):
        m.generate_greedy(ids, 2)


def test_cache_contents_through_a_generation(gpu):
    """A prompt, static steps and host-length steps of the model write the
    layers' cache as the oracle does from the same keys and values; the prefill
    on a cache that holds tokens is refused."""
    from delta_attention.model import KVCache8
    m = _small_model()
    cfg = m.config
    cache = KVCache8(cfg, 1, 200, torch.device("cuda"), torch.bfloat16)
    ref = [K8.new_cache(1, 4, 256, 128) for _ in range(2)]
    seen = []
    from delta_attention import ops
    real = ops.kv8_write

    def spy(c, k, v, pos, **kw):
        layer = next(i for i, x in enumerate(cache.layers) if x.k.data_ptr() == c.k.data_ptr())
        p = int(pos) if not isinstance(pos, torch.Tensor) else int(pos.item())
        K8.write(ref[layer], np64(k), np64(v), [p])
        seen.append((layer, p, k.shape[1]))
        return real(c, k, v, pos, **kw)

    ops.kv8_write = spy
    try:
        with torch.inference_mode():
            ids = _ids(130, 3)
            m.model(ids, None, cache)
            with pytest.raises(NotImplementedError, match="whole prompt"):
                m.model(ids[:, :3], None, cache)
            assert cache.len == [130, 130] and len(seen) == 2      # nothing appended
            cfg._attn_implementation = "sdpa_rectangle"
            m.model(ids[:, :5], None, cache)
            cache.start_static()
            for _ in range(3):
                m.model(ids[:, :1], None, cache)
                cache.advance_static()
            cache.stop_static(3)
            m.model(ids[:, :1], None, cache)
    finally:
        ops.kv8_write = real
        cfg._attn_implementation = "window"
    assert cache.seq_len() == 139 and [p for l, p, _ in seen if l == 1] == [0, 130, 135, 136, 137, 138]
    for c, r in zip(cache.layers, ref):
        got = to_oracle(c)
        for x in ("k", "v"):
            assert same(got[x][:, :, :139], r[x][:, :, :139]), x
        for x in ("ke", "ve"):
            assert np.array_equal(got[x][:, :, :3], r[x][:, :, :3])


def test_loaded_model_generates_with_the_8_bit_cache(gpu, tmp_path):
    """init_model with kv_cache "fp8" (llama and Qwen3 checkpoints), the
    user-facing generate: same shapes, prompts kept, batch of padded rows."""
    from delta_attention.config import Config
    from delta_attention.sample import init_model
    for family in ("llama", "qwen3"):
        path = tmp_path / family
        write_checkpoint(path, family, seed=2, vocab_size=512, hidden_size=1280, intermediate_size=2048,
                         num_attention_heads=10, num_key_value_heads=2, head_dim=128)
        m, _ = init_model(Config(model_str=str(path), delta_lambda=16, sliding_window=128, sink_tokens=8,
                                 kv_cache="fp8"))
        assert m.config.kv_cache == "fp8"
        ids = _ids(300, 4, b=2)
        mask = torch.ones_like(ids)
        mask[1, :77] = 0
        out = m.generate(ids, attention_mask=mask, max_new_tokens=6, graph=True)
        assert out.shape == (2, 306) and torch.equal(out[:, :300], ids)
        one = m.generate(ids[1:, 77:], max_new_tokens=6, graph=True)
        assert torch.equal(one[0, -6:], out[1, -6:])
