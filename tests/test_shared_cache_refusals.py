"""CPU checks of a cache whose sequences share their prompts: one-token steps of
the sparse and delta decodes refuse it before anything is appended."""

import types

import pytest
import torch

import conftest  # noqa: F401  (paths)
from delta_attention.llama import LlamaAttention, SharedKeys


def layer(mode, impl="sdpa_rectangle"):
    cfg = types.SimpleNamespace(hidden_size=64, num_attention_heads=2, num_key_value_heads=1, head_dim=32,
                                attention_bias=False, attention_dropout=0.0, rms_norm_eps=1e-6,
                                _attn_implementation=impl, decode_mode=mode, sliding_window=8, sink_tokens=2)
    return LlamaAttention(cfg, 0)


class Cache:
    """A shared cache that holds a prompt; an append fails the test."""
    shared, static, len = True, False, [10]

    def update(self, *a):
        raise RuntimeError("appended")


@pytest.mark.parametrize("b", [1, 3])
@pytest.mark.parametrize("mode", ["sparse", "delta"])
def test_one_token_steps_are_refused(mode, b):
    m = layer(mode)
    h, rot = torch.zeros(b, 1, 64), (torch.ones(b, 1, 32), torch.zeros(b, 1, 32))
    with pytest.raises(NotImplementedError, match=f"dense decode steps .*'{mode}'"):
        m(h, rot, past_key_value=Cache())
    # and by the attention itself
    k = torch.zeros(b, 1, 4, 32)
    with pytest.raises(NotImplementedError, match=f"dense decode steps .*'{mode}'"):
        m.sdpa_rectangle_forward(m, torch.zeros(b, 2, 1, 32), SharedKeys(k, k, k, k, 4), None)


def test_dense_steps_and_passes_of_several_tokens_go_on():
    for mode, s in (("dense", 1), ("sparse", 2), ("delta", 5)):
        with pytest.raises(RuntimeError, match="appended"):
            layer(mode)(torch.zeros(2, s, 64), (torch.ones(2, s, 32), torch.zeros(2, s, 32)), past_key_value=Cache())
