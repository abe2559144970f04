"""CPU checks of LlamaForCausalLM.generate's arguments: each sequence gets its
own random numbers and settings, also where padded rows run by themselves."""

import types

import pytest
import torch

import conftest  # noqa: F401  (paths)
from delta_attention.model import LlamaForCausalLM


class Model(types.SimpleNamespace):
    """generate's model: generate_sampled keeps what it is called with and gives
    each sequence's first draw, as per mille, for every token."""

    def generate_sampled(self, ids, n, u, **kw):
        self.calls.append((ids.shape, u, kw))
        return (u[:, :1] * 1000).long().expand(-1, n)


def draw(ids, **kw):
    m = Model(calls=[])
    out = LlamaForCausalLM.generate(m, ids, max_new_tokens=4, do_sample=True,
                                    generator=torch.Generator().manual_seed(3), **kw)
    return m.calls, out


@pytest.mark.parametrize("n_seq", [1, 3])
def test_settings_of_the_sequences_of_padded_rows(n_seq):
    b = 3
    ids = torch.arange(b * 6).view(b, 6)
    mask = torch.ones_like(ids)
    mask[1, :2] = 0
    rows = b * n_seq
    settings = dict(temperature=torch.linspace(0.5, 1.5, rows), top_k=torch.arange(rows, dtype=torch.int32),
                    top_p=torch.linspace(0.1, 0.9, rows), min_p=torch.tensor([0.25]))
    whole, out = draw(ids, num_return_sequences=n_seq, **settings)
    each, padded = draw(ids, attention_mask=mask, num_return_sequences=n_seq, **settings)
    assert len(whole) == 1 and len(each) == b
    assert [c[0] for c in each] == [(1, 6), (1, 4), (1, 6)]
    assert torch.equal(out, padded)
    (_, u, kw), = whole
    for name in ("temperature", "top_k", "top_p"):
        assert torch.equal(kw[name], settings[name])
    for i, (_, mine, own) in enumerate(each):
        at = slice(i * n_seq, (i + 1) * n_seq)
        assert torch.equal(mine, u[at])
        for name in ("temperature", "top_k", "top_p"):
            assert torch.equal(own[name], settings[name][at]) and own[name].is_contiguous()
        assert torch.equal(own["min_p"], settings["min_p"])     # (one for all)
        assert own["samples"] == n_seq


def test_numbers_are_passed_on():
    ids = torch.arange(12).view(2, 6)
    mask = torch.ones_like(ids)
    mask[0, 0] = 0
    for kw in (dict(), dict(attention_mask=mask)):
        for _, _, got in draw(ids, temperature=0.5, top_p=0.75, **kw)[0]:
            assert (got["temperature"], got["top_k"], got["top_p"], got["min_p"]) == (0.5, 50, 0.75, 0.0)


@pytest.mark.parametrize("padded", [False, True])
def test_settings_of_another_number_of_sequences_are_refused(padded):
    ids = torch.arange(12).view(2, 6)
    mask = torch.ones_like(ids)
    if padded:
        mask[0, 0] = 0
    for n in (2, 3, 5):
        with pytest.raises(AssertionError, match="temperature"):
            draw(ids, attention_mask=mask, num_return_sequences=2, temperature=torch.ones(n))
