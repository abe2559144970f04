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
