"""CPU checks of the token choice: the oracle on rows that can be counted out,
and the refusals of ops.sample_tokens and da_sample."""

import math
import os
import struct

import numpy as np
import pytest
import torch

import conftest  # noqa: F401  (paths)
from delta_attention import _lib as L
from delta_attention import ops
from oracle import sample_oracle as S


@pytest.fixture(scope="module")
def lib():
    if not os.path.exists(L.LIB_PATH):
        import build_lib
        build_lib.build()
    return L.lib()


def test_oracle_on_rows_that_can_be_counted_out():
    x = np.log([4.0, 1.0, 2.0, 1.0])             # probabilities 1/2, 1/8, 1/4, 1/8
    for u, t in ((0.0, 0), (0.49, 0), (0.51, 1), (0.62, 1), (0.63, 2), (0.87, 2), (0.88, 3), (0.999, 3)):
        assert S.sample(x, u)[0] == t
    assert S.sample(x, 0.99, top_k=2)[:2] == (2, pytest.approx(math.log(1 / 3)))
    assert S.sample(x, 0.99, top_k=3)[0] == 2 and S.sample(x, 0.6, top_k=3)[0] == 1      # ties by index
    assert S.sample(x, 0.99, top_p=0.4)[0] == 0 and S.sample(x, 0.99, top_p=0.51)[0] == 2
    assert S.sample(x, 0.99, min_p=0.4)[0] == 2 and S.sample(x, 0.99, min_p=0.2)[0] == 3
    assert S.sample(x, 0.9, temperature=0.0)[:2] == (0, 0.0)
    # temperature 1/2 squares the weights: 16, 1, 4, 1
    assert S.sample(x, 16.5 / 22, temperature=0.5)[0] == 1
    assert S.sample([-np.inf, np.nan, 3.0], 0.5)[0] == 2
    t, lp, _ = S.sample([-np.inf, np.nan], 0.5)
    assert t == 0 and math.isnan(lp)
    assert S.sample([1.0, np.inf, 0.0, np.inf], 0.6)[:2] == (3, pytest.approx(math.log(0.5)))


def test_ops_refusals():
    x, u = torch.zeros(3, 10), torch.zeros(3)
    with pytest.raises(AssertionError, match="GPU tensors"):
        ops.sample_tokens(x, u)
    for bad in (x[0], x[:, :0], x[None]):
        with pytest.raises(AssertionError, match="rows, tokens"):
            ops.sample_tokens(bad, u)
    for bad in (x.double(), x.long()):
        with pytest.raises(AssertionError, match="not supported"):
            ops.sample_tokens(bad, u)
    for bad in (u[:2], u.double(), u[:, None], torch.zeros(6)[::2]):
        with pytest.raises(AssertionError, match="u: a contiguous float32"):
            ops.sample_tokens(x, bad)
    with pytest.raises(AssertionError, match="a tensor is needed"):
        ops.sample_tokens(x, 0.5)


@pytest.mark.skipif(not torch.cuda.is_available(), reason="the settings are checked after the device")
@pytest.mark.gpu
def test_ops_refuse_settings():
    x, u = torch.zeros(3, 10, device="cuda"), torch.zeros(3, device="cuda")
    for bad in (dict(temperature=-0.5), dict(temperature=math.nan), dict(temperature=math.inf), dict(top_p=1.5),
                dict(top_p=-0.1), dict(top_p=math.nan), dict(min_p=1.01), dict(min_p=-1e-3), dict(top_k=-1),
                dict(top_k=2 ** 31), dict(temperature=torch.ones(3)), dict(top_p=torch.ones(2, device="cuda")),
                dict(min_p=torch.ones(3, device="cuda", dtype=torch.float64)),
                dict(top_k=torch.ones(3, device="cuda", dtype=torch.int64)),
                dict(top_k=torch.ones(6, device="cuda", dtype=torch.int32)[::2])):
        with pytest.raises(AssertionError):
            ops.sample_tokens(x, u, **bad)
    for bad in (dict(temperature="hot"), dict(top_k=1.5), dict(top_p=None)):
        with pytest.raises(TypeError):
            ops.sample_tokens(x, u, **bad)


# the header's struct, in native alignment
ARGS = struct.Struct("9P2q8i3f")


def test_c_refusals(lib):
    def call(**kw):
        a = dict(x=16, u=16, td=0, kd=0, pd=0, md=0, tok=16, lp=16, ws=0, nb=0, rs=100, B=2, V=100, dtype=L.DA_BF16,
                 k=0, t=1.0, p=1.0, m=0.0)
        a.update(kw)
        return lib.da_sample(ARGS.pack(a["x"], a["u"], a["td"], a["kd"], a["pd"], a["md"], a["tok"], a["lp"], a["ws"],
                                       a["nb"], a["rs"], a["B"], a["V"], a["dtype"], 0, 0, 0, 0, a["k"], a["t"], a["p"],
                                       a["m"]), None)
    assert call(dtype=3) == call(dtype=-1) == L.DA_ERR_DTYPE
    for bad in (dict(V=0), dict(V=-1), dict(V=(1 << 24) + 1), dict(B=-1), dict(B=1 << 22), dict(x=0), dict(u=0),
                dict(tok=0), dict(lp=0)):
        assert call(**bad) == L.DA_ERR_INVALID_ARG, bad
    for bad in (dict(x=17), dict(x=18, dtype=L.DA_FP32), dict(u=18), dict(tok=20), dict(lp=18), dict(td=18),
                dict(kd=17), dict(pd=18), dict(md=18)):
        assert call(**bad) == L.DA_ERR_ALIGNMENT, bad
    assert call(B=0) == L.DA_OK                  # nothing launched
    assert lib.da_sample(None, None) == L.DA_ERR_INVALID_ARG
    ws = lib.da_sample_workspace_bytes
    assert ws(0, 10, L.DA_BF16) == ws(1, 0, L.DA_BF16) == ws(1, 10, 5) == ws(1, 1 << 25, L.DA_BF16) == 0
    assert ws(1, 8192, L.DA_BF16) == ws(160, 100000, L.DA_FP32) == 0       # a workgroup a row
    need = ws(2, 100000, L.DA_BF16)
    if need:
        assert call(V=100000, rs=100000, ws=16, nb=need - 1) == call(V=100000, rs=100000, nb=need) == L.DA_ERR_WORKSPACE
        assert call(V=100000, rs=100000, ws=24, nb=need) == L.DA_ERR_ALIGNMENT


def test_a_generation_of_no_tokens_is_refused():
    import torch
    from delta_attention.model import LlamaForCausalLM
    with pytest.raises(AssertionError):
        LlamaForCausalLM.generate_sampled(None, torch.zeros(1, 4, dtype=torch.int64), 0, torch.zeros(1, 0))
