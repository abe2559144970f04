"""CPU checks of the shared-prefix rows: the refusals of ops.prefix_attention
and da_prefix_attn_fwd, and the workspace's sizes."""

import os
import struct

import pytest
import torch

import conftest  # noqa: F401  (paths)
from delta_attention import _lib as L
from delta_attention import ops


@pytest.fixture(scope="module")
def lib():
    if not os.path.exists(L.LIB_PATH):
        import build_lib
        build_lib.build()
    return L.lib()


def _tensors(B=4, P=2, H=4, Hkv=2, s=1, D=64, Np=10, n=6, dtype=torch.bfloat16):
    return [torch.zeros(*sh, dtype=dtype) for sh in ((B, H, s, D), (P, Hkv, Np, D), (P, Hkv, Np, D), (B, Hkv, n, D),
                                                     (B, Hkv, n, D))]


def test_ops_refusals():
    def call(ts, **kw):
        return ops.prefix_attention(*ts, **{**dict(sm_scale=0.1), **kw})

    ts = _tensors()
    with pytest.raises(AssertionError, match="GPU tensors"):
        call(ts)
    for bad, match in ((_tensors(P=3), "does not share"), (_tensors(P=0), "does not share"), (_tensors(H=5), "query heads"),
                       (_tensors(Hkv=0, H=4), "query heads"), (_tensors(dtype=torch.float32), "not supported"),
                       ([ts[0], ts[1], ts[2][:, :, :9], ts[3], ts[4]], "k_prefix and v_prefix"),
                       ([ts[0], ts[1][..., :32], ts[2][..., :32], ts[3], ts[4]], "k_prefix and v_prefix"),
                       ([ts[0], ts[1], ts[2], ts[3][:3], ts[4][:3]], "k and v are"),
                       ([ts[0], ts[1], ts[2], ts[3], ts[4][:, :1]], "k and v are"),
                       ([ts[0], ts[1], ts[2], ts[3], ts[4].half()], "different types"),
                       ([ts[0][0], *ts[1:]], "four dimensions"), ([None, *ts[1:]], "a tensor is needed")):
        with pytest.raises(AssertionError, match=match):
            call(bad)
    with pytest.raises(TypeError):
        L.gen_ext().prefix(*ts)


@pytest.mark.gpu
def test_ops_refuse_counts_and_results(gpu):
    ts = [t.cuda() for t in _tensors()]

    def call(**kw):
        return ops.prefix_attention(*ts, **{**dict(sm_scale=0.1), **kw})

    i32 = dict(dtype=torch.int32, device="cuda")
    for bad in (dict(n_prefix=11), dict(n_prefix=-1), dict(n_keys=7), dict(n_keys=-1), dict(n_prefix=torch.ones(3, **i32)),
                dict(n_keys=torch.ones(2, **i32)), dict(n_keys=torch.ones(4, dtype=torch.int64, device="cuda")),
                dict(n_keys=torch.ones(4, dtype=torch.int32)), dict(n_keys=torch.ones(8, **i32)[::2]),
                dict(out=ts[0].half()), dict(out=ts[0][:2]), dict(out=torch.zeros(4, 4, 1, 64, dtype=torch.bfloat16)),
                dict(out=ts[0][:1].expand(4, -1, -1, -1)), dict(sm_scale=float("nan")), dict(sm_scale=float("inf"))):
        with pytest.raises(AssertionError):
            call(**bad)
    with pytest.raises(AssertionError, match="one device"):
        ops.prefix_attention(ts[0], ts[1].cpu(), *ts[2:], sm_scale=0.1)
    with pytest.raises(TypeError):
        call(sm_scale="big")


# the header's struct, in native alignment
ARGS = struct.Struct("9P19q13if")


def test_c_refusals_and_workspace(lib):
    ws = lib.da_prefix_attn_workspace_bytes
    assert ws(16, 1, 32, 8, 1, 128, 131072, 512) > 0 and ws(2, 1, 4, 2, 1, 64, 0, 0) == 0
    for bad in ((0, 1, 4, 2, 1, 64, 9, 9), (4, 3, 4, 2, 1, 64, 9, 9), (4, 0, 4, 2, 1, 64, 9, 9), (4, 2, 5, 2, 1, 64, 9, 9),
                (4, 2, 4, 2, 0, 64, 9, 9), (4, 2, 4, 2, 1, 96, 9, 9), (4, 2, 4, 2, 1, 64, -1, 9), (4, 2, 4, 2, 1, 64, 9, -1),
                (4, 2, 4, 2, 1, 64, 2 ** 30 + 1, 9)):
        assert ws(*bad) == 0, bad
    # sizes whose products pass 32 or 64 bits
    big = 1 << 30
    for bad in ((big, 1, big, 1, big, 64, big, big), (1, 1, big, 1, 1, 64, 9, 9), (1 << 23, 1, 1, 1, 1, 64, 9, 9),
                (1, 1, 1, 1, 2 ** 31 - 1, 64, 9, 9), (2 ** 31 - 1, 1, 2 ** 31 - 1, 2 ** 31 - 1, 1, 32, 9, 9)):
        assert ws(*bad) == 0, bad

    def call(**kw):
        st = (4 * 64, 64, 64)
        a = dict(q=16, kp=16, vp=16, k=16, v=16, out=16, npd=0, nkd=0, ws=16, nb=1 << 40, qs=st, kps=(640 * 2, 640, 64),
                 vps=(640 * 2, 640, 64), ks=(128, 64, 128), vs=(128, 64, 128), os=st, B=4, P=2, Hq=4, Hkv=2, s=1, D=64, Np=10,
                 n=6, npre=10, nk=6, dtype=L.DA_BF16, scale=0.1)
        a.update(kw)
        return lib.da_prefix_attn_fwd(ARGS.pack(
            a["q"], a["kp"], a["vp"], a["k"], a["v"], a["out"], a["npd"], a["nkd"], a["ws"], a["nb"], *a["qs"], *a["kps"],
            *a["vps"], *a["ks"], *a["vs"], *a["os"], a["B"], a["P"], a["Hq"], a["Hkv"], a["s"], a["D"], a["Np"], a["n"],
            a["npre"], a["nk"], 0, 0, a["dtype"], a["scale"]), None)

    assert call(dtype=2) == call(dtype=-1) == L.DA_ERR_DTYPE and call(D=96) == L.DA_ERR_HEAD_DIM
    for bad in (dict(P=3), dict(P=0), dict(P=-2), dict(Hq=5), dict(Hq=0), dict(Hkv=0), dict(s=-1), dict(B=-2), dict(Np=-1),
                dict(n=-1), dict(npre=11), dict(npre=-1), dict(nk=7), dict(nk=-1), dict(q=0), dict(kp=0), dict(v=0), dict(out=0),
                dict(scale=float("nan")), dict(scale=float("inf")), dict(os=(0, 64, 64)), dict(os=(256, 0, 64)),
                dict(s=3, os=(256, 64, 0)), dict(ks=(128, 64, (1 << 24) + 8)), dict(kps=(1280, 640, -64)),
                dict(Np=2 ** 30 + 1, npre=1), dict(B=2 ** 30, P=1, Hkv=4)):
        assert call(**bad) == L.DA_ERR_INVALID_ARG, bad
    for bad in (dict(q=24), dict(kp=24), dict(vp=8), dict(k=20), dict(v=17), dict(out=24), dict(npd=18), dict(nkd=17),
                dict(qs=(256, 68, 64)), dict(kps=(1281, 640, 64)), dict(vs=(128, 64, 132)), dict(os=(256, 64, 12)), dict(ws=24)):
        assert call(**bad) == L.DA_ERR_ALIGNMENT, bad
    assert ws(4, 2, 4, 2, 1, 64, 10, 6) == 0             # (short keys need none)
    long = dict(Np=2000, npre=2000)
    need = ws(4, 2, 4, 2, 1, 64, 2000, 6)
    assert need > 0 and call(nb=need - 1, **long) == call(ws=0, **long) == L.DA_ERR_WORKSPACE
    assert call(s=0) == call(B=0) == L.DA_OK             # nothing launched
    assert lib.da_prefix_attn_fwd(None, None) == L.DA_ERR_INVALID_ARG


def test_keys_that_overlap_are_refused_in_c(lib):
    """Keys nearer each other than a key's own elements: what lies behind the last
    one would be its own bytes again. (ops.prefix_attention copies such tensors.)"""
    def call(Np, n, **strides):
        st = dict(kps=(1280, 640, 64), vps=(1280, 640, 64), ks=(128, 64, 128), vs=(128, 64, 128))
        st.update(strides)
        return lib.da_prefix_attn_fwd(ARGS.pack(16, 16, 16, 16, 16, 16, 0, 0, 16, 0, 256, 64, 64, *st["kps"], *st["vps"],
                                                *st["ks"], *st["vs"], 256, 64, 64, 4, 2, 4, 2, 1, 64, Np, n, Np, n, 0, 0,
                                                L.DA_BF16, 0.1), None)

    for name in ("kps", "vps", "ks", "vs"):
        for step in (0, 8, 56, -64, (1 << 24) + 8):
            assert call(2000, 2000, **{name: (1280, 640, step)}) == L.DA_ERR_INVALID_ARG, (name, step)
    # (as far as the workspace's check: strides that are taken)
    for strides in (dict(), dict(ks=(1280, 640, 1 << 24))):
        assert call(2000, 2000, **strides) == L.DA_ERR_WORKSPACE
    # a set of one key has no step
    assert call(1, 2000, kps=(1280, 640, 0), vps=(1280, 640, -8)) == call(2000, 1, ks=(64, 64, 0)) == L.DA_ERR_WORKSPACE
