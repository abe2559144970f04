"""CPU checks of the 8-bit key/value cache: its oracle against torch's e4m3
casts, its argument checks at the C entry points and in ops, its layout."""

import os
import struct

import numpy as np
import pytest
import torch

import conftest  # noqa: F401  (paths)
from delta_attention import _lib as L
from delta_attention import ops
from kv8_helpers import place, same
from oracle import kv8_oracle as K8


@pytest.fixture(scope="module")
def lib():
    if not os.path.exists(L.LIB_PATH):
        import build_lib
        build_lib.build()
    return L.lib()


def test_oracle_rounding_is_torchs():
    x = torch.cat([torch.randn(20000) * 2.0 ** s for s in (-12, -8, -4, 0, 4, 6)]).clamp(-448, 448)
    x = torch.cat([x, torch.tensor([0.0, 448.0, 2.0 ** -9, 2.0 ** -10, 3 * 2.0 ** -10, 17.0, 19.0, 0.017578125])])
    assert same(K8.round_e4m3(x.numpy()), x.to(torch.float8_e4m3fn).double().numpy())
    assert np.isnan(K8.round_e4m3([np.nan, np.inf, -np.inf])).all()


def test_oracle_exponent():
    for e in (-117, -30, 0, 7, 120):
        assert K8.block_exponent(np.array([np.ldexp(448.0, e), np.inf, np.nan])) == e
        if e < 120:
            assert K8.block_exponent(np.array([np.ldexp(448.0, e) * (1 + 2.0 ** -40)])) == e + 1
    assert K8.block_exponent(np.zeros(3)) == K8.block_exponent(np.array([np.nan])) == K8.E_MIN
    assert K8.block_exponent(np.array([float(torch.finfo(torch.bfloat16).max)])) == K8.E_MAX


def test_oracle_growth_is_one_rounding_in_the_normal_range():
    """Codes that move to a larger power of two keep their values, but for
    those that become subnormal."""
    rng = np.random.default_rng(0)
    B, D = 1, 4
    c = K8.new_cache(B, 1, 64, D)
    x = rng.standard_normal((1, 8, 1, D))
    K8.write(c, x, x, [0])
    before, _ = K8.values(c, 0, 8)
    y = np.full((1, 1, 1, D), 100.0)
    K8.write(c, y, y, [8])
    after, _ = K8.values(c, 0, 9)
    scale = 2.0 ** int(c["ke"][0, 0, 0])
    normal = np.abs(before) >= scale * 2.0 ** -6
    assert normal.any() and np.array_equal(after[:, :, :8][normal], before[normal])
    assert np.abs(after[:, :, :8] - before).max() <= scale * 2.0 ** -10
    assert np.abs(after[0, 0, 8] - 100.0).max() <= 100 * 2.0 ** -4


def test_place_is_a_permutation_of_a_block():
    p = place()
    assert sorted(p) == list(range(64)) and p[0] == 0 and p[1] == 1 and p[4] == 16 and p[16] == 4 and p[63] == 63


def test_empty_cache_and_its_slices():
    c = ops.kv8_empty(2, 3, 100, 64, "cpu")
    assert c.k.shape == (2, 3, 128, 64) and c.v.shape == (2, 3, 2, 64, 64)
    assert c.k_scale.shape == c.v_scale.shape == (2, 3, 2) and (c.k_scale == 2.0 ** -117).all()
    for cache in (c, ops.KV8(*(t[:, 1:] for t in c))):       # (its layout passes: only the GPU is missing)
        with pytest.raises(AssertionError, match="GPU tensors"):
            ops.kv8_read(cache, 0, 5)
    for bad in (dict(D=96), dict(max_len=0), dict(max_len=(1 << 30) + 1), dict(Hkv=0)):
        with pytest.raises(AssertionError):
            ops.kv8_empty(**{**dict(B=1, Hkv=1, max_len=64, D=64, device="cpu"), **bad})


def test_ops_refuse_caches_that_are_not_laid_out_so():
    c = ops.kv8_empty(1, 2, 128, 64, "cpu")
    for bad in (c._replace(k=c.k[:, :, ::2]), c._replace(k=c.k[:, :, :100]), c._replace(v=c.v[:, :, :1]),
                c._replace(v=c.v.transpose(3, 4)), c._replace(k_scale=c.k_scale[..., :1]),
                c._replace(k=c.k.view(torch.uint8)), c._replace(v_scale=c.v_scale.double()),
                c._replace(k_scale=c.k_scale[..., 0:1].expand(1, 2, 2))):
        with pytest.raises(AssertionError, match="belong together|contiguous|float8|dimensions"):
            ops.kv8_read(bad, 0, 5)
    for bad in (tuple(c)[:3], None, [*c]):
        with pytest.raises(AssertionError, match="KV8 cache"):
            L.kv8_ext().read(bad, 0, 5, None, torch.zeros(1, 2, 5, 64), torch.zeros(1, 2, 5, 64))


def test_ops_refuse_arguments_on_the_cpu():
    c = ops.kv8_empty(1, 2, 128, 64, "cpu")
    k = torch.zeros(1, 3, 2, 64, dtype=torch.bfloat16)
    q = torch.zeros(1, 4, 1, 64, dtype=torch.bfloat16)
    with pytest.raises(AssertionError, match="GPU tensors"):
        ops.kv8_write(c, k, k, 0)
    with pytest.raises(AssertionError, match="k and v are"):
        ops.kv8_write(c, k[..., :32], k[..., :32], 0)
    with pytest.raises(AssertionError, match="different types"):
        ops.kv8_write(c, k, k.half(), 0)
    with pytest.raises(AssertionError, match="not supported"):
        ops.kv8_write(c, k.float(), k.float(), 0)
    with pytest.raises(AssertionError, match="a tensor is needed"):
        ops.kv8_write(c, None, k, 0)
    with pytest.raises(TypeError):
        L.kv8_ext().write(c, k)
    with pytest.raises(AssertionError, match="GPU tensors"):
        ops.kv8_attention(q, c, n_keys=1, sm_scale=1.0)
    with pytest.raises(AssertionError, match="multiple of 2"):
        ops.kv8_attention(q[:, :3], c, n_keys=1, sm_scale=1.0)
    for start, n in ((100, 29), (-1, 2), (0, -1)):
        with pytest.raises(AssertionError, match="rows"):
            ops.kv8_read(c, start, n)


def test_ops_refuse_a_cache_without_heads():
    """An empty slice over the heads is no cache, whatever the call."""
    c = ops.KV8(*(t[:, :0] for t in ops.kv8_empty(1, 2, 128, 64, "cpu")))
    k = torch.zeros(1, 3, 0, 64, dtype=torch.bfloat16)
    for call in (lambda: ops.kv8_write(c, k, k, 0), lambda: ops.kv8_read(c, 0, 5),
                 lambda: ops.kv8_attention(torch.zeros(1, 2, 1, 64, dtype=torch.bfloat16), c, n_keys=1, sm_scale=1.0)):
        with pytest.raises(AssertionError, match="kv head"):
            call()


def test_the_extension_refuses_what_is_no_cache_or_no_result():
    """Through its own signature: (cache, start, n, n_keys, dtype, results)."""
    c = ops.kv8_empty(1, 2, 128, 64, "cpu")
    read = L.kv8_ext().read
    k = torch.zeros(1, 2, 5, 64, dtype=torch.bfloat16)
    for bad in (tuple(c)[:3], None, [*c], c.k):
        with pytest.raises(AssertionError, match="KV8 cache"):
            read(bad, 0, 5, None, torch.bfloat16, (k, k.clone()))
    for bad in (k, (k,), [k, k]):
        with pytest.raises(AssertionError, match="out: two tensors"):
            read(c, 0, 5, None, torch.bfloat16, bad)
    for bad in ((k, None), (None, k)):
        with pytest.raises(AssertionError, match="a tensor is needed"):
            read(c, 0, 5, None, torch.bfloat16, bad)
    for bad in ((k, k[:, :, :4]), (k[:, :1], k[:, :1]), (k, k.half()), (k, k.transpose(2, 3).contiguous().transpose(2, 3))):
        with pytest.raises(AssertionError, match="the results are two"):
            read(c, 0, 5, None, torch.bfloat16, bad)
    with pytest.raises(AssertionError, match="not supported"):
        read(c, 0, 5, None, torch.bfloat16, (k.float(), k.float()))
    for bad in (None, "bfloat16", 5):
        with pytest.raises(AssertionError, match="torch.dtype"):
            read(c, 0, 5, None, bad, None)
    with pytest.raises(AssertionError, match="not supported"):
        read(c, 0, 5, None, torch.float32, None)
    with pytest.raises(TypeError):
        read(c, 0, 5, None, k, k, k)


# the header's structs, in native alignment
_CACHE = "4P8q4i"                                # k, v, k_scale, v_scale; {batch, head} strides; B, Hkv, cap, D
WRITE = struct.Struct(_CACHE + "4P7q4i")         # k, v, pos_dev, counts_dev; strides, pos; S, 2 flags, dtype
READ = struct.Struct(_CACHE + "3P6q4i")          # k, v, n_keys_dev; strides; start, n, flag, dtype
ATTN = struct.Struct(_CACHE + "5P10q7if")        # q, out, addend, n_keys_dev, workspace; its bytes, strides;
                                                 # Hq, s, flag, n_keys, window, sink, dtype; sm_scale
CACHE = dict(kc=16, vc=16, sk=16, sv=16, cs=(128 * 128, 64 * 128, 128 * 128, 64 * 128, 4, 2, 4, 2), B=1, Hkv=2,
             cap=128, D=64)


def _head(a):
    return (a["kc"], a["vc"], a["sk"], a["sv"], *a["cs"], a["B"], a["Hkv"], a["cap"], a["D"])


def test_c_write_refusals(lib):
    def call(**kw):
        a = dict(CACHE, k=16, v=16, ks=(3 * 128, 128, 64), vs=(3 * 128, 128, 64), S=3, pos=0, pos_dev=0, counts=0,
                 dtype=L.DA_BF16)
        a.update(kw)
        return lib.da_kv8_write(WRITE.pack(*_head(a), a["k"], a["v"], a["pos_dev"], a["counts"], *a["ks"],
                                                 *a["vs"], a["pos"], a["S"], 0, 0, a["dtype"]), None)
    assert call(dtype=5) == L.DA_ERR_DTYPE
    assert call(D=96) == L.DA_ERR_HEAD_DIM
    for bad in (dict(cap=100), dict(cap=0), dict(cap=-64), dict(cap=(1 << 30) + 64), dict(Hkv=0), dict(B=-1), dict(S=-1),
                dict(k=0), dict(v=0), dict(kc=0), dict(vc=0), dict(sk=0), dict(sv=0), dict(pos=-1), dict(pos=126),
                dict(S=129), dict(pos=2 ** 62), dict(Hkv=2 ** 30), dict(B=2, cs=(0, 64 * 128, 0, 64 * 128, 0, 2, 0, 2)),
                dict(cs=(128 * 128, 64 * 128, 128 * 128, 64 * 128, 4, 0, 4, 2))):
        assert call(**bad) == L.DA_ERR_INVALID_ARG, bad
    for bad in (dict(k=24), dict(vc=24), dict(sk=18), dict(ks=(3 * 128, 129, 64)), dict(pos_dev=20), dict(counts=18),
                dict(cs=(128 * 128 + 8, 64 * 128, 128 * 128, 64 * 128, 4, 2, 4, 2))):
        assert call(**bad) == L.DA_ERR_ALIGNMENT, bad
    assert call(S=0) == L.DA_OK and call(B=0) == L.DA_OK       # nothing launched
    assert lib.da_kv8_write(None, None) == L.DA_ERR_INVALID_ARG


def test_c_read_refusals(lib):
    def call(**kw):
        a = dict(CACHE, start=0, n=5, nk=0, ko=16, vo=16, st=(2 * 5 * 64, 5 * 64, 64), dtype=L.DA_FP16)
        a.update(kw)
        return lib.da_kv8_read(READ.pack(*_head(a), a["ko"], a["vo"], a["nk"], *a["st"], *a["st"], a["start"],
                                               a["n"], 0, a["dtype"]), None)
    assert call(dtype=2) == L.DA_ERR_DTYPE and call(D=48) == L.DA_ERR_HEAD_DIM
    for bad in (dict(start=-1), dict(n=-1), dict(start=124), dict(start=2 ** 31 - 1, n=2 ** 31 - 1), dict(ko=0),
                dict(kc=0), dict(cap=65)):
        assert call(**bad) == L.DA_ERR_INVALID_ARG, bad
    for bad in (dict(ko=24), dict(st=(640, 321, 64)), dict(nk=2)):
        assert call(**bad) == L.DA_ERR_ALIGNMENT, bad
    assert call(n=0) == L.DA_OK and call(B=0) == L.DA_OK
    assert lib.da_kv8_read(None, None) == L.DA_ERR_INVALID_ARG


def test_c_rows_refusals_and_workspace(lib):
    ws = lib.da_kv8_attn_workspace_bytes
    assert ws(1, 32, 8, 1, 128, 131072, 0, 0) > 0
    assert ws(1, 32, 8, 1, 128, 131072, 2048, 128) <= ws(1, 32, 8, 1, 128, 131072, 0, 0)
    assert ws(1, 32, 8, 1, 128, 64, 0, 0) == 0                 # one block: nothing to join
    assert ws(1, 32, 8, 1, 96, 131072, 0, 0) == 0 and ws(1, 30, 8, 1, 128, 131072, 0, 0) == 0
    assert ws(1, 32, 8, 0, 128, 131072, 0, 0) == 0 and ws(1, 32, 8, 1, 128, -1, 0, 0) == 0

    def call(**kw):
        a = dict(CACHE, cap=1024, q=16, qs=(8 * 64, 64, 64), out=16, Hq=8, s=1, nk=0, n=1000, window=0, sink=0, add=0,
                 as_=(8, 8, 8), ws=16, nb=1 << 30, dtype=L.DA_BF16)
        a.update(kw)
        return lib.da_kv8_attn_fwd(ATTN.pack(*_head(a), a["q"], a["out"], a["add"], a["nk"], a["ws"], a["nb"],
                                                   *a["qs"], 8 * 64, 64, 64, *a["as_"], a["Hq"], a["s"], 0, a["n"],
                                                   a["window"], a["sink"], a["dtype"], 0.1), None)
    assert call(dtype=3) == L.DA_ERR_DTYPE and call(D=512) == L.DA_ERR_HEAD_DIM
    for bad in (dict(Hq=9), dict(Hq=0), dict(s=-1), dict(window=-1), dict(sink=-1), dict(n=-1), dict(n=1025), dict(q=0),
                dict(out=0), dict(kc=0), dict(cap=1000), dict(s=1 << 30)):
        assert call(**bad) == L.DA_ERR_INVALID_ARG, bad
    assert ws(1, 8, 2, 1, 64, 1000, 0, 0) == 0                 # short lists stay whole
    need, long = ws(1, 8, 2, 1, 64, 4000, 0, 0), dict(cap=4096, n=4000)
    assert need > 0 and call(nb=need - 1, **long) == L.DA_ERR_WORKSPACE and call(ws=0, **long) == L.DA_ERR_WORKSPACE
    for bad in (dict(q=24), dict(out=24), dict(qs=(512, 65, 64)), dict(nk=18), dict(ws=24), dict(add=24),
                dict(add=16, as_=(8, 8, 4))):
        assert call(**bad) == L.DA_ERR_ALIGNMENT, bad
    assert call(s=0) == L.DA_OK and call(B=0) == L.DA_OK
    assert lib.da_kv8_attn_fwd(None, None) == L.DA_ERR_INVALID_ARG


def test_c_rows_of_sizes_past_any_launch(lib):
    """Products of sequences, heads and row tiles that pass 64 bits (2^64 = 0)
    are refused, and have no workspace."""
    big = 1 << 30
    for B, Hkv, G, s, keys in ((big, big, 1, 1024, 1000000), (big, big, 1, 1, 64), (1, 1, big, big, 1000000),
                               (1, 1, 1, 2 ** 31 - 1, 2 ** 31 - 1), (1 << 23, 1, 1, 1, 4096)):
        assert lib.da_kv8_attn_workspace_bytes(B, Hkv * G, Hkv, s, 32, keys, 0, 0) == 0
        a = dict(CACHE, B=B, Hkv=Hkv, cap=1 << 20, D=32)
        rc = lib.da_kv8_attn_fwd(ATTN.pack(*_head(a), 16, 16, 0, 16, 16, 1 << 40, *((32,) * 6), *((0,) * 3), Hkv * G, s, 0,
                                           0, 0, 0, L.DA_BF16, 0.1), None)
        assert rc == L.DA_ERR_INVALID_ARG, (B, Hkv, G, s)


def test_c_results_that_share_their_place(lib):
    """Results with a zero stride over sequences, heads or rows are refused;
    over a single entry a stride counts for nothing (no launch: n or s = 0)."""
    def read(ks, vs, B=2, n=5):
        a = dict(CACHE, B=B)
        return lib.da_kv8_read(READ.pack(*_head(a), 16, 16, 0, *ks, *vs, 0, n, 0, L.DA_BF16), None)

    def rows(os, B=2, Hq=4, s=3):
        a = dict(CACHE, B=B)
        return lib.da_kv8_attn_fwd(ATTN.pack(*_head(a), 16, 16, 0, 0, 16, 1 << 30, 3 * 256, 64, 256, *os, 0, 0, 0, Hq, s, 0,
                                             100, 0, 0, L.DA_BF16, 0.1), None)
    good = (640, 320, 64)
    for i in range(3):
        bad = tuple(0 if j == i else x for j, x in enumerate(good))
        assert read(bad, good) == read(good, bad) == L.DA_ERR_INVALID_ARG, bad
        assert rows(bad) == L.DA_ERR_INVALID_ARG, bad
    assert read((0, 0, 0), (0, 0, 0), n=0) == rows((0, 0, 0), s=0) == L.DA_OK


def test_c_rows_past_a_grids_threads(lib):
    """2^22 row tiles, dealt to the XCDs by eights, pass a grid's 2^32 threads."""
    a = dict(CACHE, Hkv=1, D=32)
    rc = lib.da_kv8_attn_fwd(ATTN.pack(*_head(a), 16, 16, 0, 0, 0, 0, *((32,) * 6), *((0,) * 3), 1, 1 << 28, 0, 64, 0, 0,
                                       L.DA_BF16, 0.1), None)
    assert rc == L.DA_ERR_INVALID_ARG
