"""What the 8-bit cache, prefix attention and sampling entry points refuse, without a GPU: every check of
the C ABI comes before anything touches the device, and the Python ops raise RuntimeError."""
import pytest
import torch

import twilight_amd.kernel as K
from twilight_amd.cache import QuantPagedKVCache

F = 0x1000  # never dereferenced: validation fails first


def _append(L, **kw):
    g = kw.get
    return L.twl_kv_quant_append(
        g("k", F), g("v", F), g("dt", 0), g("nts", 128), g("nhs", 128), g("ip", F), g("tokens", 4), g("kc", F),
        g("vc", F), g("fmt", 3), g("ps", 4096), g("ts", 256), g("hs", 128), g("ks", F), g("vs", F), 32, 2, 1,
        g("pages", 5), g("ids", F), g("ptr", F), g("last", F), g("b", 2), g("hkv", 2), 0)


def _read(L, **kw):
    g = kw.get
    return L.twl_kv_quant_read(
        g("k", F), g("v", F), g("dt", 0), g("ip", F), g("tokens", 4), g("kc", F), g("vc", F), g("fmt", 3),
        g("ps", 4096), g("ts", 256), g("hs", 128), g("ks", F), g("vs", F), 32, 2, 1, g("pages", 5), g("ids", F),
        g("ptr", F), g("last", F), g("b", 2), g("hkv", 2), 0)


def test_quant_cache_checks(hip_lib):
    for call in (_append, _read):
        c = lambda **kw: call(hip_lib, **kw)  # noqa: E731,B023
        for name in ("k", "v", "ip", "kc", "vc", "ks", "vs", "ids", "ptr", "last"):
            assert c(**{name: 0}) == -1, name
        assert c(fmt=0) == -3 and c(fmt=5) == -3 and c(dt=3) == -3
        assert c(tokens=0) == -2 and c(b=0) == -2 and c(hkv=0) == -2 and c(pages=0) == -2 and c(tokens=1 << 31) == -2
        assert c(ps=4100) == -4 and c(ts=252) == -4 and c(hs=130) == -4 and c(kc=F + 4) == -4 and c(ks=F + 2) == -4
        assert c(k=F + 8) == -4
    assert _append(hip_lib, dt=2) == -3                     # rows come in 16 bits
    assert _append(hip_lib, nts=132) == -4 and _append(hip_lib, nhs=4) == -4


def _attn(L, **kw):
    g = kw.get
    return L.twl_prefix_attn(
        g("q", F), g("out", F), g("dt", 0), g("k", F), g("v", F), g("fmt", 0), g("ps", 4096), g("ts", 256),
        g("hs", 128), g("ks", 0), g("vs", 0), 0, g("sts", 0), 0, g("pages", 9), g("pids", F), g("pptr", F), g("plast", F),
        g("gptr", F), g("groups", 1), g("mp", 100), g("mg", 2), g("ids", F), g("ptr", F), g("last", F), g("mt", 2000),
        g("b", 2), g("hq", 4), g("hkv", 2), g("scale", 0.1), 0, g("ws", F), g("wsb", 1 << 30), 0)


def test_prefix_attention_checks(hip_lib):
    c = lambda **kw: _attn(hip_lib, **kw)  # noqa: E731
    for name in ("q", "out", "k", "v", "ids", "ptr", "last", "pids", "pptr", "plast", "gptr", "ws"):
        assert c(**{name: 0}) == -1, name
    assert c(fmt=3) == -1 and c(fmt=4, ks=F) == -1           # 8-bit pages need both scales
    assert c(dt=2) == -3 and c(fmt=1) == -3 and c(fmt=2) == -3
    assert c(b=0) == -2 and c(hkv=0) == -2 and c(hq=3) == -2 and c(pages=0) == -2
    assert c(groups=3) == -2 and c(mg=0) == -2 and c(mg=3) == -2
    assert c(mt=(1 << 24) + 1) == -2 and c(mp=(1 << 24) + 1) == -2 and c(ts=1 << 25) == -2
    assert c(b=40000, hq=4, mg=1) == -2                      # more than 65535 rows
    assert c(scale=float("nan")) == -2
    need = hip_lib.twl_prefix_attn_workspace_bytes(2, 4, 2, 1, 100, 2, 2000)
    assert need > 0 and c(wsb=need - 1) == -2
    assert c(ps=4100) == -4 and c(hs=4) == -4 and c(q=F + 8) == -4 and c(out=F + 4) == -4 and c(ws=F + 8) == -4
    assert c(fmt=3, ks=F, vs=F, hs=136) == -4                # 8-bit rows start at 16 bytes
    # a context that is one part needs no workspace; many parts of many rows do not overflow
    w = hip_lib.twl_prefix_attn_workspace_bytes
    assert w(2, 4, 2, 0, 0, 0, 1024) == 0 and w(1, 4, 2, 0, 0, 0, 1 << 24) <= 4 * 257 * 130 * 4
    assert w(0, 4, 2, 0, 0, 0, 5) == 0 and w(1, 3, 2, 0, 0, 0, 5000) == 0


def _sample(L, **kw):
    g = kw.get
    return L.twl_sample_tokens(
        g("x", F), g("dt", 0), 64, g("rows", 2), g("v", 64), g("u", F), 0, g("t", 1.0), 0, 0, 0, g("p", 1.0), 0,
        g("m", 0.0), g("out", F), g("ws", F), g("wsb", 1 << 30), 0)


def test_sampling_checks(hip_lib):
    c = lambda **kw: _sample(hip_lib, **kw)  # noqa: E731
    for name in ("x", "u", "out", "ws"):
        assert c(**{name: 0}) == -1, name
    assert c(dt=3) == -3
    assert c(rows=0) == -2 and c(v=0) == -2 and c(v=(1 << 18) + 1) == -2 and c(rows=65536) == -2
    nan = float("nan")
    assert c(t=nan) == -2 and c(p=nan) == -2 and c(m=nan) == -2
    need = hip_lib.twl_sample_tokens_workspace_bytes(2, 64)
    assert need > 0 and c(wsb=need - 1) == -2
    assert c(x=F + 1) == -4 and c(dt=2, x=F + 2) == -4 and c(u=F + 2) == -4 and c(out=F + 4) == -4 and c(ws=F + 4) == -4
    assert hip_lib.twl_sample_tokens_workspace_bytes(2, (1 << 18) + 1) == 0


def _cpu_cache():
    k = torch.zeros(3, 16, 2, 128, dtype=torch.int8)
    s = torch.zeros(3, 16, 2)
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32)  # noqa: E731
    return (k, k.clone(), s, s.clone()), (i32(0), i32(0, 1), i32(3)), i32


def test_python_ops_refuse_cpu_tensors_and_wrong_types(hip_lib):
    pools, table, i32 = _cpu_cache()
    rows = torch.zeros(3, 2, 128, dtype=torch.float16)
    q = torch.zeros(1, 4, 128, dtype=torch.float16)
    with pytest.raises(RuntimeError, match="CUDA"):
        K.kv_quant_append(rows, rows, i32(0, 3), *pools, *table)
    with pytest.raises(RuntimeError, match="CUDA"):
        K.kv_quant_read(*pools, *table, i32(0, 3), 3)
    with pytest.raises(RuntimeError, match="CUDA"):
        K.quant_paged_decode_attention(q, *pools, *table, max_tokens=3)
    with pytest.raises(RuntimeError, match="need k_scale"):
        K.quant_paged_decode_attention(q, pools[0], pools[1], None, None, *table, max_tokens=3)
    with pytest.raises(RuntimeError, match="CUDA"):
        K.prefix_paged_decode_attention(q, *pools[:2], *table, i32(0, 1), *table, 3, 1, 3, *pools[2:])
    with pytest.raises(RuntimeError, match="CUDA"):
        K.sample_tokens(torch.zeros(1, 9), torch.zeros(1))
    with pytest.raises(RuntimeError, match="int8 or float8"):
        QuantPagedKVCache(4, 2, torch.float16, "cpu")


def test_quant_cache_shares_the_page_table(hip_lib):
    c = QuantPagedKVCache(6, 2, torch.int8, "cpu")
    assert c.k_cache.shape == (6, 16, 2, 128) and c.k_cache.stride() == (4096, 128, 2048, 1)
    assert c.k_scale.shape == (6, 16, 2) and c.k_scale.stride() == (32, 1, 16)
    c.set_page_table(torch.tensor([0, 1]), torch.tensor([0, 1, 2]), torch.tensor([16, 3]))
    assert c.batch == 2 and c.max_seq_len == 16
    free = [4, 5]
    c.advance_host(free)
    assert c.kv_page_indices.tolist() == [0, 4, 1] and c.kv_last_page_len.tolist() == [0, 3] and free == [5]
    assert c._seq_lens == [17, 4]


def test_calls_too_large_for_one_launch_and_scales_that_are_no_number(hip_lib):
    # 2^28 rows of 16 lanes are 2^32 threads
    assert _append(hip_lib, tokens=1 << 26, hkv=4) == -2 and _read(hip_lib, tokens=1 << 26, hkv=4) == -2
    assert _attn(hip_lib, scale=float("inf")) == -2 and _attn(hip_lib, scale=float("-inf")) == -2


def test_arguments_that_are_no_tensors(hip_lib):
    pools, table, i32 = _cpu_cache()
    q = torch.zeros(1, 4, 128, dtype=torch.float16)
    with pytest.raises(RuntimeError, match="[Tt]ensor"):
        K.quant_paged_decode_attention(None, *pools, *table, max_tokens=3)
    with pytest.raises(RuntimeError, match="[Tt]ensor"):
        K.quant_paged_decode_attention(q, [1], *pools[1:], *table, max_tokens=3)
    with pytest.raises(RuntimeError, match="[Tt]ensor"):
        K.kv_quant_read(None, *pools[1:], *table, i32(0, 3), 3)
    with pytest.raises(RuntimeError, match="CUDA"):
        K.kv_quant_append(None, None, [0, 3], *pools, *table)


def test_quant_cache_counts_its_appends_with_the_table(hip_lib):
    # the row counts of an append exist before a step is recorded, not from the recording on
    c = QuantPagedKVCache(6, 2, torch.float8_e4m3fn, "cpu")
    c.set_page_table(torch.tensor([0, 1, 2]), torch.tensor([0, 1, 2, 3]), torch.tensor([16, 3, 1]))
    assert c._one_each.tolist() == [0, 1, 2, 3]
