"""Requests that start without a page: the host bookkeeping of a decode append, and the tokens on the device."""
import pytest
import torch

import twilight_amd.kernel as K
from twilight_amd.cache import PagedKVCache, QuantPagedKVCache
from _quant import attention64, check_attention, decode, encode

i32 = lambda *v: torch.tensor(v, dtype=torch.int32)  # noqa: E731


def _make(kind, dev, pages=8, Hkv=2):
    return PagedKVCache(pages, Hkv, torch.float16, dev) if kind == "paged" else QuantPagedKVCache(pages, Hkv, kind, dev)


@pytest.mark.parametrize("kind", ["paged", torch.int8])
@pytest.mark.parametrize("empty_last", [0, 16, 5])          # a request without pages has no tokens whatever this says
def test_an_empty_request_takes_a_page_with_its_first_token(hip_lib, kind, empty_last):
    c = _make(kind, "cpu")
    c.set_page_table(i32(0), i32(0, 1, 1), i32(3, empty_last))
    assert c._seq_lens == [3, 0] and c.max_seq_len == 3
    free = [5, 6]
    c.advance_host(free)
    assert free == [6] and c.kv_page_indices.tolist() == [0, 5] and c.kv_page_indptr.tolist() == [0, 1, 2]
    assert c.kv_last_page_len.tolist() == [3, 0] and c._last == [4, 1] and c._seq_lens == [4, 1]
    for _ in range(12):
        c.advance_host(free)
    assert free == [6] and c._last == [16, 13]
    c.advance_host(free)                                     # request 0 fills up before request 1
    assert free == [] and c.kv_page_indices.tolist() == [0, 6, 5] and c._seq_lens == [17, 14]


@pytest.mark.parametrize("kind", ["paged", torch.int8])
def test_all_requests_empty_and_a_reserved_table(hip_lib, kind):
    c = _make(kind, "cpu")
    c.set_page_table(i32(), i32(0, 0, 0), i32(0, 0))
    assert c._seq_lens == [0, 0] and c.max_seq_len == 0 and c.max_pages_per_req == 0
    c.reserve_page_table(2)
    ids, free = c.kv_page_indices, [7, 3]
    c.advance_host(free)
    assert c.kv_page_indices is ids and ids.tolist() == [7, 3, 0, 0] and c.kv_page_indptr.tolist() == [0, 1, 2]
    assert c._last == [1, 1] and c._seq_lens == [1, 1]
    c = _make(kind, "cpu")
    c.set_page_table(i32(), i32(0, 0, 0), i32(0, 0))
    with pytest.raises(RuntimeError, match="no free page"):
        c.advance_host()


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", [torch.int8, torch.float8_e4m3fn])
def test_tokens_appended_to_an_empty_request_are_kept(dev, fmt):
    H, Hkv, g = 4, 2, torch.Generator().manual_seed(1)
    rows = lambda *s: torch.randn(s, generator=g).half()  # noqa: E731
    k0, v0 = rows(3, Hkv, 128), rows(3, Hkv, 128)
    c = QuantPagedKVCache(8, Hkv, fmt, dev)
    c.set_page_table(i32(2), i32(0, 0, 1, 1), i32(0, 3, 0))  # the first and the last request hold nothing
    K.kv_quant_append(k0.to(dev), v0.to(dev), i32(0, 0, 3, 3).to(dev), *c.pools, *c.table)
    ks, vs, free = [], [], [5, 4, 7, 6, 1]
    for _ in range(18):
        ks.append(rows(3, Hkv, 128)), vs.append(rows(3, Hkv, 128))
        c.append(ks[-1].to(dev), vs[-1].to(dev), free)
    want = []
    for first, steps in ((k0, ks), (v0, vs)):
        per = [torch.stack([s[b] for s in steps]) for b in range(3)]
        per[1] = torch.cat([first, per[1]])
        want.append([decode(*encode(x, fmt)) for x in per])
    got = c.read(torch.float32)
    for x, w in zip(got, want):
        assert torch.equal(x.cpu(), torch.cat(w))
    q = rows(3, H, 128)
    out, lse = K.quant_paged_decode_attention(q.to(dev), *c.pools, *c.table, max_tokens=c.max_seq_len, return_lse=True)
    for b in range(3):
        k, v = (w[b].double() for w in want)
        check_attention(out[b].cpu(), lse[b].cpu(), attention64(q[b], k, v, 128 ** -0.5), len(k), torch.float16,
                        torch.float16)


@pytest.mark.gpu
def test_16_bit_pages_too(dev):
    c = PagedKVCache(4, 2, torch.float16, dev)
    c.set_page_table(i32(1), i32(0, 0, 1), i32(0, 2))
    new = torch.randn(2, 2, 128).half()
    c.append(new.to(dev), -new.to(dev), [3])
    assert torch.equal(c.k_cache[3, 0].cpu(), new[0]) and torch.equal(c.v_cache[1, 2].cpu(), -new[1])
    assert c.kv_last_page_len.tolist() == [1, 3] and torch.count_nonzero(c.k_cache).item() == torch.count_nonzero(new).item()


@pytest.mark.gpu
def test_a_cache_from_no_tokens(dev):
    none = torch.zeros(2, 3, 0, 128, dtype=torch.float16)
    c = QuantPagedKVCache.from_dense(none, none, torch.int8, dev, spare_pages=4)
    assert c._seq_lens == [0, 0] and [t.shape[0] for t in c.read()] == [0, 0]
    new, free = torch.randn(2, 3, 128).half(), [3, 0, 1]
    c.append(new.to(dev), -new.to(dev), free)
    k, v = c.read(torch.float32)
    assert free == [1] and torch.equal(k.cpu(), decode(*encode(new, torch.int8))) and torch.equal(v, -k)
