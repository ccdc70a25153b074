"""An append that is refused leaves the cache as it was: page lists, lengths on both sides, the free list."""
import pytest
import torch

from twilight_amd.cache import PagedKVCache, QuantPagedKVCache

i32 = lambda *v: torch.tensor(v, dtype=torch.int32)  # noqa: E731


def _make(kind, dev="cpu"):
    c = PagedKVCache(10, 1, torch.float16, dev) if kind == "paged" else QuantPagedKVCache(10, 1, kind, dev)
    c.set_page_table(i32(0, 1, 2), i32(0, 1, 2, 3), i32(16, 16, 4))
    return c


def _state(c):
    return ([t.tolist() for t in (c.kv_page_indices, c.kv_page_indptr, c.kv_last_page_len)], [list(r) for r in c._per_req],
            list(c._last), list(c._seq_lens), c._room, c.max_pages_per_req)


@pytest.mark.parametrize("kind", ["paged", torch.int8])
def test_too_few_free_pages(hip_lib, kind):
    c, free = _make(kind), [7]
    before = _state(c)
    with pytest.raises(RuntimeError, match=f"{type(c).__name__}.append: no free page"):
        c.advance_host(free)                    # two requests need a page
    assert _state(c) == before and free == [7]
    free.append(8)
    c.advance_host(free)
    assert c.kv_page_indices.tolist() == [0, 7, 1, 8, 2] and c._seq_lens == [17, 17, 5] and free == []


@pytest.mark.parametrize("kind", ["paged", torch.int8])
def test_a_reserved_table_that_is_full(hip_lib, kind):
    c, free = _make(kind), [7, 8]
    c.reserve_page_table(1)
    before = _state(c)
    for _ in range(2):                          # a second try is refused too
        with pytest.raises(RuntimeError, match="outgrew reserve_page_table"):
            c.advance_host(free)
        assert _state(c) == before and free == [7, 8]


def test_a_plane_buffer_that_is_full(hip_lib):
    c, free = _make("paged"), [7, 8]
    c.meta_planes = torch.zeros(3, 1, 128, 2, 1)
    before = _state(c)
    for _ in range(2):
        with pytest.raises(RuntimeError, match="outgrew the plane buffer"):
            c.advance_host(free)
        assert _state(c) == before and free == [7, 8]
