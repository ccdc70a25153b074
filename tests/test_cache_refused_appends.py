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


BAD_ROWS = [
    (torch.zeros(2, 1, 128, dtype=torch.float16),) * 2,                    # a row is missing
    (torch.zeros(4, 1, 128, dtype=torch.float16),) * 2,                    # one too many
    (torch.zeros(3, 2, 128, dtype=torch.float16),) * 2,                    # other heads
    (torch.zeros(3, 1, 64, dtype=torch.float16),) * 2,
    (torch.zeros(3, 128, dtype=torch.float16),) * 2,
    (torch.zeros(3, 1, 128), torch.zeros(3, 1, 128)),                      # fp32
    (torch.zeros(3, 1, 128, dtype=torch.float16), torch.zeros(3, 1, 128, dtype=torch.bfloat16)),
    (torch.zeros(3, 1, 128, dtype=torch.float16), None)]


def _room(c):                                   # a table whose requests need no page
    c.set_page_table(i32(0, 1, 2), i32(0, 1, 2, 3), i32(3, 1, 15))
    return c


@pytest.mark.parametrize("rows", BAD_ROWS)
@pytest.mark.parametrize("half", ["append", "append_device"])
def test_rows_that_do_not_fit_an_8_bit_cache(hip_lib, rows, half):
    c = _room(_make(torch.int8))
    before = _state(c)
    with pytest.raises(RuntimeError, match="k_new|v_new"):
        getattr(c, half)(*rows)
    assert _state(c) == before
    # rows in host memory are no rows of a cache on the GPU
    with pytest.raises(RuntimeError, match="CUDA"):
        getattr(c, half)(*(torch.zeros(3, 1, 128, dtype=torch.float16),) * 2)
    assert _state(c) == before


@pytest.mark.parametrize("rows", BAD_ROWS[:5])
def test_rows_that_do_not_fit_a_16_bit_cache(hip_lib, rows):
    c = _room(_make("paged"))
    before = _state(c)
    with pytest.raises(RuntimeError, match="k_new|v_new"):
        c.append(*rows)
    assert _state(c) == before


@pytest.mark.gpu
@pytest.mark.parametrize("rows", BAD_ROWS)
def test_a_refused_append_and_one_behind_it(dev, rows):
    c = _room(_make(torch.int8, dev))
    before = _state(c)
    with pytest.raises(RuntimeError, match="k_new|v_new"):
        c.append(*(None if r is None else r.to(dev) for r in rows))
    assert _state(c) == before
    new = torch.randn(3, 1, 128).to(torch.bfloat16).to(dev)
    c.append(new, -new)
    assert c.kv_last_page_len.tolist() == [4, 2, 16] and c._seq_lens == [4, 2, 16]
    k, v = c.read(torch.bfloat16)
    assert torch.equal(k, -v) and all(k[n - 1].any() for n in (4, 6, 22)) and torch.count_nonzero(k.abs().sum((1, 2))) == 3


@pytest.mark.gpu
def test_rows_at_odd_places_are_accepted(dev):
    # rows that 16-byte loads cannot take as they are: an odd start, an odd stride, channels apart
    x = torch.randn(3, 1, 128).half()
    wide = torch.zeros(3 * 131 + 1, dtype=torch.float16)
    wide[1:].view(3, 131)[:, :128] = x[:, 0]
    apart = torch.zeros(3, 1, 128, 2, dtype=torch.float16)
    apart[..., 1] = x
    want = None
    flat = torch.zeros(3 * 128 + 4, dtype=torch.float16)
    flat[4:] = x.flatten()
    for rows in (x.to(dev), wide.to(dev)[1:].view(3, 131)[:, :128].unflatten(1, (1, 128)), apart.to(dev)[..., 1],
                 flat.to(dev)[4:].view(3, 1, 128)):
        c = _room(_make(torch.int8, dev))
        c.append(rows, rows)
        got = [t.float().cpu() for t in c.pools]
        want = want or got
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        assert c.kv_last_page_len.tolist() == [4, 2, 16]
