"""Page tables none of whose lists holds a page: the tensor of page ids has no elements."""
import math

import pytest
import torch

import twilight_amd.kernel as K
from twilight_amd.cache import QuantPagedKVCache
from test_gpu_prefix_attn import Case
from test_operators_host import _attn

BF16, F16, I8 = torch.bfloat16, torch.float16, torch.int8


def test_page_ids_are_needed_where_there_are_pages(hip_lib):
    # null ids get past the null check where the bound is 0: what is refused there is the query's alignment
    c = lambda **kw: _attn(hip_lib, q=0x1008, **kw)  # noqa: E731
    assert c() == -4
    assert c(ids=0) == -1 and c(pids=0) == -1 and c(ids=0, mp=0) == -1 and c(pids=0, mt=0) == -1
    assert c(ids=0, mt=0) == -4 and c(pids=0, mp=0) == -4 and c(ids=0, pids=0, mt=0, mp=0) == -4
    assert c(ids=0, mt=0, groups=0) == -4 and c(pids=0, groups=0) == -4
    assert c(ptr=0, mt=0) == -1 and c(pptr=0, mp=0) == -1


def _bare(c):
    """The tables of a Case without the element that stands in for no page id."""
    cut = lambda t: (t[0][:int(t[1][-1])],) + tuple(t[1:])  # noqa: E731
    c.table = cut(c.table)
    if c.plens:
        c.ptable = cut(c.ptable)
    return c


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", [None, I8])
@pytest.mark.parametrize("max_tokens", [None, 40, 3000])
def test_samples_without_tokens_of_their_own(dev, fmt, max_tokens):
    # the first step behind a shared prompt
    c = _bare(Case(dev, BF16, fmt, 8, 2, [0] * 5, [333, 20], [3, 2]))
    assert c.table[0].numel() == 0
    c.check(c.call(max_tokens=max_tokens))
    need = K.prefix_attention_workspace_bytes(5, 8, 2, 2, 333, 3, max_tokens or 0)
    c.check(c.call(max_tokens=max_tokens, workspace=torch.empty(need, dtype=torch.uint8, device=dev)))


@pytest.mark.gpu
@pytest.mark.parametrize("max_prefix_tokens", [0, 100])
def test_prefixes_without_tokens(dev, max_prefix_tokens):
    c = _bare(Case(dev, F16, I8, 8, 2, [20, 0, 3], [0, 0], [2, 1]))
    assert c.ptable[0].numel() == 0
    c.check(c.call(max_prefix_tokens=max_prefix_tokens))


@pytest.mark.gpu
@pytest.mark.parametrize("max_tokens", [1, 5000])
def test_nothing_at_all(dev, max_tokens):
    c = _bare(Case(dev, F16, I8, 4, 2, [0, 0]))
    out, lse = c.call(max_tokens=max_tokens)
    assert not out.any() and torch.all(lse == -math.inf)
    c = _bare(Case(dev, BF16, None, 4, 2, [0, 0], [0], [2]))
    out, lse = c.call(max_tokens=max_tokens, max_prefix_tokens=7)
    assert not out.any() and torch.all(lse == -math.inf)


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", [I8, torch.float8_e4m3fn])
def test_an_8_bit_cache_without_tokens(dev, fmt):
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device=dev)  # noqa: E731
    c = QuantPagedKVCache(2, 3, fmt, dev)
    c.set_page_table(i32(), i32(0, 0, 0), i32(0, 0))
    rows = torch.randn(4, 3, 128, device=dev).half()
    K.kv_quant_append(rows, rows, i32(0, 1, 3), *c.pools, *c.table)           # no place: skipped
    assert not c.k_cache.float().any() and not c.k_scale.any()
    outs = [torch.full((4, 3, 128), 7.0, dtype=BF16, device=dev) for _ in range(2)]
    for x in K.kv_quant_read(*c.pools, *c.table, i32(0, 1, 3), 4, k_out=outs[0], v_out=outs[1]):
        assert not x[:3].any() and torch.all(x[3:] == 7.0)                     # rows behind the last request stay
    k, v = c.read()
    assert k.shape == v.shape == (0, 3, 128)
