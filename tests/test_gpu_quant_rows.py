"""New rows of the 8-bit cache whose strides differ in a dimension of one element, where a stride means nothing."""
import pytest
import torch

import twilight_amd.kernel as K
from twilight_amd.cache import QuantPagedKVCache
from _quant import decode, encode

pytestmark = pytest.mark.gpu
i32 = lambda *v: torch.tensor(v, dtype=torch.int32)  # noqa: E731


@pytest.mark.parametrize("fmt", [torch.int8, torch.float8_e4m3fn])
@pytest.mark.parametrize("T,Hkv,strides", [(1, 4, (1536, 128)), (1, 4, (1531, 128)), (3, 1, (128, 77)), (1, 1, (3, 5)),
                                           (1, 1, (0, 0))])
def test_strides_of_single_rows_and_heads(dev, fmt, T, Hkv, strides):
    g = torch.Generator().manual_seed(T + Hkv)
    k, v = (torch.randn(T, Hkv, 128, generator=g).to(torch.bfloat16) for _ in range(2))
    odd = torch.zeros(8192, dtype=torch.bfloat16, device=dev).as_strided((T, Hkv, 128), (*strides, 1))
    odd.copy_(v)
    c = QuantPagedKVCache(3, Hkv, fmt, dev)
    c.set_page_table(i32(1), i32(0, 1), i32(T))
    for one, two in ((k.to(dev), odd), (odd, k.to(dev))):
        K.kv_quant_append(one, two, i32(0, T).to(dev), *c.pools, *c.table)
        got = K.kv_quant_read(*c.pools, *c.table, i32(0, T).to(dev), T, dtype=torch.float32)
        for x, y in zip(got, (one, two)):
            assert torch.equal(x.cpu(), decode(*encode(y.cpu(), fmt)))


def test_one_request_of_a_fused_projection(dev):
    # K rotated into rows of its own, V still inside [1, q heads + 2 kv heads, 128]
    Hkv = 4
    v = torch.randn(1, 8 + 2 * Hkv, 128).half().to(dev)[:, -Hkv:]
    k = torch.randn(1, Hkv, 128).half().to(dev)
    assert v.stride(0) != k.stride(0)
    c = QuantPagedKVCache(3, Hkv, torch.int8, dev)
    c.set_page_table(i32(1), i32(0, 1), i32(2))
    c.append(k, v)
    K.kv_quant_append(k, v, i32(0, 1).to(dev), *c.pools, *c.table)
    got = c.read(torch.float32)
    for x, y in zip(got, (k, v)):
        assert torch.equal(x[-1:].cpu(), decode(*encode(y.cpu(), torch.int8)))


def test_strides_that_count_still_have_to_agree(dev):
    c = QuantPagedKVCache(3, 2, torch.int8, dev)
    c.set_page_table(i32(1), i32(0, 1), i32(4))
    x = torch.zeros(2, 2, 256, dtype=torch.float16, device=dev)
    with pytest.raises(RuntimeError, match="strides"):
        K.kv_quant_append(x[..., :128], x[..., :128].contiguous(), i32(0, 2).to(dev), *c.pools, *c.table)
