"""The 8-bit cache and prefix attention where their work is cut differently: bulk calls with an odd number
of heads, parts of more than 64 pages, and scales of the logits that are zero, negative, tiny."""
import math

import pytest
import torch

import twilight_amd.kernel as K
from _quant import attention64, check_attention, decode, encode, table
from test_gpu_prefix_attn import Case

pytestmark = pytest.mark.gpu
I8, E4 = torch.int8, torch.float8_e4m3fn
F16, BF16 = torch.float16, torch.bfloat16


@pytest.mark.parametrize("fmt,Hkv", [(I8, 6), (E4, 5)])
def test_bulk_calls_with_heads_that_are_no_multiple_of_four(dev, fmt, Hkv):
    # 33000 tokens of two sets of up to four heads: 66000 sets, more than 1024 workgroups of 16
    g = torch.Generator().manual_seed(Hkv)
    lens = [20011, 0, 12989]
    T, pages = sum(lens), sum((n + 15) // 16 for n in lens) + 3
    tab, per = table(lens, torch.randperm(pages, generator=g))
    k, v = (torch.randn((T, Hkv, 128), generator=g).to(BF16) for _ in range(2))
    codes = [torch.full((pages, 16, Hkv, 128), 0x5A, dtype=torch.uint8, device=dev).view(fmt) for _ in range(2)]
    scales = [torch.full((pages, 16, Hkv), 3.0, device=dev) for _ in range(2)]
    args = [t.to(dev) for t in tab]
    indptr = torch.tensor([0, lens[0], lens[0], T], dtype=torch.int32, device=dev)
    K.kv_quant_append(k.to(dev), v.to(dev), indptr, *codes, *scales, *args)
    page = torch.cat([p[torch.arange(n) // 16] for p, n in zip(per, lens)])
    slot = torch.cat([torch.arange(n) % 16 for n in lens])
    got = K.kv_quant_read(*codes, *scales, *args, indptr, T, dtype=torch.float32)
    for i, x in enumerate((k, v)):
        c, s = encode(x, fmt)
        want = torch.full((pages, 16, Hkv, 128), 0x5A, dtype=torch.uint8)
        want[page, slot] = c.view(torch.uint8)
        assert torch.equal(codes[i].view(torch.uint8).cpu(), want)
        ws = torch.full((pages, 16, Hkv), 3.0)
        ws[page, slot] = s
        assert torch.equal(scales[i].cpu(), ws)
        assert torch.equal(got[i].cpu(), decode(c, s))


@pytest.mark.parametrize("fmt", [None, I8])
def test_streamed_parts_of_more_than_64_pages(dev, fmt):
    # 512 (request, kv head) pairs: parts of 2048 tokens, two windows of 64 page ids
    lens = [3] * 64
    lens[5], lens[63] = 2100, 1999
    if fmt is not None:
        c = Case(dev, BF16, fmt, 8, 8, lens, seed=1)
    else:
        # and 64 groups of one request each, the prefix of one of them long
        plens = [1] * 64
        plens[40] = 2333
        c = Case(dev, F16, None, 8, 8, lens, plens, [1] * 64, seed=2)
    c.check(c.call())


@pytest.mark.parametrize("fmt", [None, E4])
def test_staged_parts_of_more_than_64_pages(dev, fmt):
    # 1000 requests of 8 rows per kv head: 63 tiles of rows times 8 kv heads leave two parts of 1280
    # and 1220 tokens
    c = Case(dev, BF16, fmt, 64, 8, [b % 3 for b in range(1000)], [2500], [1000], seed=3)
    out, lse = (t.cpu() for t in c.call())
    assert torch.isfinite(out.float()).all() and torch.isfinite(lse).all()
    for b in (0, 15, 16, 517, 998, 999):
        k, v = c.seen(b)
        check_attention(out[b], lse[b], attention64(c.q[b], k, v, 128 ** -0.5), k.shape[0], BF16,
                        F16 if fmt is not None else BF16)


@pytest.mark.parametrize("fmt", [None, I8, E4])
@pytest.mark.parametrize("scale", [0.0, -0.25, 2.0 ** -40])
def test_scales_of_the_logits(dev, fmt, scale):
    # 20 and 40 rows a kv head: streamed and staged prefixes, and own tokens
    for members in (5, 10):
        c = Case(dev, BF16, fmt, 8, 2, [7] * members, [333], [members], seed=members)
        got = c.call(sm_scale=scale)
        if scale < 0:
            c.q = -c.q
        c.check(got, scale=abs(scale))
        if scale == 0:
            assert torch.allclose(got[1].cpu(), torch.full((members, 8), math.log(340)))


def test_scale_of_zero_with_large_values(dev):
    # products up to 2^100 must not survive a scale of zero; a query of zeros needs a scale of its own
    c = Case(dev, BF16, None, 4, 2, [100, 20], gain=2.0 ** 50, plens=[40], members=[2])
    c.q = (c.q.float() * 2.0 ** 50).to(BF16)
    c.check(c.call(sm_scale=0.0), scale=0.0)
    c = Case(dev, BF16, I8, 4, 2, [100, 20])
    c.q = torch.zeros_like(c.q)
    c.check(c.call(sm_scale=2.0 ** -40), scale=2.0 ** -40)


@pytest.mark.parametrize("scale", [math.inf, -math.inf, math.nan])
def test_scales_that_are_no_number_are_refused(dev, scale):
    c = Case(dev, F16, None, 4, 2, [9], [5], [1])
    with pytest.raises(RuntimeError):
        c.call(sm_scale=scale)
