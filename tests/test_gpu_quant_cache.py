"""8-bit K / V pages: what is written against the formula (codes and scales bit for bit, and each value
within half a step in 64 bits), what is read back, ragged and odd calls, rows without a place."""
import math

import pytest
import torch

import twilight_amd.kernel as K
from _quant import TOP, decode, encode, table

pytestmark = pytest.mark.gpu
FORMATS = [torch.int8, torch.float8_e4m3fn]


def _pool(pages, Hkv, fmt, dev, nhd=False):
    """Pages whose every byte is 0x5A and whose scales are 3: stale contents."""
    shape = (pages, 16, Hkv) if nhd else (pages, Hkv, 16)
    k, v = (torch.full(shape + (128,), 0x5A, dtype=torch.uint8, device=dev).view(fmt) for _ in range(2))
    ks, vs = (torch.full(shape, 3.0, device=dev) for _ in range(2))
    return [t if nhd else t.transpose(1, 2) for t in (k, v, ks, vs)]


def _bytes(t):
    return t.view(torch.uint8).cpu()


def _indptr(counts):
    p = [0]
    for c in counts:
        p.append(p[-1] + c)
    return torch.tensor(p, dtype=torch.int32)


def _run(dev, dtype, fmt, Hkv, new, old, nhd=False, extra_rows=0, seed=0, x=None):
    g = torch.Generator().manual_seed(seed)
    lens = [a + b for a, b in zip(new, old)]
    pages = sum((n + 15) // 16 for n in lens) + 2
    tab, per = table(lens, torch.randperm(pages, generator=g))
    T = sum(new) + extra_rows
    k = torch.randn((T, Hkv, 128), generator=g).to(dtype) if x is None else x
    v = (torch.randn((T, Hkv, 128), generator=g) * 37).to(dtype)
    pool = _pool(pages, Hkv, fmt, dev, nhd)
    args = [t.to(dev) for t in tab]
    K.kv_quant_append(k.to(dev), v.to(dev), _indptr(new).to(dev), *pool, *args)
    want = [t.cpu().clone() for t in _pool(pages, Hkv, fmt, "cpu", nhd)]
    t = 0
    for b, n in enumerate(new):
        for j in range(n):
            pos = old[b] + j
            page, slot = int(per[b][pos // 16]), pos % 16
            for i, rows in ((0, k), (1, v)):
                codes, scale = encode(rows[t], fmt)
                want[i].view(torch.uint8)[page, slot] = codes.view(torch.uint8)
                want[2 + i][page, slot] = scale
            t += 1
    return pool, want, args, per, k, v, lens


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("Hkv,new,old,nhd", [
    (8, [1] * 8, [0, 1, 15, 16, 17, 31, 32, 100], False),      # a decode step
    (3, [5, 0, 33, 1], [11, 4, 0, 16], False),                 # ragged, one request without new tokens
    (1, [300], [7], True),                                     # one head, heads inside the token
    (5, [2] * 40, [3] * 40, False),                            # more requests than one search step
    (2, [1] * 270, [0] * 270, True)])                          # more than two
def test_append_writes_the_formula_and_nothing_else(dev, dtype, fmt, Hkv, new, old, nhd):
    pool, want, *_ = _run(dev, dtype, fmt, Hkv, new, old, nhd, extra_rows=3)
    for got, exp in zip(pool, want):
        if got.dtype == torch.float32:
            assert torch.equal(got.cpu(), exp)
        else:
            assert torch.equal(_bytes(got), exp.view(torch.uint8))


@pytest.mark.parametrize("fmt", FORMATS)
def test_values_are_within_half_a_step(dev, fmt):
    # int8: half of the scale; e4m3: 2^-4 of the value, or half of 2^-9 scales below 2^-6 of them.
    # One fp32 rounding of x / scale can move a value across a midpoint: 2^-22 of it on top
    pool, _, args, per, k, v, lens = _run(dev, torch.bfloat16, fmt, 4, [200, 77], [0, 0], seed=3)
    kk, vv = K.kv_quant_read(*pool, *args, _indptr(lens).to(dev), sum(lens), dtype=torch.float32)
    for got, x in ((kk, k), (vv, v)):
        x, got = x.double(), got.cpu().double()
        scale = x.abs().amax(-1, keepdim=True) / TOP[fmt]
        half = scale / 2 if fmt == torch.int8 else torch.maximum(x.abs() * 2.0 ** -4, scale * 2.0 ** -10)
        assert torch.all((got - x).abs() <= half * (1 + 2.0 ** -20) + x.abs() * 2.0 ** -22)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
def test_read_back(dev, dtype, fmt):
    lens_new, old = [9, 40, 0, 1], [8, 3, 20, 0]
    pool, want, args, per, *_, lens = _run(dev, torch.bfloat16, fmt, 3, lens_new, old, seed=5)
    # whole contexts, then the last few tokens of each into given outputs with rows to spare
    for counts, spare in ((lens, 0), ([4, 17, 20, 0], 2)):
        T = sum(counts) + spare
        outs = [torch.full((T, 3, 128), 7.0, dtype=dtype, device=dev) for _ in range(2)]
        got = K.kv_quant_read(*pool, *args, _indptr(counts).to(dev), T, dtype=dtype, k_out=outs[0], v_out=outs[1])
        assert got[0] is outs[0] and got[1] is outs[1]
        for i in range(2):
            rows = []
            for b, c in enumerate(counts):
                pos = torch.arange(lens[b] - c, lens[b])
                pages = per[b][pos // 16] if c else torch.zeros(0, dtype=torch.long)
                codes = want[i].view(torch.uint8)[pages, pos % 16].view(fmt)
                rows.append(decode(codes, want[2 + i][pages, pos % 16]).to(dtype))
            exp = torch.cat(rows + [torch.full((spare, 3, 128), 7.0, dtype=dtype)])
            assert torch.equal(got[i].cpu(), exp)


@pytest.mark.parametrize("fmt", FORMATS)
def test_special_rows(dev, fmt):
    # zeros, one value, the type's extremes, subnormal numbers, infinities and NaN
    dtype = torch.bfloat16
    x = torch.zeros(8, 1, 128)
    x[1, 0, 5] = -3.0
    x[2] = torch.finfo(dtype).max
    x[2, 0, 64:] = -torch.finfo(dtype).max
    x[3] = 2.0 ** -130
    x[4, 0, 9] = math.inf
    x[5, 0, 127] = math.nan
    x[6] = torch.linspace(-1, 1, 128)
    x[7, 0, 0], x[7, 0, 1] = 1.0, 2.0 ** -20
    pool, want, args, per, *_ = _run(dev, dtype, fmt, 1, [8], [0], x=x.to(dtype))
    assert torch.equal(pool[2].cpu().isnan(), want[2].isnan())
    ok = ~want[2].isnan()
    assert torch.equal(pool[2].cpu()[ok], want[2][ok])
    assert torch.equal(_bytes(pool[0]), want[0].view(torch.uint8))
    k, _ = K.kv_quant_read(*pool, *args, _indptr([8]).to(dev), 8, dtype=torch.float32)
    k = k.cpu()
    assert torch.all(k[0] == 0) and k[1, 0, 5] == -3.0 and torch.count_nonzero(k[1]) == 1
    assert torch.all(torch.isnan(k[4])) and torch.all(torch.isnan(k[5])) and not torch.isnan(k[[0, 1, 2, 3, 6, 7]]).any()


def test_every_e4m3_value_and_midpoint(dev):
    # rows whose largest magnitude is 448 have scale 1: the codes are the type's own rounding of x.
    # All 16-bit patterns of fp16 up to 448, 127 a row
    bits = torch.arange(0, 1 << 16, dtype=torch.int32).to(torch.int16).view(torch.float16)
    bits = bits[torch.isfinite(bits) & (bits.abs() <= 448)]
    pad = (-len(bits)) % 127
    rows = torch.cat([bits, bits[:pad]]).reshape(-1, 127)
    x = torch.cat([rows, torch.full((rows.shape[0], 1), 448.0, dtype=torch.float16)], 1).unsqueeze(1)
    pool, want, *_ = _run(dev, torch.float16, torch.float8_e4m3fn, 1, [x.shape[0]], [0], x=x)
    assert torch.equal(_bytes(pool[0]), want[0].view(torch.uint8))


def test_rows_without_a_place(dev):
    # more new tokens than the request holds, a request without pages, page ids outside the cache
    fmt, Hkv = torch.int8, 2
    pool = _pool(6, Hkv, fmt, dev)
    tab = (torch.tensor([4, 99, -1], dtype=torch.int32), torch.tensor([0, 1, 1, 3], dtype=torch.int32),
           torch.tensor([3, 0, 5], dtype=torch.int32))
    args = [t.to(dev) for t in tab]
    counts = [5, 2, 21]
    k = torch.randn((sum(counts), Hkv, 128)).half()
    before = [_bytes(t).clone() for t in pool[:2]]
    K.kv_quant_append(k.to(dev), k.to(dev), _indptr(counts).to(dev), *pool, *args)
    for i in range(2):
        changed = (_bytes(pool[i]) != before[i]).flatten(2).any(-1)
        assert set(map(tuple, changed.nonzero().tolist())) <= {(4, 0), (4, 1), (4, 2)}
    got, _ = K.kv_quant_read(*pool, *args, _indptr(counts).to(dev), sum(counts), dtype=torch.float32)
    codes, scale = encode(k[2:5], fmt)
    exp = torch.zeros(sum(counts), Hkv, 128)
    exp[2:5] = decode(codes, scale)
    assert torch.equal(got.cpu(), exp)


def test_strided_rows_and_offsets_beyond_32_bits(dev):
    # rows inside a fused projection (strides of 3 * Hkv * 128), and a pool whose last page lies
    # beyond 2^32 bytes
    Hkv, fmt, dtype = 4, torch.int8, torch.bfloat16
    fused = torch.randn((6, 3 * Hkv, 128)).to(dtype).to(dev)
    pages = (1 << 32) // (16 * Hkv * 128) + 3
    k = torch.zeros((pages, 16, Hkv, 128), dtype=fmt, device=dev)
    scale = torch.zeros((pages, 16, Hkv), device=dev)
    v, vscale = torch.zeros_like(k), torch.zeros_like(scale)
    args = [t.to(dev) for t in (torch.tensor([pages - 1], dtype=torch.int32), torch.tensor([0, 1], dtype=torch.int32),
                                torch.tensor([6], dtype=torch.int32))]
    K.kv_quant_append(fused[:, Hkv:2 * Hkv], fused[:, 2 * Hkv:], _indptr([6]).to(dev), k, v, scale, vscale, *args)
    for cache, sc, rows in ((k, scale, fused[:, Hkv:2 * Hkv]), (v, vscale, fused[:, 2 * Hkv:])):
        codes, s = encode(rows.cpu(), fmt)
        assert torch.equal(cache[-1, :6].cpu(), codes) and torch.equal(sc[-1, :6].cpu(), s)
        assert not cache[:-1].any() and not cache[-1, 6:].any()
    got, _ = K.kv_quant_read(k, v, scale, vscale, *args, _indptr([6]).to(dev), 6, dtype=torch.float32)
    assert torch.equal(got.cpu(), decode(*encode(fused[:, Hkv:2 * Hkv].cpu(), fmt)))
