"""Decode attention over 8-bit pages and with shared prefixes against attention in 64 bits on the values
the pages hold; the bounds are derived in ``_quant.check_attention``."""
import math

import pytest
import torch

import twilight_amd.kernel as K
from _quant import attention64, check_attention, decode, encode, table, tokens_of

pytestmark = pytest.mark.gpu
I8, E4 = torch.int8, torch.float8_e4m3fn
F16, BF16 = torch.float16, torch.bfloat16


class Case:
    """Random pages with stale NaN in every slot no request owns, requests, groups and their tables."""

    def __init__(self, dev, dtype, fmt, H, Hkv, lens, plens=(), members=(), seed=0, nhd=False, gain=1.0, vgain=None):
        g = torch.Generator().manual_seed(seed)
        self.dev, self.dtype, self.fmt, self.H, self.Hkv, self.lens = dev, dtype, fmt, H, Hkv, list(lens)
        self.plens, self.members = list(plens), list(members)
        total = sum((n + 15) // 16 for n in self.lens + self.plens) + 1
        ids = torch.randperm(total, generator=g)
        self.table, self.per = table(self.lens, ids)
        used = sum(len(p) for p in self.per)
        self.ptable, self.pper = table(self.plens, ids[used:])
        x = torch.randn((2, total, 16, Hkv, 128), generator=g) * gain
        if vgain is not None:
            x[1] *= torch.exp2(torch.randint(-vgain, vgain + 1, (total, 16, Hkv, 1), generator=g).float())
        owned = torch.zeros(total, 16, dtype=torch.bool)
        for n, p in list(zip(self.lens, self.per)) + list(zip(self.plens, self.pper)):
            for t in range(n):
                owned[p[t // 16], t % 16] = True
        self.scales = [None, None]
        if fmt is None:
            x = x.to(dtype)
            self.values = [x[0].double(), x[1].double()]
            x[:, ~owned] = math.nan
            self.pools = [x[0].to(dev), x[1].to(dev)]
        else:
            self.pools, self.values = [], []
            for i in range(2):
                codes, scale = encode(x[i], fmt)
                self.values.append(decode(codes, scale).double())
                codes.view(torch.uint8)[~owned] = 0x7F          # NaN in e4m3
                scale[~owned] = math.nan
                if not nhd:
                    codes, scale = (t.transpose(1, 2).contiguous().transpose(1, 2) for t in (codes, scale))
                self.pools.append(codes.to(dev))
                self.scales[i] = scale.to(dev)
        self.q = torch.randn((len(self.lens), H, 128), generator=g).to(dtype)

    def indptr(self):
        p = [0]
        for m in self.members:
            p.append(p[-1] + m)
        return torch.tensor(p, dtype=torch.int32)

    def call(self, max_tokens=None, **kw):
        d = lambda ts: [t.to(self.dev) for t in ts]  # noqa: E731
        n = max(self.lens) if max_tokens is None else max_tokens
        q = kw.pop("q", self.q).to(self.dev)
        if not self.plens:
            return K.quant_paged_decode_attention(q, *self.pools, *self.scales, *d(self.table),
                                                  max_tokens=max(n, 1), return_lse=True, **kw)
        kw = {"max_prefix_tokens": max(self.plens), "max_group_size": max(self.members), **kw}
        return K.prefix_paged_decode_attention(q, *self.pools, *d(self.ptable), self.indptr().to(self.dev), *d(self.table),
                                               max_tokens=n, k_scale=self.scales[0], v_scale=self.scales[1],
                                               return_lse=True, **kw)

    def seen(self, b, max_tokens=1 << 30, max_prefix=1 << 30):
        n = min(self.lens[b], max_tokens)
        parts = [[tokens_of(v, self.per[b], n)] for v in self.values]
        at = 0
        for g, m in enumerate(self.members):
            if at <= b < at + m:
                np = min(self.plens[g], max_prefix)
                for part, v in zip(parts, self.values):
                    part.insert(0, tokens_of(v, self.pper[g], np))
            at += m
        return [torch.cat(p) for p in parts]

    def check(self, got, scale=128 ** -0.5, **bounds):
        out, lse = got[0].cpu(), got[1].cpu()
        for b in range(len(self.lens)):
            k, v = self.seen(b, **bounds)
            check_attention(out[b], lse[b], attention64(self.q[b], k, v, scale), k.shape[0], self.dtype,
                            F16 if self.fmt is not None else self.dtype)


@pytest.mark.parametrize("fmt", [I8, E4])
@pytest.mark.parametrize("dtype,H,Hkv,lens,nhd", [
    (BF16, 8, 2, [777, 1, 0, 16, 33], False),        # lengths from none, pages that end inside a tile
    (F16, 4, 4, [1, 2, 15, 17, 31, 32, 33, 47], True),
    (BF16, 3, 3, [129, 128, 127, 255], False),       # parts that end at a tile and inside one
    (F16, 20, 1, [500, 3], False),                   # more q heads than one tile of rows
    (BF16, 35, 5, [70], True),                       # seven q heads per kv head
    (F16, 32, 8, [2100, 0, 4000], False)])           # several parts
def test_quant_attention(dev, dtype, fmt, H, Hkv, lens, nhd):
    c = Case(dev, dtype, fmt, H, Hkv, lens, nhd=nhd, seed=len(lens))
    c.check(c.call())


@pytest.mark.parametrize("fmt", [None, I8, E4])
@pytest.mark.parametrize("dtype,H,Hkv,plens,members,lens", [
    (F16, 4, 4, [100], [3], [5, 0, 17]),                        # up to 16 rows a kv head
    (BF16, 8, 2, [333, 31], [5, 2], [1, 2, 3, 0, 40, 0, 129]),  # two groups, 20 rows
    (F16, 8, 1, [700], [6], [33] * 6),                          # 48 rows
    (BF16, 8, 2, [260, 0, 1], [25, 1, 2], [3] * 28),            # 100 rows; an empty prefix; one token
    (F16, 4, 1, [1300], [40], [7, 0] * 20),                     # 160 rows
    (BF16, 8, 1, [511], [37], [1] * 37),                        # 296 rows: a second tile of rows
    (F16, 2, 2, [48, 64], [0, 3], [0, 16, 40])])                # a group without requests
def test_prefix_attention(dev, dtype, fmt, H, Hkv, plens, members, lens):
    c = Case(dev, dtype, fmt, H, Hkv, lens, plens, members, seed=len(lens))
    c.check(c.call())


def test_prefix_alone_and_requests_outside_groups(dev):
    c = Case(dev, F16, None, 4, 2, [0, 0, 0], [70], [3])
    c.check(c.call(max_tokens=0))                               # no own tokens at all: one part
    c = Case(dev, F16, None, 4, 2, [0, 5, 20, 3], [70], [2])    # requests 2 and 3 belong to no group
    c.check(c.call())
    c = Case(dev, BF16, I8, 4, 2, [0, 9], [0], [2])             # an empty prefix and an empty request
    c.check(c.call(max_prefix_tokens=0))
    c.check(c.call(max_prefix_tokens=0, max_tokens=9))


def test_bounds_cut_what_is_attended_to(dev):
    c = Case(dev, BF16, I8, 4, 2, [300, 20], [500], [2])
    c.check(c.call(max_tokens=100, max_prefix_tokens=333), max_tokens=100, max_prefix=333)
    # members beyond max_group_size see their own tokens only
    got = c.call(max_group_size=1)
    c.members = [1]
    c.check(got)


@pytest.mark.parametrize("fmt", [None, I8, E4])
def test_rows_that_rescale_and_scales_of_all_sizes(dev, fmt):
    # logits that grow along the row (every tile raises the maximum) and V rows that differ by 2^24
    c = Case(dev, BF16, fmt, 4, 2, [400, 90], seed=9, vgain=12, **({} if fmt is not None else dict(plens=[64], members=[2])))
    c.check(c.call())
    big = c.q.float() * 12
    c.q = big.to(BF16)
    c.check(c.call())


@pytest.mark.parametrize("gain", [2.0 ** -60, 2.0 ** 40])
def test_scales_far_from_one(dev, gain):
    # bf16 values outside fp16's range: K and V scales of 2^-66 and 2^34, a query that makes up for K
    c = Case(dev, BF16, I8, 4, 2, [200, 33], gain=gain)
    c.q = (c.q.float() / gain).to(BF16)
    got = c.call()
    assert torch.isfinite(got[0]).all()
    c.check(got)


def test_infinite_and_nan_tokens_stay_in_their_request(dev):
    c = Case(dev, F16, None, 4, 2, [40, 40, 40], [50], [2])
    clean = c.call()
    c.pools[1][c.per[0][1], 3, :, 7] = math.inf                 # a visible V of request 0
    c.pools[0][c.per[1][0], 2] = math.nan                       # a visible K of request 1
    out, lse = c.call()
    assert torch.isinf(out[0, :, 7]).all() and torch.isfinite(out[0, :, :7]).all()
    assert torch.isnan(out[1]).all() and torch.isnan(lse[1]).all()
    assert torch.equal(out[2], clean[0][2]) and torch.equal(lse[2], clean[1][2])


def test_workspace_out_scale_and_repeat(dev):
    c = Case(dev, BF16, E4, 8, 2, [900, 40], [600], [2])
    need = K.prefix_attention_workspace_bytes(2, 8, 2, 1, 600, 2, 900)
    ws = torch.full((need,), 0xFF, dtype=torch.uint8, device=dev)      # NaN everywhere
    out = torch.full((2, 8, 128), math.nan, dtype=BF16, device=dev)
    first = c.call(workspace=ws, out=out, sm_scale=0.03)
    assert first[0] is out
    c.check(first, scale=0.03)
    second = c.call(workspace=ws, sm_scale=0.03)                       # the call's own leftovers
    assert torch.equal(first[0], second[0]) and torch.equal(first[1], second[1])
    with pytest.raises(RuntimeError, match="workspace"):
        c.call(workspace=ws[:need - 1])


def test_page_ids_outside_the_cache_read_the_last_page(dev):
    c = Case(dev, F16, I8, 2, 2, [40])
    last = c.pools[0].shape[0] - 1
    c.values = [v.clone() for v in c.values]
    c.per[0][1] = last
    for i in range(2):                                                  # the last page is nobody's: fill it
        codes, scale = encode(torch.randn(16, 2, 128), I8)
        c.pools[i][last], c.scales[i][last] = codes.to(dev), scale.to(dev)
        c.values[i][last] = decode(codes, scale).double()
    want = c.table[0].clone()
    for bad in (last + 1, -1, 2 ** 31 - 1):
        ids = want.clone()
        ids[1] = bad
        c.table = (ids,) + tuple(c.table[1:])
        c.check(c.call())


def test_offsets_beyond_32_bits(dev):
    # the request's pages are the last ones of pools of more than 2^32 bytes each
    Hkv = 8
    pages = (1 << 32) // (16 * Hkv * 128) + 5
    k, v = (torch.zeros((pages, Hkv, 16, 128), dtype=I8, device=dev).transpose(1, 2) for _ in range(2))
    ks, vs = (torch.ones((pages, Hkv, 16), device=dev).transpose(1, 2) for _ in range(2))
    x = torch.randn(2, 4, 16, Hkv, 128)
    vals = []
    for t, s, y in ((k, ks, x[0]), (v, vs, x[1])):
        codes, scale = encode(y, I8)
        t[-4:], s[-4:] = codes.to(dev), scale.to(dev)
        vals.append(decode(codes, scale).double())
    ids = torch.tensor([pages - 1, pages - 3, pages - 4, pages - 2], dtype=torch.int32)
    q = torch.randn(1, 16, 128).half()
    out, lse = K.quant_paged_decode_attention(q.to(dev), k, v, ks, vs, ids.to(dev),
                                              torch.tensor([0, 4], dtype=torch.int32).to(dev),
                                              torch.tensor([9], dtype=torch.int32).to(dev), 57, return_lse=True)
    order = ids.long() - (pages - 4)
    kk, vv = (tokens_of(t, order, 57) for t in vals)
    check_attention(out[0].cpu(), lse[0].cpu(), attention64(q[0], kk, vv, 128 ** -0.5), 57, F16, F16)
