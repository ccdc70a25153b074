"""Decode attention where a few tokens take nearly all of the softmax and the answer comes from the others:
dominant tokens whose V is zero or small, and V rows of very different size, attended to or not.

Bounds. The rows are compared with attention in 64 bits on the values the pages hold, element by element and
relative to the sum of p |v| that the element is made of. A weight that enters an fp16 product is off by half
a step (2^-11 of it); below fp16's normal range by 2^-25 of the product's unit, but never by more than
itself. The largest weight that a wavefront has seen is at least 2^12 units, so that 2^-25 is 2^-37 of it.
Over 8-bit pages the weight is taken times its V scale relative to a power of two that is less than twice
the largest V scale seen: 2^-36 of the largest weight times that scale. Logits are fp32 sums of 128 exact
products (130 * 2^-24 of their summed magnitudes, in numerator and denominator), sums of n terms and exp2
(n + 64) * 2^-24, the output's own rounding half a step."""
import math

import pytest
import torch

from _quant import HALF_STEP, decode, encode
from test_gpu_prefix_attn import Case

pytestmark = pytest.mark.gpu
I8, E4 = torch.int8, torch.float8_e4m3fn
F16, BF16 = torch.float16, torch.bfloat16


class Sink(Case):
    """One kv head whose query reads channel 0 of K only: token ``at`` has a logit ``gap`` (nats) above all
    others. ``vsize[t]`` is the size of token t's V. Several ``samples`` share the tokens as a prefix."""

    def __init__(self, dev, dtype, fmt, H, n, gap, vsize, at=3, samples=1, seed=0):
        prefix = dict(plens=[n], members=[samples], lens=[0] * samples) if fmt is None or samples > 1 else dict(lens=[n])
        super().__init__(dev, dtype, fmt, H, 1, seed=seed, **prefix)
        per = (self.pper if self.plens else self.per)[0]
        g = torch.Generator().manual_seed(seed + 1)
        k = torch.randn(n, 1, 128, generator=g)
        k[:, :, 0] = 0.0
        k[at, :, 0] = 4.0
        v = (1 + torch.rand(n, 1, 128, generator=g)) * torch.as_tensor(vsize).float().reshape(-1, 1, 1)
        self.q = torch.zeros(len(self.lens), H, 128)
        self.q[:, :, 0] = gap * math.sqrt(128) / 4
        self.q = self.q.to(dtype)
        page, slot = per[torch.arange(n) // 16], torch.arange(n) % 16
        for i, x in enumerate((k, v)):
            if fmt is None:
                self.pools[i][page, slot] = x.to(dtype).to(dev)
                self.values[i][page, slot] = x.to(dtype).double()
            else:
                codes, scale = encode(x, fmt)
                self.pools[i].view(torch.uint8)[page, slot] = codes.view(torch.uint8).to(dev)
                self.scales[i][page, slot] = scale.to(dev)
                self.values[i][page, slot] = decode(codes, scale).double()


def scales_seen(c, b):
    """V scales [n, Hkv] of the tokens that request b sees (ones over 16-bit pages)."""
    if c.fmt is None:
        return torch.ones(c.seen(b)[0].shape[:2], dtype=torch.float64)
    pool = c.scales[1].cpu().double()
    parts, at = [pool[c.per[b]].flatten(0, 1)[:c.lens[b]]], 0
    for g, m in enumerate(c.members):
        if at <= b < at + m:
            parts.insert(0, pool[c.pper[g]].flatten(0, 1)[:c.plens[g]])
        at += m
    return torch.cat(parts)


def check_small(c, got, scale=128 ** -0.5):
    out = got[0].cpu().double()
    G = c.H // c.Hkv
    half, unit = 2.0 ** -11, (2.0 ** -36 if c.fmt is not None else 2.0 ** -37)
    if c.fmt is None and c.dtype == BF16:
        half, unit = 2.0 ** -8, 0.0
    for b in range(len(c.lens)):
        keys, values = c.seen(b)
        sizes, n = scales_seen(c, b), keys.shape[0]
        if n == 0:
            assert not out[b].any()
            continue
        for h in range(c.Hkv):
            k, v, vs = keys[:, h], values[:, h], sizes[:, h]               # [n, 128], [n]
            q = c.q[b, h * G:(h + 1) * G].double()
            p = torch.softmax(torch.matmul(q, k.T.contiguous()) * scale, -1)   # [G, n]
            ref, mag = torch.matmul(p, v), torch.matmul(p, v.abs())
            dz = 130 * 2.0 ** -24 * (torch.matmul(q.abs(), k.abs().T.contiguous()) * scale).amax(-1, keepdim=True)
            lost = unit * p.amax(-1, keepdim=True) * vs.max() / vs         # per weight
            floor = torch.matmul(torch.minimum(p, lost), v.abs())
            rel = half + 2 * dz + (n + 64) * 2.0 ** -24
            bound = rel * mag + floor
            bound = bound + HALF_STEP[c.dtype] * (ref.abs() + bound) + (2.0 ** -25 if c.dtype == F16 else 0.0) + 1e-30
            err = (out[b, h * G:(h + 1) * G] - ref).abs()
            assert torch.all(err <= bound), f"off by {(err / bound).max():.2f} bounds, {(err / mag).max():.4f} of sum p|v|"


@pytest.mark.parametrize("samples", [1, 5, 12])         # 4 rows are streamed; 20 and 48 go through LDS
@pytest.mark.parametrize("fmt", [None, I8, E4])
@pytest.mark.parametrize("gap", [12.0, 17.5, 18.5, 20.0])
def test_dominant_token_without_a_value(dev, fmt, gap, samples):
    # 17.5 nats are 2^-25.2, where weights relative to the largest one leave fp16. V of 2^20 keeps an fp16 answer
    # in its normal range
    n = 1500
    v = torch.full((n,), 2.0 ** 10 if fmt is None else 2.0 ** 20)
    v[3] = 0.0
    c = Sink(dev, F16, fmt, 4, n, gap, v, samples=samples)
    check_small(c, c.call())


@pytest.mark.parametrize("samples", [1, 5])
@pytest.mark.parametrize("fmt", [I8, E4])
@pytest.mark.parametrize("gap,big", [(11.5, 8), (12.5, 8), (18.0, 0), (12.0, 20)])
def test_values_of_very_different_size(dev, fmt, gap, big, samples):
    # a dominant token with a small V, and one token of weight e^-gap like the rest whose V is 2^big times theirs, in
    # the same tile
    n = 1024
    v = torch.full((n,), 1.0)
    v[3], v[20] = 2.0 ** -18, 2.0 ** big
    c = Sink(dev, BF16, fmt, 4, n, gap, v, samples=samples)
    check_small(c, c.call())


@pytest.mark.parametrize("samples", [1, 5])
@pytest.mark.parametrize("fmt", [I8, E4])
@pytest.mark.parametrize("big", [8, 16, 22])
def test_answer_made_of_small_values_beside_a_large_one_nobody_attends_to(dev, fmt, big, samples):
    # all tokens weigh the same but token 3 (e^-18) whose V is 2^big times the others'
    n = 1024
    v = torch.full((n,), 1.0)
    v[3] = 2.0 ** big
    c = Sink(dev, BF16, fmt, 4, n, -18.0, v, samples=samples)
    check_small(c, c.call())


@pytest.mark.parametrize("samples", [1, 5, 12])
@pytest.mark.parametrize("fmt", [I8, E4])
@pytest.mark.parametrize("down", [12, 20, 24])
def test_query_channels_of_very_different_size(dev, fmt, down, samples):
    # a bf16 query whose largest channel meets zeros in K, so that the logits come from channels 2^down smaller:
    # each of them keeps its 8 bits, so that the bounds are those of any other query
    prefix = dict(plens=[300], members=[samples], lens=[7] * samples) if samples > 1 else dict(lens=[300])
    c = Case(dev, BF16, fmt, 8, 2, seed=down, **prefix)
    c.pools[0].view(torch.uint8)[..., 0] = 0
    c.values[0][..., 0] = 0.0
    q = c.q.float() * 2.0 ** -down
    q[:, :, 0] = 1.5
    c.q = q.to(BF16)
    c.check(c.call(sm_scale=2.0 ** down * 128 ** -0.5), scale=2.0 ** down * 128 ** -0.5)


@pytest.mark.parametrize("samples", [1, 5])
@pytest.mark.parametrize("fmt", [I8, E4])
def test_tiny_queries_over_huge_keys(dev, fmt, samples):
    # K scales of 2^103 and a query that makes up for them: products stay below fp32's largest number
    prefix = dict(plens=[200], members=[samples], lens=[7] * samples) if samples > 1 else dict(lens=[200])
    c = Case(dev, BF16, fmt, 8, 2, gain=2.0 ** 108, seed=1, **prefix)
    c.q = (c.q.float() * 2.0 ** -108).to(BF16)
    got = c.call()
    assert torch.isfinite(got[0]).all()
    c.check(got)


@pytest.mark.parametrize("fmt", [I8, E4])
@pytest.mark.parametrize("prefix", [False, True])
@pytest.mark.parametrize("gain", [1, 12])
def test_random_rows_whose_values_differ_by_powers_of_two(dev, fmt, prefix, gain):
    # V rows of 2^-12 to 2^12, flat and peaked weights, streamed parts and parts through LDS
    more = dict(plens=[300, 64], members=[6, 1]) if prefix else {}
    c = Case(dev, BF16, fmt, 8, 2, [400, 90, 1, 33, 0, 170, 16], seed=9, vgain=12, **more)
    c.q = (c.q.float() * gain).to(BF16)
    check_small(c, c.call())


@pytest.mark.parametrize("samples", [1, 5, 12])
@pytest.mark.parametrize("fmt", [I8, E4])
def test_large_values_of_one_sign(dev, fmt, samples):
    # V around 2^112 over 3000 tokens of equal weight: sums of weights times V stay below fp32's largest number
    n = 3000
    c = Sink(dev, BF16, fmt, 4, n, 0.0, torch.full((n,), 2.0 ** 112), samples=samples)
    got = c.call()
    assert torch.isfinite(got[0]).all()
    check_small(c, got)
    assert torch.allclose(got[1].cpu(), torch.full((len(c.lens), 4), math.log(n)))


@pytest.mark.parametrize("samples", [1, 5])
@pytest.mark.parametrize("fmt", [None, I8])
@pytest.mark.parametrize("e", [4, 10, 15, 20, 23, 24, 25, 26, 27])
def test_logits_of_all_sizes(dev, fmt, e, samples):
    # logits around 2^e in base 2, where fp32's steps grow to 16: every third token has the largest one, the others lie
    # 2^-9 of it below, which from e = 15 on leaves them nothing
    n = 500
    c = Sink(dev, F16, fmt, 4, n, 1.0, torch.ones(n), samples=samples)
    per = (c.pper if c.plens else c.per)[0]
    page, slot = per[torch.arange(n) // 16], torch.arange(n) % 16
    k = torch.zeros(n, 1, 128)
    k[:, 0, 0] = torch.where(torch.arange(n) % 3 == 0, 1.0, 1.0 - 2.0 ** -9)
    if fmt is None:
        c.pools[0][page, slot] = k.half().to(dev)
        c.values[0][page, slot] = k.double()
    else:
        codes, scale = encode(k, fmt)
        c.pools[0][page, slot], c.scales[0][page, slot] = codes.to(dev), scale.to(dev)
        c.values[0][page, slot] = decode(codes, scale).double()
    c.q[:] = 0
    c.q[:, :, 0] = 1.0
    out, lse = c.call(sm_scale=2.0 ** e * math.log(2))
    assert torch.isfinite(out).all() and torch.isfinite(lse).all()
    if e >= 15:
        for b in range(len(c.lens)):
            v = c.seen(b)[1][::3, 0]                    # [n / 3, 128], equal weights
            err = (out[b].cpu().double() - v.mean(0)).abs()
            assert torch.all(err <= 2.0 ** -10 * v.abs().mean(0))
    else:
        check_small(c, (out, lse), scale=2.0 ** e * math.log(2))
