"""Rows whose nucleus ends exactly on a border: the token drawn does not depend on how many rows are drawn at
once, nor on where in the vocabulary the tokens stand.

Weights are held as multiples of 2^-45. With logits 0 and -a at temperature T, a and T integers whose quotient
is within 2e-14 of ln 2, the second weight is 2^44 such units to within a fraction of one: held, it is exactly
one half. Sums of such weights meet the border exactly, so that the answer follows by hand, while their
real numbers (and anything computed from rounded sums) lie beside it."""
import math
from fractions import Fraction

import pytest
import torch

import twilight_amd.kernel as K

pytestmark = pytest.mark.gpu


def _halves():
    """(a, T), exact in fp32, with a / T in ln 2 - 2e-14 .. ln 2 - 1e-15: the weight is a little above a half."""
    ln2 = Fraction(0)
    for n in range(1, 120):                             # sum of 1 / (n 2^n)
        ln2 += Fraction(1, n * 2 ** n)
    p0, q0, p1, q1, x = 0, 1, 1, 0, ln2
    found = []
    while q1 < 1 << 24:
        t = x.numerator // x.denominator
        for j in range(1, t + 1):                       # the convergent and what lies before it
            p, q = p0 + j * p1, q0 + j * q1
            if p < 1 << 23 and q < 1 << 24 and 1e-15 < float(ln2 - Fraction(p, q)) < 2e-14:
                found.append((p, q))
        p0, q0, p1, q1 = p1, q1, p0 + t * p1, q0 + t * q1
        if x == t:
            break
        x = 1 / (x - t)
    return [(p * m, q * m) for p, q in found for m in (1, 2) if q * m < 1 << 24] or found


HALVES = _halves()
LAST = 1.0 - 2.0 ** -24                                 # u that draws the last kept token in the vocabulary


def test_there_are_such_temperatures():
    assert HALVES
    for a, t in HALVES:
        assert float(torch.tensor(a, dtype=torch.float32)) == a and float(torch.tensor(t, dtype=torch.float32)) == t
        assert 0.5 < math.exp(-a / t) < 0.5 + 2 ** -46


def _draw(dev, x, rows, T, **kw):
    u = torch.full((rows,), LAST, device=dev)
    return K.sample_tokens(x.to(dev).expand(rows, -1).contiguous(), u, temperature=float(T), **kw).tolist()


@pytest.mark.parametrize("rows", [1, 3, 100, 300, 600])  # slices of 4096, 8192 and 16384 tokens
@pytest.mark.parametrize("ones,spread", [(300, False), (300, True), (2600, False), (2600, True)])
def test_the_border_is_met_exactly(dev, rows, ones, spread):
    # `ones` tokens of weight 1 and m of a half: p = 1/2 is reached by all ones and m / 2 - ones halves
    halves = 2 * ones if ones == 2600 else 8000          # 2600: the ones alone reach it, at the border of two bins
    V = ones + halves
    at = torch.arange(0, V, V // ones)[:ones] if spread else torch.arange(ones)
    half = torch.ones(V, dtype=torch.bool)
    half[at] = False
    kept = halves // 2 - ones
    last = max(int(at[-1]), int(half.nonzero()[kept - 1]) if kept else -1)
    for a, T in HALVES:
        x = torch.zeros(1, V)
        x[0, half] = -float(a)
        assert _draw(dev, x, rows, T, top_p=0.5) == [last] * rows
        # a filter that lets all of them pass changes nothing
        assert _draw(dev, x, rows, T, top_p=0.5, min_p=0.25) == [last] * rows
        # and one that lets the halves fall is applied behind the nucleus
        assert _draw(dev, x, rows, T, top_p=0.5, min_p=0.75) == [int(at[-1])] * rows


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V", [20000, 50001, 128256])
def test_a_row_alone_and_in_a_batch(dev, dtype, V):
    # rows of one batch, and each of them alone and in a batch of another size: the same tokens. u and p spread
    # over their ranges
    g = torch.Generator().manual_seed(V)
    rows = 640 if V == 20000 else 160
    x = (torch.randn(rows, V, generator=g) * 2.5).to(dtype).to(dev)
    u = torch.rand(rows, generator=g).to(dev)
    p = (0.05 + 0.94 * torch.rand(rows, generator=g)).to(dev)
    m = (0.02 * torch.rand(rows, generator=g)).to(dev)
    for kw in (dict(top_p=p), dict(top_p=p, min_p=m), dict(top_p=p, top_k=torch.full((rows,), 3000, dtype=torch.int32, device=dev))):
        cut = lambda a, b: {k: v[a:b].contiguous() for k, v in kw.items()}  # noqa: E731
        want = K.sample_tokens(x, u, **kw)
        some = torch.cat([K.sample_tokens(x[b:b + 1], u[b:b + 1], **cut(b, b + 1)) for b in range(40)])
        assert torch.equal(some, want[:40])
        some = torch.cat([K.sample_tokens(x[b:b + 33], u[b:b + 33], **cut(b, b + 33)) for b in range(0, 132, 33)])
        assert torch.equal(some, want[:132])


@pytest.mark.parametrize("T", [1e-30, 1e-19, 1e-10, 1e10, 1e19, 1e38, math.inf])
@pytest.mark.parametrize("rows", [1, 600])
def test_temperatures_of_all_sizes(dev, T, rows):
    # logits in steps of the temperature (where fp32 holds them): weights 1, e^-1, .. beside masked tokens and one
    # far below; at an infinite temperature all weigh the same, but the masked ones
    step = min(T, 1e37) if T < 1e37 else 0.0
    x = torch.full((1, 9000), -math.inf)
    x[0, 4000:4040] = -step * torch.arange(40).float()
    x[0, 8999] = -3e38
    flat = step == 0.0 and T == math.inf
    far = math.exp(-3e38 / T) if T < math.inf else 1.0
    w = [1.0 if step == 0.0 else math.exp(float(x[0, 4000 + i]) / float(torch.tensor(T))) for i in range(40)] + [far]
    total = math.fsum(w)
    for p in (0.5, 0.8, 0.97):
        goal, run, n = float(torch.tensor(p)) * total, 0.0, 0
        while run < goal:
            run += w[n]
            n += 1
        assert abs(run - goal) > 1e-6 and abs(run - w[n - 1] - goal) > 1e-6       # no case at a border
        want = 4000 + n - 1 if n <= 40 else 8999
        t = torch.full((rows,), T, device=dev)
        got = K.sample_tokens(x.to(dev).expand(rows, -1).contiguous(), torch.full((rows,), LAST, device=dev), temperature=t,
                              top_p=p)
        assert got.tolist() == [want] * rows, (p, flat)


@pytest.mark.parametrize("below", [14, 18, 20, 24])
@pytest.mark.parametrize("V", [9001, 50001])
def test_a_nucleus_of_nearly_everything(dev, below, V):
    # p = 1 - 2^-below: the cut lies among tokens of next to no weight, found with the same sums
    g = torch.Generator().manual_seed(300 + below)
    x = torch.randn(3, V, generator=g) * 3
    x[:, -1] = x.min() - 0.5                             # the worst token, last in the vocabulary
    p = 1.0 - 2.0 ** -below
    want = []
    for row in x.double():
        w, order = torch.sort(torch.exp(row - row.max()), descending=True, stable=True)
        before = torch.cumsum(w, 0) - w
        gap = (before - p * w.sum()).abs().min() / w.sum()
        assert gap > 1e-11, "a case too close to a border to be decided"
        want.append(int(order[before < p * w.sum()].max()))
    u = torch.full((3,), 1.0, device=dev)                # the last kept token
    assert K.sample_tokens(x.to(dev), u, top_p=p).tolist() == want
    assert K.sample_tokens(x.to(dev).repeat(200, 1), u.repeat(200), top_p=p).tolist() == want * 200


def test_what_a_workspace_holds_does_not_matter(dev):
    # all bits set (NaN, counts of -1), and what a call of other sizes left
    x = (torch.randn(5, 40000, generator=torch.Generator().manual_seed(1)) * 3).to(dev)
    u = torch.rand(5, generator=torch.Generator().manual_seed(2)).to(dev)
    need = K.sample_tokens_workspace_bytes(5, 40000)
    for kw in (dict(), dict(top_p=0.9), dict(top_k=30), dict(top_k=3000, top_p=0.5, min_p=0.01), dict(temperature=0.0),
               dict(top_k=20000), dict(top_p=0.99999)):
        ws = torch.full((need,), 0xFF, dtype=torch.uint8, device=dev)
        want = K.sample_tokens(x, u, workspace=ws, **kw)
        assert torch.equal(want, K.sample_tokens(x, u, workspace=ws, **kw))
        K.sample_tokens(x[:2, :777], u[:2], workspace=ws, top_p=0.3)
        assert torch.equal(want, K.sample_tokens(x, u, workspace=ws, **kw)) and torch.equal(want, K.sample_tokens(x, u, **kw))


def test_a_recorded_draw(dev):
    # replayed with other logits, filters and numbers in the same tensors, and eager work in between
    g = torch.Generator().manual_seed(3)
    B, V = 7, 50001
    x, u, p = torch.zeros(B, V, device=dev), torch.zeros(B, device=dev), torch.ones(B, device=dev)
    k = torch.zeros(B, dtype=torch.int32, device=dev)
    ws = torch.empty(K.sample_tokens_workspace_bytes(B, V), dtype=torch.uint8, device=dev)
    out = torch.zeros(B, dtype=torch.int64, device=dev)
    call = lambda o, w: K.sample_tokens(x, u, top_p=p, top_k=k, out=o, workspace=w)  # noqa: E731
    call(out, ws)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(out, ws)
    for step in range(6):
        x.copy_(torch.randn(B, V, generator=g) * (1 + step))
        u.copy_(torch.rand(B, generator=g))
        p.copy_(torch.rand(B, generator=g))
        k.copy_(torch.randint(-50, 50, (B,), generator=g).to(torch.int32))
        graph.replay()
        got = out.clone()
        assert torch.equal(got, call(torch.zeros_like(out), None))
        torch.cuda.synchronize()
