"""Token sampling against the definition in 64 bits, token for token. Every drawn case keeps its
decisions at least 1e-11 of the deciding mass away from their borders (2^18 tokens off by 2^-46 each
reach 4e-9 of the best weight in the worst case and 1e-12 as they fall), which is checked on the CPU;
borders that are met exactly have tests of their own."""
import math

import pytest
import torch

import twilight_amd.kernel as K
from _quant import sample64

pytestmark = pytest.mark.gpu


def _rows(B, V, dtype, seed, spread=2.5, peaks=8):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn((B, V), generator=g) * spread
    for b in range(B):
        at = torch.randint(0, V, (min(peaks, V),), generator=g)
        x[b, at] = 6 + 5 * torch.rand(len(at), generator=g)
    return x.to(dtype), torch.rand(B, generator=g)


def _check(dev, x, u, t, k, p, m, **kw):
    B = x.shape[0]
    col = lambda v, dt: v if isinstance(v, torch.Tensor) else torch.full((B,), v, dtype=dt)  # noqa: E731
    t, k, p, m = col(t, torch.float32), col(k, torch.int32), col(p, torch.float32), col(m, torch.float32)
    want, margin = zip(*(sample64(x[b], float(u[b]), float(t[b]), int(k[b]), float(p[b]), float(m[b])) for b in range(B)))
    assert min(margin) > 1e-11, "a case too close to a border to be decided"
    got = K.sample_tokens(x.to(dev) if x.is_contiguous() else x, u.to(dev), temperature=t.to(dev), top_k=k.to(dev),
                          top_p=p.to(dev), min_p=m.to(dev), **kw)
    assert got.dtype == torch.int64 and got.tolist() == list(want)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("B,V", [(1, 1), (3, 2), (5, 63), (4, 64), (3, 65), (2, 1000), (3, 1025), (2, 5003), (1, 50001)])
def test_filters(dev, dtype, B, V):
    for n, (t, k, p, m) in enumerate([(1.0, 0, 1.0, 0.0), (0.7, 0, 0.9, 0.0), (1.3, 40, 1.0, 0.0), (1.0, 20, 0.8, 0.01),
                                      (2.0, 0, 0.99, 0.05), (0.2, 5, 0.5, 0.0), (1.0, V, 0.3, 0.3)]):
        x, u = _rows(B, V, dtype, 100 * n + V)
        _check(dev, x, u, t, k, p, m)


def test_rows_with_filters_of_their_own(dev):
    x, u = _rows(6, 2000, torch.bfloat16, 5)
    _check(dev, x, u, torch.tensor([0.0, 0.5, 1.0, 1.5, -1.0, math.nan]), torch.tensor([0, 3, 100, 0, -7, 9], dtype=torch.int32),
           torch.tensor([0.9, 0.9, 0.0, 1.0, 0.5, 0.5]), torch.tensor([0.0, 0.1, 0.0, 1.0, 0.0, 0.0]))


def test_flat_rows_large_vocabulary(dev):
    # the nucleus of a flat row is most of the vocabulary
    x, u = _rows(2, 262144, torch.float32, 6, spread=0.3, peaks=0)
    _check(dev, x, u, 1.0, 0, 0.95, 0.0)
    _check(dev, x, u, 1.0, 100000, 0.9, 0.0)


def test_equal_logits_are_ranked_by_index(dev):
    V = 1500
    x = torch.zeros(4, V)
    x[:, ::3] = 2.0                                  # 500 best tokens, all equal
    # top-k 10 keeps indices 0, 3, .. 27; uniform over them
    got = K.sample_tokens(x.to(dev), torch.tensor([0.0, 0.05, 0.55, 0.99]).to(dev), top_k=10)
    assert got.tolist() == [0, 0, 15, 27]
    # one value everywhere: top-p 0.5 of 1500 keeps the ranks before which less than 750 lie
    y = torch.full((3, V), -4.0)
    got = K.sample_tokens(y.to(dev), torch.tensor([0.0, 0.5, 0.9999]).to(dev), top_p=0.5)
    assert got.tolist() == [0, 375, 749]
    # the cut falls inside the lower value
    got = K.sample_tokens(x.to(dev), torch.tensor([0.0, 0.3, 0.9999, 0.9999]).to(dev), top_k=502, temperature=1e30)
    # weights are equal at this temperature: kept are every third index and indices 1, 2
    kept = sorted(set(range(0, V, 3)) | {1, 2})
    assert got.tolist() == [kept[0], kept[int(0.3 * 502)], kept[501], kept[501]]
    # the two zeros are one value
    z = torch.tensor([[-0.0, 0.0, -0.0, -1.0]])
    assert K.sample_tokens(z.to(dev), torch.tensor([0.0]).to(dev), temperature=0.0).tolist() == [0]
    assert K.sample_tokens(z.to(dev), torch.tensor([0.9]).to(dev), top_k=2).tolist() == [1]


def test_masked_and_extreme_logits(dev):
    inf = math.inf
    x = torch.full((7, 130), -inf)
    x[1, 77] = -5.0
    x[2, 5], x[2, 9] = inf, 3.0
    x[3, 3], x[3, 8], x[3, 100] = inf, inf, 0.0
    x[4] = math.nan
    x[5] = math.nan
    x[5, 129] = torch.finfo(torch.float32).min
    x[6, 0], x[6, 64] = 3e38, -3e38
    u = torch.tensor([0.5, 0.9, 0.9, 0.6, 0.2, 0.9, 0.999])
    for kw in (dict(), dict(top_p=0.9), dict(top_k=50), dict(min_p=0.1), dict(temperature=0.0)):
        got = K.sample_tokens(x.to(dev), u.to(dev), **kw).tolist()
        assert got == [-1, 77, 5, 3 if kw.get("temperature") == 0.0 else 8, -1, 129, 0], kw


def test_u_at_its_ends(dev):
    x = torch.zeros(5, 100)
    x[:, 0] = -math.inf
    u = torch.tensor([0.0, -1.0, 1.0, 2.0, math.nan])
    assert K.sample_tokens(x.to(dev), u.to(dev)).tolist() == [1, 1, 99, 99, 1]


def test_strided_and_unaligned_rows(dev):
    # the last position of [B, S, V] logits, and a slice that starts at an odd element
    g = torch.Generator().manual_seed(1)
    full = (torch.randn((3, 4, 1001), generator=g) * 3).to(torch.bfloat16).to(dev)
    u = torch.rand(3, generator=g)
    for x in (full[:, -1], full[:, 1, 1:], full[:, 0, 3:700], full[0, :3, 5:]):
        want = [sample64(x[b].cpu(), float(u[b]), 1.0, 0, float(torch.tensor(0.9)), 0.0)[0] for b in range(3)]
        assert K.sample_tokens(x, u.to(dev), top_p=0.9).tolist() == want
    out = torch.zeros(3, dtype=torch.int64, device=dev)
    assert K.sample_tokens(full[:, -1], u.to(dev), out=out) is out


def test_shares_follow_the_weights(dev):
    # 4096 evenly spaced u over one row: every kept token is hit in proportion to its weight, to within one
    V = 300
    g = torch.Generator().manual_seed(4)
    row = torch.randn(V, generator=g) * 2
    n = 4096
    got = K.sample_tokens(row.expand(n, V).to(dev), ((torch.arange(n) + 0.5) / n).to(dev), top_k=50).cpu()
    w = torch.zeros(V, dtype=torch.float64)
    at = torch.argsort(row, descending=True, stable=True)[:50]
    w[at] = torch.softmax(row[at].double(), 0)
    assert torch.all((torch.bincount(got, minlength=V).double() - n * w).abs() <= 1.0)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("B,V", [(520, 5003), (200, 20000), (130, 50001)])
def test_batches_whose_slices_are_several_tiles(dev, dtype, B, V):
    # enough rows for slices of two and four tiles of 4096 tokens, one or several slices a row; a few rows are
    # drawn on the CPU too
    x, u = _rows(B, V, dtype, B)
    for t, k, p, m in ((0.8, 0, 0.9, 0.0), (1.0, 60, 0.95, 0.02), (1.5, 0, 1.0, 0.01), (0.0, 0, 1.0, 0.0)):
        got = K.sample_tokens(x.to(dev), u.to(dev), temperature=t, top_k=k, top_p=p, min_p=m).cpu()
        f32 = lambda v: float(torch.tensor(v))  # noqa: E731
        for b in (0, 1, B // 2, B - 1):
            want, margin = sample64(x[b], float(u[b]), f32(t), k, f32(p), f32(m))
            assert margin > 1e-11, "a case too close to a border to be decided"
            assert int(got[b]) == want
        assert torch.equal(got, K.sample_tokens(x.to(dev), u.to(dev), temperature=t, top_k=k, top_p=p, min_p=m).cpu())


def test_many_equal_candidates_at_the_cut(dev):
    # bf16 rows whose cut falls among thousands of equal logits: the cut is found by index, and above 8192 of
    # them over the whole row
    for V, same in ((30000, 3000), (30000, 8000), (60000, 20000)):
        g = torch.Generator().manual_seed(same)
        x = torch.full((3, V), -30.0)
        at = torch.randperm(V, generator=g)[:same].sort().values
        x[:, at] = 1.0
        x[:, at[5]] = 2.0
        x = x.to(torch.bfloat16)
        # top-k keeps the best one and the first k - 1 of the equal ones
        k = same // 2
        kept = at[:k]
        u = torch.tensor([0.0, 0.4, 0.9999])
        got = K.sample_tokens(x.to(dev), u.to(dev), top_k=k, temperature=1e30).tolist()
        # equal weights: the running sum exceeds u k first after floor(u k) + 1 of them (the fp32 nearest to 0.9999
        # is below it: 9998 of 10000)
        assert got == [int(kept[int(float(v) * k)]) for v in u]
        # top-p 0.25: the best one (e) and as many equal ones (1 each) as it takes to reach a quarter of the mass
        p, total = 0.25, same - 1 + math.e
        n = math.ceil(p * total - math.e)
        ones = torch.cat([at[:5], at[6:]])[:n]
        last = int(torch.cat([ones, at[5:6]]).max())
        assert K.sample_tokens(x.to(dev), torch.full((3,), 1.0).to(dev), top_p=p).tolist() == [last] * 3
