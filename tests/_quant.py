"""Plain forms of the 8-bit pages, paged attention and token sampling, for the tests."""
import math

import torch

TOP = {torch.int8: 127.0, torch.float8_e4m3fn: 448.0}
HALF_STEP = {t: torch.finfo(t).eps / 2 for t in (torch.float16, torch.bfloat16, torch.float32)}


def encode(x, fmt):
    """x [..., 128] -> (codes, scale [...]) by the definition, in fp32 on the CPU."""
    x = x.float()
    amax = x.abs().amax(-1, keepdim=True)
    scale = (amax / TOP[fmt]).clamp(min=2.0 ** -126)
    y = x / scale
    codes = y.round().to(torch.int8) if fmt == torch.int8 else y.clamp(-448, 448).to(fmt)
    bad = ~torch.isfinite(amax)
    codes = torch.where(bad, torch.zeros_like(codes.view(torch.uint8)), codes.view(torch.uint8)).view(fmt)
    return codes, torch.where(bad, torch.full_like(scale, math.nan), scale)[..., 0]


def decode(codes, scale):
    return codes.float() * scale[..., None]


def table(lens, ids):
    """CSR page table of requests of these lengths over the page ids ``ids``; and the ids per request."""
    per, at = [], 0
    for n in lens:
        k = (n + 15) // 16
        per.append(ids[at:at + k])
        at += k
    ptr = [0]
    for x in per:
        ptr.append(ptr[-1] + len(x))
    flat = torch.cat(per) if at else torch.zeros(1, dtype=torch.long)
    last = [n - (len(x) - 1) * 16 if n else 0 for n, x in zip(lens, per)]
    i32 = lambda v: torch.as_tensor(v, dtype=torch.int32)  # noqa: E731
    return (i32(flat), i32(ptr), i32(last)), per


def tokens_of(pool, pages, n):
    """First n tokens [n, Hkv, 128] of the pages of a [pages, 16, Hkv, 128] pool, in 64 bits."""
    if n == 0:
        return torch.zeros((0,) + tuple(pool.shape[2:]), dtype=torch.float64)
    return pool[pages].double().flatten(0, 1)[:n]


def attention64(q, k, v, scale):
    """q [H, 128], k / v [n, Hkv, 128] in 64 bits -> out [H, 128], lse [H] and, per element of out,
    sum of p |v|, the row's largest sum |q k| scale and the largest |v|."""
    H, Hkv = q.shape[0], k.shape[1]
    if k.shape[0] == 0:
        z = torch.zeros(H, 128, dtype=torch.float64)
        return z, torch.full((H,), -math.inf, dtype=torch.float64), z, torch.zeros(H, dtype=torch.float64), 0.0
    q = q.double().reshape(Hkv, H // Hkv, 128)
    kt = k.permute(1, 2, 0)
    s = torch.matmul(q, kt) * scale
    p = torch.softmax(s, -1)
    out = torch.matmul(p, v.transpose(0, 1)).reshape(H, 128)
    mag = torch.matmul(p, v.abs().transpose(0, 1)).reshape(H, 128)
    big = (torch.matmul(q.abs(), kt.abs()) * scale).amax(-1).reshape(H)
    return out, torch.logsumexp(s, -1).reshape(H), mag, big, float(v.abs().max())


def check_attention(out, lse, ref, n, dtype, weight_type):
    """The kernel's row set [H, 128] against attention64's answer. Bounds: the weights are rounded to
    ``weight_type`` (half a step of each, relative; below fp16's normal range 2^-25 of the largest
    weight), the output to ``dtype``; logits are fp32 sums of 128 exact products (an error of 130 *
    2^-24 of their summed magnitudes, entering numerator and denominator); sums of n terms and exp2
    (n + 64) * 2^-24."""
    r_out, r_lse, mag, big, vmax = ref
    f = 2.0 ** -24
    dz = 130 * f * big[:, None]
    rel = HALF_STEP[weight_type] + 2 * dz + (n + 64) * f
    floor = n * 2.0 ** -24 * vmax if weight_type == torch.float16 else 0.0
    bound = rel * mag + HALF_STEP[dtype] * (r_out.abs() + rel * mag) + floor + 1e-30
    if dtype == torch.float16:
        bound = bound + 2.0 ** -25            # half a step below fp16's normal range
    err = (out.double() - r_out).abs()
    assert torch.all(err <= bound), f"out off by {(err / bound).max():.2f} bounds (n {n})"
    if n == 0:
        assert torch.all(torch.isneginf(lse))
        return
    lerr = (lse.double() - r_lse).abs()
    assert torch.all(lerr <= dz[:, 0] + (n + 64) * f + r_lse.abs() * 2 * f), f"lse off by {lerr.max()}"


def sample64(x, u, temperature, top_k, top_p, min_p):
    """One row by the definition, in 64 bits: (token, distance of the nearest decision from its border
    relative to the mass that decides it)."""
    x = x.double()
    x = torch.where(torch.isnan(x), -math.inf, x)
    best = float(x.max())
    if best == -math.inf:
        return -1, math.inf
    order = sorted(range(len(x)), key=lambda i: (-float(x[i]), i))
    if not temperature > 0 or top_k == 1:
        return order[0], math.inf
    w = [1.0 if float(x[i]) == best else math.exp((float(x[i]) - best) / temperature) for i in order]
    if top_k > 0:
        order, w = order[:top_k], w[:top_k]
    margin, keep = math.inf, len(order)
    if top_p <= 0:
        keep = 1                              # nothing lies before the best rank: no border is near
    elif top_p < 1:
        goal, before = top_p * math.fsum(w), 0.0
        keep = 0
        while keep < len(w) and (keep == 0 or before < goal):
            before += w[keep]
            keep += 1
        before = math.fsum(w[:keep])
        margin = min(margin, abs(before - goal), abs(before - w[keep - 1] - goal)) / math.fsum(w)
    kept = [(i, wi) for r, (i, wi) in enumerate(zip(order[:keep], w[:keep])) if r == 0 or not wi < min_p]
    if min_p > 0:
        margin = min([margin] + [abs(wi - min_p) for wi in w[1:keep] if wi != 1.0])
    kept.sort()
    total = math.fsum(wi for _, wi in kept)
    run = 0.0
    for i, wi in kept:
        run += wi
        if run > u * total:
            return i, min([margin] + [abs(b - u * total) / total for b in (run, run - wi) if 0 < b < total])
    return [i for i, wi in kept if wi > 0][-1], margin
