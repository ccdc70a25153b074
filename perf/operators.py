"""Cases, plain forms and 64-bit values of the operators of one sampled decode step over an 8-bit
cache: quantising K / V as they are written and reading them back, decode attention over the
quantised pages, decode attention of requests that share a prefix, and drawing the next tokens.

``run(state)`` computes a case in elementary tensor operations (``own`` false) or through
``twilight_amd.kernel`` (``own`` true). Pages hold 16 tokens, heads 128 channels; page tables are
the CSR triples (page indices, indptr, length of the last page) of ``twilight_amd.cache``.
"""
import math

import torch

own = False

PAGE, D = 16, 128
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
FORMATS = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}
TOP = {"int8": 127.0, "e4m3": 448.0}      # the largest value a code stands for
TINY = 2.0 ** -126


def listed():
    return [
        # one decode step of eight requests: one new token each is written, and read again
        dict(name="cache_step", kind="cache", dtype="bf16", fmt="int8", B=8, Hkv=8, new=1, old=4096, ragged=False, whole=False),
        # a chunk of ragged prompts joins what is cached, and the whole contexts are read back for
        # the chunk's own attention
        dict(name="cache_chunk", kind="cache", dtype="fp16", fmt="e4m3", B=5, Hkv=8, new=1037, old=3001, ragged=True, whole=True),
        # bulk fill after a long prefill, 32 kv heads
        dict(name="cache_prefill", kind="cache", dtype="bf16", fmt="int8", B=4, Hkv=32, new=8192, old=0, ragged=False, whole=False),
        # a single short request: latency
        dict(name="quant_attn_one", kind="attn", dtype="bf16", fmt="int8", B=1, H=32, Hkv=8, n=777, ragged=False),
        # decode at batch 8, 32 q / 8 kv heads, 32k context
        dict(name="quant_attn_32k", kind="attn", dtype="bf16", fmt="int8", B=8, H=32, Hkv=8, n=32768, ragged=False),
        # one q head per kv head, ragged lengths, one request empty
        dict(name="quant_attn_mha", kind="attn", dtype="fp16", fmt="e4m3", B=16, H=32, Hkv=32, n=8191, ragged=True),
        # a few samples of one short prompt: latency
        dict(name="prefix_short", kind="prefix", dtype="fp16", fmt="none", B=4, H=32, Hkv=8, groups=1, prefix=1000, n=33, ragged=True),
        # many samples of one 32k prompt
        dict(name="prefix_wide", kind="prefix", dtype="bf16", fmt="none", B=64, H=32, Hkv=8, groups=1, prefix=32768, n=600, ragged=True),
        # three prompts with different numbers of samples over an 8-bit cache
        dict(name="prefix_groups", kind="prefix", dtype="bf16", fmt="int8", B=33, H=32, Hkv=8, groups=3, prefix=16001, n=300, ragged=True),
        # one row: latency
        dict(name="sample_one", kind="sample", dtype="fp32", B=1, V=32000, top_k=0, top_p=0.9, min_p=0.0),
        # a batch over a large vocabulary, nucleus sampling
        dict(name="sample_batch", kind="sample", dtype="bf16", B=64, V=128256, top_k=0, top_p=0.95, min_p=0.0),
        # an odd vocabulary, every filter in use
        dict(name="sample_filters", kind="sample", dtype="fp16", B=17, V=50001, top_k=200, top_p=0.9, min_p=0.02),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["cache", "attn", "prefix", "sample"])
    dtype = rng.choice(["bf16", "fp16"])
    ragged = rng.random() < 0.6
    if kind == "cache":
        B, Hkv = _log(rng, 1, 32), rng.choice([1, 2, 3, 8, 32])
        room = 4 * 8192 * 32 // (B * Hkv)                 # tokens per request within the largest case
        new = _log(rng, 1, max(1, min(8192, room // 2)))
        return dict(kind=kind, dtype=dtype, fmt=rng.choice(["int8", "e4m3"]), B=B, Hkv=Hkv, new=new,
                    old=rng.choice([0, _log(rng, 1, max(1, min(8192, room // 2)))]), ragged=ragged,
                    whole=rng.random() < 0.5)
    if kind == "sample":
        V = _log(rng, 1000, 128256)
        return dict(kind=kind, dtype=rng.choice(["bf16", "fp16", "fp32"]), B=_log(rng, 1, min(128, 64 * 128256 // V)),
                    V=V, top_k=rng.choice([0, 0, _log(rng, 1, 1000)]), top_p=round(rng.uniform(0.3, 1.0), 3),
                    min_p=rng.choice([0.0, round(rng.uniform(0.0, 0.1), 4)]))
    Hkv = rng.choice([1, 2, 4, 8, 32])
    G = rng.choice([1, 2, 4, 8] if Hkv < 32 else [1, 2])
    B = _log(rng, 1, 64)
    if kind == "attn":
        n = _log(rng, 1, max(16, min(32768, 8 * 32768 * 8 // (B * Hkv))))
        return dict(kind=kind, dtype=dtype, fmt=rng.choice(["int8", "e4m3"]), B=B, H=Hkv * G, Hkv=Hkv, n=n, ragged=ragged)
    groups = min(B, rng.choice([1, 1, 2, 5]))
    prefix = _log(rng, 16, max(64, min(32768, 64 * 32768 * 32 // (2 * B * Hkv * G * groups))))
    return dict(kind=kind, dtype=dtype, fmt=rng.choice(["none", "int8", "e4m3"]), B=B, H=Hkv * G, Hkv=Hkv,
                groups=groups, prefix=prefix, n=_log(rng, 1, max(16, min(600, 64 * 600 * 8 // (B * Hkv)))), ragged=ragged)


# ---- inputs ------------------------------------------------------------------------------------
def _lens(B, n, ragged, gen, least=0):
    """Lengths up to n: the first request has n tokens, and of a ragged batch of three or more the
    second has ``least``."""
    if not ragged:
        return [n] * B
    got = torch.randint(min(max(1, least), n), n + 1, (B,), generator=gen).tolist()
    got[0] = n
    if B >= 3:
        got[1] = least
    return got


def _table(lens, pages, dev):
    """CSR page table of requests of these lengths over the page ids ``pages`` (used from the
    front), and how many it took."""
    per = [(n + PAGE - 1) // PAGE for n in lens]
    ptr = [0]
    for x in per:
        ptr.append(ptr[-1] + x)
    last = [n - (x - 1) * PAGE if x else 0 for n, x in zip(lens, per)]
    i32 = dict(dtype=torch.int32, device=dev)
    ids = pages[:ptr[-1]].to(torch.int32)
    if ptr[-1] == 0:
        ids = torch.zeros(1, **i32)
    return (ids, torch.tensor(ptr, **i32), torch.tensor(last, **i32)), ptr[-1]


def _encode(x, fmt):
    """x [..., 128] in 32 bits -> codes and one scale per row of 128."""
    amax = x.abs().amax(-1, keepdim=True)
    scale = (amax / TOP[fmt]).clamp(min=TINY)
    y = x / scale
    if fmt == "int8":
        codes = y.round().clamp(-127, 127).to(torch.int8)
    else:
        codes = y.clamp(-448, 448).to(torch.float8_e4m3fn)
    return codes, scale[..., 0]


def _pool(num_pages, Hkv, case, gen, dev):
    """Filled K or V pages as [pages, 16, Hkv, 128] views, heads outermost inside a page for the
    8-bit formats; with the scales [pages, 16, Hkv] or None. Channels differ in magnitude."""
    dtype = DTYPES[case["dtype"]]
    gain = torch.exp(torch.randn(Hkv, 1, D, generator=gen, device=dev) * 0.4)
    if case["fmt"] == "none":
        x = torch.randn(num_pages, PAGE, Hkv, D, generator=gen, device=dev, dtype=dtype)
        return x * gain[:, 0].to(dtype), None
    codes = torch.empty(num_pages, Hkv, PAGE, D, dtype=FORMATS[case["fmt"]], device=dev)
    scale = torch.empty(num_pages, Hkv, PAGE, device=dev)
    for a in range(0, num_pages, 4096):
        n = min(4096, num_pages - a)
        x = torch.randn(n, Hkv, PAGE, D, generator=gen, device=dev) * gain
        codes[a:a + n], scale[a:a + n] = _encode(x, case["fmt"])
    return codes.transpose(1, 2), scale.transpose(1, 2)


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    host = torch.Generator().manual_seed(seed)
    s = dict(case=dict(case))
    dtype = DTYPES[case["dtype"]]
    B = case["B"]
    if case["kind"] == "sample":
        V = case["V"]
        x = torch.randn(B, V, generator=gen, device=dev) * 2.2
        # a few likely tokens at random places, as a trained model's rows have them
        at = torch.randint(0, V, (B, 24), generator=gen, device=dev)
        x.scatter_(1, at, 9.0 + 4.0 * torch.rand(B, 24, generator=gen, device=dev))
        s["logits"] = x.to(dtype)
        s["u"] = torch.rand(B, generator=gen, device=dev)
        spread = torch.rand(3, B, generator=gen, device=dev)
        s["temperature"] = 0.6 + 0.8 * spread[0]
        s["top_k"] = torch.full((B,), case["top_k"], dtype=torch.int32, device=dev)
        s["top_p"] = (case["top_p"] * (1.0 - 0.05 * spread[1])).float()
        s["min_p"] = (case["min_p"] * spread[2]).float()
        return s
    Hkv = case["Hkv"]
    if case["kind"] == "cache":
        host = torch.Generator().manual_seed(case["new"] + case["old"])   # one shape of outputs for a case
        new = _lens(B, case["new"], case["ragged"], host, 1)
        old = _lens(B, case["old"], case["ragged"], host) if case["old"] else [0] * B
        lens = [a + b for a, b in zip(new, old)]
        total = sum((n + PAGE - 1) // PAGE for n in lens) + 3
        perm = torch.randperm(total, generator=gen, device=dev)
        s["table"], _ = _table(lens, perm, dev)
        s["k"], s["k_scale"] = _pool(total, Hkv, case, gen, dev)
        s["v"], s["v_scale"] = _pool(total, Hkv, case, gen, dev)
        read = lens if case["whole"] else new
        for key, counts in (("new", new), ("read", read)):
            ptr = [0]
            for n in counts:
                ptr.append(ptr[-1] + n)
            s[key + "_indptr"] = torch.tensor(ptr, dtype=torch.int32, device=dev)
            s[key + "_tokens"] = ptr[-1]
        shape = (s["new_tokens"], Hkv, D)
        s["k_new"] = torch.randn(shape, generator=gen, device=dev, dtype=dtype)
        s["v_new"] = torch.randn(shape, generator=gen, device=dev, dtype=dtype)
        return s
    G = case["H"] // Hkv
    lens = _lens(B, case["n"], case["ragged"], host)
    groups = case.get("groups", 0)
    plens = _lens(groups, case["prefix"], case["ragged"], host, 1) if groups else []
    pages = sum((n + PAGE - 1) // PAGE for n in lens + plens) + 2
    perm = torch.randperm(pages, generator=gen, device=dev)
    s["table"], used = _table(lens, perm, dev)
    s["max_tokens"] = max(1, max(lens))
    if groups:
        s["prefix"], _ = _table(plens, perm[used:], dev)
        # every group has a sample, the others fall where they may
        cut = sorted(torch.randperm(B - 1, generator=host)[:groups - 1].add(1).tolist()) if groups > 1 else []
        ptr = [0] + cut + [B]
        s["group_indptr"] = torch.tensor(ptr, dtype=torch.int32, device=dev)
        s["max_prefix"] = max(plens)
        s["max_group"] = max(b - a for a, b in zip(ptr, ptr[1:]))
    s["k"], s["k_scale"] = _pool(pages, Hkv, case, gen, dev)
    s["v"], s["v_scale"] = _pool(pages, Hkv, case, gen, dev)
    q = torch.randn(B, Hkv * G, D, generator=gen, device=dev) * 1.2
    s["q"] = q.to(dtype)
    return s


# ---- plain forms -------------------------------------------------------------------------------
def _tokens(cache, scale, pages):
    """Pages [..., P] of the cache as tokens [..., P * 16, Hkv, 128] in 32 bits."""
    if scale is None:
        return cache[pages].float().flatten(-4, -3)
    codes = cache.view(torch.uint8)[pages].view(cache.dtype).float()
    return (codes * scale[pages][..., None]).flatten(-4, -3)


def _page_matrix(table, tokens):
    """Padded page ids [requests, P] and lengths [requests]."""
    ids, ptr, last = (t.long() for t in table)
    count = ptr[1:] - ptr[:-1]
    at = ptr[:-1, None] + torch.arange((tokens + PAGE - 1) // PAGE, device=ids.device)
    return ids[at.clamp(max=ids.numel() - 1)], torch.where(count > 0, (count - 1) * PAGE + last, 0)


def _places(table, indptr, tokens):
    """Page and slot of the last indptr[b + 1] - indptr[b] tokens of every request, in order."""
    ids, ptr, last = (t.long() for t in table)
    start = indptr.long()
    t = torch.arange(tokens, device=ids.device)
    b = torch.searchsorted(start[1:], t, right=True)
    pos = (ptr[b + 1] - ptr[b] - 1) * PAGE + last[b] - start[b + 1] + t
    return ids[ptr[b] + pos // PAGE], pos % PAGE


def _plain_cache(s):
    fmt = s["case"]["fmt"]
    page, slot = _places(s["table"], s["new_indptr"], s["new_tokens"])
    rpage, rslot = _places(s["table"], s["read_indptr"], s["read_tokens"])
    got = []
    for x, cache, scale in ((s["k_new"], s["k"], s["k_scale"]), (s["v_new"], s["v"], s["v_scale"])):
        codes, sc = _encode(x.float(), fmt)
        cache.view(torch.uint8)[page, slot] = codes.view(torch.uint8)
        scale[page, slot] = sc
        back = cache.view(torch.uint8)[rpage, rslot].view(cache.dtype).float() * scale[rpage, rslot][..., None]
        got.append(back.to(x.dtype))
    return {"k": got[0], "v": got[1]}


def _hidden(logits, lens):
    at = torch.arange(logits.shape[-1], device=logits.device)
    gone = at >= lens.reshape(-1, *[1] * (logits.dim() - 1))
    return logits.masked_fill(gone, -math.inf)


def _plain_attention(s):
    q = s["q"].float()
    B, H, _ = q.shape
    Hkv = s["case"]["Hkv"]
    G = H // Hkv
    q = q.view(B, Hkv, G, D) / math.sqrt(D)
    pages, lens = _page_matrix(s["table"], s["max_tokens"])
    k = _tokens(s["k"], s["k_scale"], pages)                                     # [B, N, Hkv, 128]
    lo = _hidden(torch.matmul(q, k.permute(0, 2, 3, 1).contiguous()), lens)      # [B, Hkv, G, N]
    top = lo.amax(-1, keepdim=True)
    if "prefix" in s:
        ppages, plens = _page_matrix(s["prefix"], s["max_prefix"])
        NG, M = plens.numel(), s["max_group"]
        start = s["group_indptr"].long()
        member = (start[:-1, None] + torch.arange(M, device=q.device)).clamp(max=B - 1)
        group = torch.searchsorted(start[1:], torch.arange(B, device=q.device), right=True)
        place = torch.arange(B, device=q.device) - start[group]
        qg = q[member].transpose(1, 2).reshape(NG, Hkv, M * G, D)
        kp = _tokens(s["k"], s["k_scale"], ppages)                               # [NG, P, Hkv, 128]
        lp = _hidden(torch.matmul(qg, kp.permute(0, 2, 3, 1).contiguous()), plens)
        ptop = lp.amax(-1, keepdim=True).view(NG, Hkv, M, G, 1).transpose(1, 2)[group, place]
        top = torch.maximum(top, ptop)
    top = top.clamp(min=-3e38)                                                   # rows without a token
    w = torch.exp(lo - top)
    v = _tokens(s["v"], s["v_scale"], pages)
    total = w.sum(-1, keepdim=True)
    acc = torch.matmul(w, v.transpose(1, 2).contiguous())
    if "prefix" in s:
        gtop = top[member].transpose(1, 2).reshape(NG, Hkv, M * G, 1)
        wp = torch.exp(lp - gtop)
        vp = _tokens(s["v"], s["v_scale"], ppages)
        pacc = torch.matmul(wp, vp.transpose(1, 2).contiguous())
        total = total + wp.sum(-1, keepdim=True).view(NG, Hkv, M, G, 1).transpose(1, 2)[group, place]
        acc = acc + pacc.view(NG, Hkv, M, G, D).transpose(1, 2)[group, place]
    out = torch.where(total > 0, acc / total, 0.0)
    lse = torch.where(total > 0, top + torch.log(total), -math.inf)
    return {"out": out.reshape(B, H, D).to(s["q"].dtype), "lse": lse.reshape(B, H)}


def _plain_sample(s):
    x = s["logits"].float()
    B, V = x.shape
    x = torch.where(torch.isnan(x), -math.inf, x)
    x, order = torch.sort(x, dim=-1, descending=True, stable=True)
    x = x.double()
    t = s["temperature"].double()[:, None]
    w = torch.where(x == x[:, :1], 1.0, torch.exp((x - x[:, :1]) / t))
    rank = torch.arange(V, device=x.device)
    k = s["top_k"].long()[:, None]
    keep = (rank < k) | (k <= 0)
    w = w * keep
    upto = torch.cumsum(w, -1)
    p = s["top_p"].double()[:, None]
    keep &= (upto - w < p * upto[:, -1:]) | (p >= 1)
    keep &= w >= s["min_p"].double()[:, None]
    keep |= rank == 0
    in_place = torch.zeros_like(w).scatter_(1, order, w * keep)
    upto = torch.cumsum(in_place, -1)
    beyond = upto > s["u"].double()[:, None] * upto[:, -1:]
    return {"tokens": beyond.to(torch.int8).argmax(-1)}


def run(s):
    kind = s["case"]["kind"]
    if not own:
        return {"cache": _plain_cache, "sample": _plain_sample}.get(kind, _plain_attention)(s)
    from twilight_amd import kernel as K
    if kind == "sample":
        return {"tokens": K.sample_tokens(s["logits"], s["u"], temperature=s["temperature"], top_k=s["top_k"],
                                          top_p=s["top_p"], min_p=s["min_p"])}
    if kind == "cache":
        K.kv_quant_append(s["k_new"], s["v_new"], s["new_indptr"], s["k"], s["v"], s["k_scale"], s["v_scale"], *s["table"])
        k, v = K.kv_quant_read(s["k"], s["v"], s["k_scale"], s["v_scale"], *s["table"], s["read_indptr"],
                               s["read_tokens"], dtype=s["k_new"].dtype)
        return {"k": k, "v": v}
    if kind == "attn":
        out, lse = K.quant_paged_decode_attention(s["q"], s["k"], s["v"], s["k_scale"], s["v_scale"], *s["table"],
                                                  max_tokens=s["max_tokens"], return_lse=True)
    else:
        out, lse = K.prefix_paged_decode_attention(
            s["q"], s["k"], s["v"], *s["prefix"], s["group_indptr"], *s["table"], max_prefix_tokens=s["max_prefix"],
            max_group_size=s["max_group"], max_tokens=s["max_tokens"], k_scale=s["k_scale"], v_scale=s["v_scale"],
            return_lse=True)
    return {"out": out, "lse": lse}


# ---- what a pass cannot do without ---------------------------------------------------------------
def work(case):
    """Bytes and operations of one pass; ragged batches at the mean of their lengths."""
    B = case["B"]
    size = {"bf16": 2, "fp16": 2, "fp32": 4}[case["dtype"]]
    if case["kind"] == "sample":
        return {"bytes": B * case["V"] * size + 28 * B, "flops": 4 * B * case["V"]}

    def mean(n):
        return (n + 1) / 2 if case["ragged"] and n else n

    Hkv = case["Hkv"]
    held = 2 * D * size if case["fmt"] == "none" else 2 * (D + 4)                # K and V of a token and head
    if case["kind"] == "cache":
        new = B * mean(case["new"])
        read = B * (mean(case["new"]) + mean(case["old"])) if case["whole"] else new
        return {"bytes": (new + read) * Hkv * (2 * D * size + held), "flops": (6 * new + 2 * read) * Hkv * 2 * D}
    H, NG = case["H"], case.get("groups", 0)
    own_tokens = B * mean(case["n"])
    shared = NG * mean(case["prefix"]) if NG else 0
    seen = own_tokens + (B * mean(case["prefix"]) if NG else 0)
    return {"bytes": (own_tokens + shared) * Hkv * held + B * H * (2 * D * size + 4), "flops": 4 * D * H * seen}


# ---- 64-bit values -------------------------------------------------------------------------------
def _grid(fmt, x):
    """x [..., 128] rounded to what its codes stand for, from the definition of the format."""
    x = x.double()
    scale = (x.abs().amax(-1, keepdim=True) / TOP[fmt]).clamp(min=TINY)
    scale = scale.float().double()                        # the cache holds the scale in 32 bits
    y = x / scale
    if fmt == "int8":
        return torch.round(y) * scale
    # e4m3: steps of 2^(exponent - 3), of 2^-9 below 2^-6
    step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.round(y / step) * step * scale


def _list_of(table, b):
    ids, ptr, last = table
    a, e = int(ptr[b]), int(ptr[b + 1])
    return ids[a:e].long(), 0 if e == a else (e - a - 1) * PAGE + int(last[b])


def _exact_tokens(s, which, table, b):
    """All tokens [n, Hkv, 128] of request b in 64 bits."""
    pages, n = _list_of(table, b)
    Hkv = s["case"]["Hkv"]
    if n == 0:
        return torch.zeros(0, Hkv, D, dtype=torch.float64, device="cuda")
    cache, scale = s[which], s[which + "_scale"]
    if scale is None:
        return cache[pages].double().reshape(-1, Hkv, D)[:n]
    x = cache.view(torch.uint8)[pages].view(cache.dtype).to(torch.float32).double()
    return (x * scale[pages].double().unsqueeze(-1)).reshape(-1, Hkv, D)[:n]


def exact(case, seed):
    if case["kind"] == "sample":
        return None                                       # token ids: compared as whole numbers
    s = prepare(case, seed)
    B, Hkv = case["B"], case["Hkv"]
    if case["kind"] == "cache":
        result = {}
        for which in ("k", "v"):
            parts = []
            for b in range(B):
                a, e = int(s["new_indptr"][b]), int(s["new_indptr"][b + 1])
                seen = _exact_tokens(s, which, s["table"], b)
                seen[seen.shape[0] - (e - a):] = _grid(case["fmt"], s[which + "_new"][a:e])
                back = int(s["read_indptr"][b + 1]) - int(s["read_indptr"][b])
                parts.append(seen[seen.shape[0] - back:])
            result[which] = torch.cat(parts)
        return result
    H = case["H"]
    out = torch.zeros(B, H, D, dtype=torch.float64, device="cuda")
    lse = torch.full((B, H), -math.inf, dtype=torch.float64, device="cuda")
    shared, bounds = [], [0, B]
    if "prefix" in s:
        bounds = s["group_indptr"].tolist()
        shared = [(_exact_tokens(s, "k", s["prefix"], g), _exact_tokens(s, "v", s["prefix"], g)) for g in range(case["groups"])]
    for b in range(B):
        k, v = _exact_tokens(s, "k", s["table"], b), _exact_tokens(s, "v", s["table"], b)
        pairs = [(k, v)]
        if shared:
            g = max(i for i in range(len(bounds) - 1) if bounds[i] <= b)
            pairs.append(shared[g])
        q = s["q"][b].double().view(Hkv, H // Hkv, D)
        z = torch.cat([torch.bmm(q, x.permute(1, 2, 0).contiguous()) for x, _ in pairs], -1) * D ** -0.5
        if z.shape[-1] == 0:
            continue
        part = torch.softmax(z, -1)
        n = pairs[0][0].shape[0]
        o = torch.bmm(part[..., :n].contiguous(), v.transpose(0, 1).contiguous())
        if shared:
            o = o + torch.bmm(part[..., n:].contiguous(), pairs[1][1].transpose(0, 1).contiguous())
        out[b] = o.reshape(H, D)
        lse[b] = torch.logsumexp(z, -1).reshape(H)
    return {"out": out, "lse": lse}
