"""The operators together, as a decode step of several samples of one prompt uses them: append to an 8-bit
cache, attention with the prompt as a shared prefix, the next token of every sample. Eagerly, on another
stream, recorded into HIP graphs, and inside a Hugging Face model."""
import json

import pytest
import torch

import twilight_amd.kernel as K
from twilight_amd import hf
from twilight_amd.cache import QuantPagedKVCache
from _quant import attention64, check_attention, decode, encode, sample64
from test_gpu_hf import CFG, _tiny_llama

pytestmark = pytest.mark.gpu
H, HKV, V = 8, 2, 301


class Step:
    """Samples of one prompt: prompt pages 0.., one page list per sample behind them."""

    def __init__(self, dev, fmt, samples, prompt, dtype=torch.bfloat16, seed=0):
        g = torch.Generator().manual_seed(seed)
        r = lambda *s: torch.randn(s, generator=g)  # noqa: E731
        self.dev, self.fmt, self.B, self.prompt, self.dtype = dev, fmt, samples, prompt, dtype
        self.k0, self.v0 = r(prompt, HKV, 128).to(dtype), r(prompt, HKV, 128).to(dtype)
        pages = (prompt + 15) // 16
        self.cache = c = QuantPagedKVCache(pages + 3 * samples, HKV, fmt, dev)
        c.set_page_table(torch.arange(pages), torch.tensor([0, pages]), torch.tensor([prompt - 16 * (pages - 1)]))
        self.prefix = c.table
        K.kv_quant_append(self.k0.to(dev), self.v0.to(dev), torch.tensor([0, prompt], dtype=torch.int32).to(dev), *c.pools,
                          *c.table)
        # every sample starts with an empty page of its own
        c.set_page_table(torch.arange(pages, pages + samples), torch.arange(samples + 1),
                         torch.zeros(samples, dtype=torch.int32))
        self.free = list(range(pages + samples, pages + 3 * samples))
        self.group = torch.tensor([0, samples], dtype=torch.int32, device=dev)
        self.head = (r(H * 128, V) * 0.2).to(dev)
        self.steps = [(r(samples, H, 128).to(dtype), r(samples, HKV, 128).to(dtype), r(samples, HKV, 128).to(dtype),
                       torch.rand(samples, generator=g)) for _ in range(20)]

    def device(self, q, k, v, u, **ws):
        """The recorded half of a step."""
        c = self.cache
        c.append_device(k, v)
        out, lse = K.prefix_paged_decode_attention(
            q, c.k_cache, c.v_cache, *self.prefix, self.group, *c.table, max_prefix_tokens=self.prompt,
            max_group_size=self.B, max_tokens=64, k_scale=c.k_scale, v_scale=c.v_scale, return_lse=True, **ws)
        logits = out.float().reshape(self.B, -1) @ self.head
        return out, lse, logits, K.sample_tokens(logits, u, temperature=0.8, top_k=50, top_p=0.9, min_p=0.01)

    def run(self, n):
        got = []
        for i in range(n):
            self.cache.advance_host(self.free)
            got.append([t.clone() for t in self.device(*(t.to(self.dev) for t in self.steps[i]))])
        return got


def _check(s, got):
    val = lambda x: decode(*encode(x, s.fmt)).double()  # noqa: E731
    for i, (out, lse, logits, tok) in enumerate(got):
        for b in range(s.B):
            k = torch.cat([val(s.k0)] + [val(st[1][b:b + 1]) for st in s.steps[:i + 1]])
            v = torch.cat([val(s.v0)] + [val(st[2][b:b + 1]) for st in s.steps[:i + 1]])
            check_attention(out[b].cpu(), lse[b].cpu(), attention64(s.steps[i][0][b], k, v, 128 ** -0.5), k.shape[0],
                            s.dtype, torch.float16)
            f32 = lambda x: float(torch.tensor(x))  # noqa: E731
            want, margin = sample64(logits[b].cpu(), float(s.steps[i][3][b]), f32(0.8), 50, f32(0.9), f32(0.01))
            assert margin < 1e-9 or int(tok[b]) == want


@pytest.mark.parametrize("fmt", [torch.int8, torch.float8_e4m3fn])
@pytest.mark.parametrize("samples,prompt", [(1, 17), (5, 100), (12, 700)])
def test_decode_steps_of_samples(dev, fmt, samples, prompt):
    s = Step(dev, fmt, samples, prompt)
    _check(s, s.run(18))                                   # crosses into a second page


def test_steps_on_another_stream_equal_the_default_stream(dev):
    a, b = (Step(dev, torch.int8, 4, 90, seed=3) for _ in range(2))
    want = a.run(4)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        got = b.run(4)
    stream.synchronize()
    for x, y in zip(want, got):
        assert all(torch.equal(p, q) for p, q in zip(x, y))


def test_two_recorded_steps_with_workspaces_of_their_own(dev):
    # two caches, a graph each, replayed in turn with eager work and synchronisation in between
    eager = [Step(dev, torch.float8_e4m3fn, 3, 200, seed=i) for i in range(2)]
    want = [s.run(9) for s in eager]
    steps = [Step(dev, torch.float8_e4m3fn, 3, 200, seed=i) for i in range(2)]
    graphs = []
    for s in steps:
        s.cache.reserve_page_table(3)
        s.inputs = [t.to(dev).clone() for t in s.steps[0]]
        s.ws = torch.full((K.prefix_attention_workspace_bytes(3, H, HKV, 1, 200, 3, 64),), 0xFF, dtype=torch.uint8, device=dev)
        s.cache.advance_host(s.free)
        first = [t.clone() for t in s.device(*s.inputs, workspace=s.ws)]   # the first step runs eagerly
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            s.result = s.device(*s.inputs, workspace=s.ws)
        graphs.append(g)
        s.got = [first]
    for i in range(1, 9):
        for s, g in zip(steps, graphs):
            s.cache.advance_host(s.free)
            for dst, src in zip(s.inputs, s.steps[i]):
                dst.copy_(src)
            g.replay()
            s.got.append([t.clone() for t in s.result])
        torch.cuda.synchronize()
        torch.zeros(1000, device=dev).add_(1)
    for s, w in zip(steps, want):
        for x, y in zip(s.got, w):
            assert all(torch.equal(p, q) for p, q in zip(x, y))


def test_two_streams_at_once(dev):
    # no state is shared between calls: two steps in flight on two streams equal the same steps in turn
    want = [Step(dev, torch.int8, 6, 1500, seed=i).run(3) for i in range(2)]
    steps = [Step(dev, torch.int8, 6, 1500, seed=i) for i in range(2)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for i in range(3):
        for n in range(2):
            with torch.cuda.stream(streams[n]):
                s = steps[n]
                s.cache.advance_host(s.free)
                got[n].append([t.clone() for t in s.device(*(t.to(dev) for t in s.steps[i]))])
    torch.cuda.synchronize()
    for w, g in zip(want, got):
        for x, y in zip(w, g):
            assert all(torch.equal(p, q) for p, q in zip(x, y))


def test_cache_from_dense_and_read(dev):
    k, v = torch.randn(2, 3, 45, 128).half(), torch.randn(2, 3, 45, 128).half()
    c = QuantPagedKVCache.from_dense(k, v, torch.int8, dev, spare_pages=2)
    new = torch.randn(2, 3, 128).half()
    free = [6, 7]
    for _ in range(4):                                     # 45 -> 49 tokens: a page more
        c.append(new.to(dev), new.to(dev), free)
    kk, vv = c.read(torch.float32)
    assert free == [] and kk.shape == (98, 3, 128)
    for got, x in ((kk, k), (vv, v)):
        for b in range(2):
            rows = torch.cat([x[b].transpose(0, 1)] + [new[b][None]] * 4)
            assert torch.equal(got[49 * b:49 * b + 49].cpu(), decode(*encode(rows, torch.int8)))


@pytest.mark.parametrize("dense_kv", ["int8", "e4m3"])
def test_model_with_8_bit_dense_layers(dev, dense_kv):
    """The patched model with its dense layers over 8-bit pages: close to the model over 16-bit pages (the
    codes are off by half a step: 2^-8 of a row's largest magnitude, or 2^-4 of a value, in two of four
    layers), and its recorded step equals its eager one."""
    model = _tiny_llama(layers=4, heads=4, kv_heads=2, dtype=torch.float16).to(dev)
    ids = torch.randint(0, 97, (2, 150), generator=torch.Generator().manual_seed(11)).to(dev)
    toks = torch.randint(0, 97, (2, 20), generator=torch.Generator().manual_seed(12)).to(dev)

    def decode_all(kv, graphed):
        hf.enable_sparse_attention(model, json.loads(json.dumps(CFG)), reserve_tokens=64, dense_layers="paged",
                                   keep_hf_cache=False, dense_kv=kv)
        logits, step = [], None
        with torch.no_grad():
            past = model(ids, use_cache=True).past_key_values
            for s in range(toks.shape[1]):
                if graphed and s:
                    step = step or hf.GraphedDecodeStep(model)
                    logits.append(step(toks[:, s:s + 1])[:, -1].float().clone())
                    torch.cuda.synchronize()
                else:
                    pos = torch.full((2, 1), 150 + s, device=dev)
                    logits.append(model(toks[:, s:s + 1], past_key_values=past, use_cache=True,
                                        position_ids=pos).logits[:, -1].float().clone())
        kinds = [type(layer.self_attn._twilight_state.cache).__name__ for layer in model.model.layers]
        hf.disable_sparse_attention(model)
        return torch.stack(logits), kinds

    want, _ = decode_all("model", False)
    got, kinds = decode_all(dense_kv, False)
    assert kinds == ["QuantPagedKVCache"] * 2 + ["PagedKVCache"] * 2
    assert not torch.equal(got, want)
    # a value's error of at most 2^-4 (e4m3) relative, in rows of an attention average: bounded by the
    # same share of the logits' range
    assert (got - want).abs().max() <= 2.0 ** -4 * want.abs().max() * 2
    again, _ = decode_all(dense_kv, True)
    assert torch.equal(again, got)
    with pytest.raises(RuntimeError, match="dense_layers"):
        hf.enable_sparse_attention(model, CFG, dense_kv=dense_kv)
    with pytest.raises(RuntimeError, match="dense_kv"):
        hf.enable_sparse_attention(model, CFG, dense_layers="paged", dense_kv="int4")
