"""Models with a sliding window, pools of 8-bit codes and scores of given tokens, end to end:
the operators together, as decoding and scoring use them.

Reference: the same layers in float64 on the CPU (`reference`), attention by the definition.
Over 8-bit pools its keys and values are those that the pool holds after the pass, so that
quantisation is not part of the comparison; the pool's first-layer rows are held to the
rows that went in by half a step of the block's scale for each rounding.

Tolerances. fp32: a product sum of n terms is off by at most n 2^-24 of the sum of its
magnitudes; a tiny layer's sums have 128 to 256 terms and two layers of seven sums follow
one another, 2 * 7 * 256 * 2^-24 = 2.1e-4, of the largest logit, where magnitudes do not
cancel by more than a few times: 1e-3 of it. bf16: every one of some 20 roundings a layer is
off by half a step, 2^-8, so 40 * 2^-8 = 0.16 at worst, 5 sigma of their random walk
sqrt(40) 2^-9.8 * 5 = 0.036: 5e-2.
"""

import math

import pytest
import torch

from kvengine_amd import kernels
from kvengine_amd.arch import TINY, TINY128
from kvengine_amd.decode import greedy_own_cache, greedy_paged, score_tokens
from kvengine_amd.forward import forward_hidden, forward_packed, forward_with_own_cache
from kvengine_amd.model import build_model
from kvengine_amd.paged import ContiguousKVCache, PagedKVCache
from kvengine_amd.speculative import speculative_greedy

pytestmark = pytest.mark.gpu
DEV = "cuda"
TOL = {torch.float32: 1e-3, torch.bfloat16: 5e-2}
Q8 = [torch.int8, torch.float8_e4m3fn]


def model_of(arch=TINY, dtype=torch.float32, window=None, sinks=0, fused=True):
    m = build_model(arch, seed=3, dtype=dtype, device=DEV)
    for i, layer in enumerate(m.model.layers):
        if window is not None and i % 2 == 0:  # every other layer, as mixed models have them
            layer.self_attn.sliding_window = window
            layer.self_attn.window_sinks = sinks
        if not fused:
            del layer.self_attn.qkv_weight
    return m


def reference(model, ids, held=None):
    """Logits [T, V] in float64; held(layer) -> the K and V [Hkv, T, D] to attend to."""
    m, f = model.model, torch.nn.functional
    w = lambda t: t.detach().double().cpu()
    arch = model.arch
    T, D, G = len(ids), arch.head_dim, arch.group
    x = w(m.embed_tokens.weight)[ids]
    freq = torch.outer(torch.arange(T, dtype=torch.float64), w(m.rotary_emb.inv_freq))
    cos, sin = (torch.cat([t, t], -1)[:, None] for t in (freq.cos(), freq.sin()))

    def norm(x, mod):
        return x / torch.sqrt((x * x).mean(-1, keepdim=True) + mod.variance_epsilon) * w(mod.weight)

    def rope(t):
        return t * cos + torch.cat([-t[..., D // 2:], t[..., :D // 2]], -1) * sin

    i = torch.arange(T)
    for li, layer in enumerate(m.layers):
        a, mlp = layer.self_attn, layer.mlp
        h = norm(x, layer.input_layernorm)
        q, k, v = (f.linear(h, w(p.weight), w(p.bias)).view(T, -1, D) for p in (a.q_proj, a.k_proj, a.v_proj))
        q, k, v = rope(q).transpose(0, 1), rope(k).transpose(0, 1), v.transpose(0, 1)
        if held is not None:
            k, v = held(li)
        sees = i[None] <= i[:, None]
        if a.sliding_window is not None:
            sees &= (i[None] > i[:, None] - a.sliding_window) | (i[None] < a.window_sinks)
        s = (q @ k.repeat_interleave(G, 0).transpose(1, 2) * D ** -0.5).masked_fill(~sees, -math.inf)
        o = (torch.softmax(s, -1) @ v.repeat_interleave(G, 0)).transpose(0, 1).reshape(T, -1)
        x = x + f.linear(o, w(a.o_proj.weight))
        h = norm(x, layer.post_attention_layernorm)
        x = x + f.linear(f.silu(f.linear(h, w(mlp.gate_proj.weight))) * f.linear(h, w(mlp.up_proj.weight)),
                         w(mlp.down_proj.weight))
    return f.linear(norm(x, m.norm), w(model.lm_head.weight))


def prompt(n, vocab=1000, seed=1):
    return torch.randint(0, vocab, (1, n), generator=torch.Generator().manual_seed(seed))


def close(got, want, dtype):
    off = (got.double().cpu() - want).abs().max()
    assert float(off) <= TOL[dtype] * float(want.abs().max()), float(off / want.abs().max())


def passes(model, ids, cache, cuts):
    """Logits of all tokens from passes over ids in pieces."""
    out, a = [], 0
    for b in cuts + [ids.shape[1]]:
        out.append(forward_with_own_cache(model, ids[:, a:b].to(DEV), cache, all_logits=True)[0])
        a = b
    return torch.cat(out)


@pytest.mark.parametrize("fused", [True, False])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("arch,window,sinks", [(TINY, 24, 0), (TINY, 7, 5), (TINY128, 64, 4)])
def test_a_windowed_model(arch, window, sinks, dtype, fused):
    model = model_of(arch, dtype, window, sinks, fused)
    ids = prompt(150)
    pool = PagedKVCache.for_model(model, 16)
    got = passes(model, ids, pool.new_sequence("a"), [90, 91, 92, 97, 130])
    close(got, reference(model, ids[0]), dtype)
    # the contiguous cache, of any capacity
    for room in (160, 151):
        got = passes(model, ids, ContiguousKVCache.for_model(model, room), [149])
        close(got, reference(model, ids[0]), dtype)


@pytest.mark.parametrize("pool_dtype", Q8)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("arch,window,bs", [(TINY, None, 16), (TINY, 20, 32), (TINY128, None, 16)])
def test_a_pass_over_an_8bit_pool(arch, window, bs, dtype, pool_dtype):
    model = model_of(arch, dtype, window, 3)
    ids = prompt(100)
    pool = PagedKVCache.for_model(model, 16, block_size=bs, dtype=pool_dtype)
    assert pool.nbytes() < PagedKVCache.for_model(model, 16, block_size=bs).nbytes() * 0.6
    seq = pool.new_sequence("a")
    got = forward_with_own_cache(model, ids.to(DEV), seq, all_logits=True)[0]
    held = lambda li: tuple(t[0].double().cpu() for t in seq._gather(li, 100))
    close(got, reference(model, ids[0], held), dtype)
    if dtype is torch.float32:
        plain = PagedKVCache.for_model(model, 16, block_size=bs)
        ref = plain.new_sequence("b")
        forward_with_own_cache(model, ids.to(DEV), ref)
        for got, want, s in zip(seq._gather(0, 100), ref._gather(0, 100), (pool.k_scale, pool.v_scale)):
            # (K and V of one pass, rounded once: half a code's step; fp32 differences of the
            # two passes' products, 128 terms, are below 2^-16 of the largest value)
            step = s[0][torch.tensor(seq.blocks, device=DEV)].repeat_interleave(bs, 0)[:100].t()[None, :, :, None]
            half = step / 2 if pool_dtype is torch.int8 else torch.maximum(want.abs() * 2.0 ** -4, step * 2.0 ** -10)
            assert bool(((got - want).abs() <= half * 1.001 + want.abs().max() * 2.0 ** -16).all())


@pytest.mark.parametrize("pool_dtype", Q8)
def test_decoding_over_an_8bit_pool_reads_what_it_wrote(pool_dtype):
    """Token after token, with a rollback between: each step's logits are those of attention
    to what the pool holds."""
    model = model_of(TINY, torch.float32, 33, 2)
    ids = prompt(80)
    pool = PagedKVCache.for_model(model, 16, dtype=pool_dtype)
    seq = pool.new_sequence("a")
    forward_with_own_cache(model, ids[:, :50].to(DEV), seq)
    forward_with_own_cache(model, prompt(9, seed=5).to(DEV), seq)  # drafts that are rejected
    seq.truncate(50)
    for t in range(50, 80):
        got = forward_with_own_cache(model, ids[:, t:t + 1].to(DEV), seq)[0]
        if t % 7 == 0 or t > 77:
            n = t + 1
            held = lambda li: tuple(x[0].double().cpu() for x in seq._gather(li, n))
            close(got[0], reference(model, ids[0, :n], held)[-1], torch.float32)


@pytest.mark.parametrize("pool_dtype,window", [(None, 40), (torch.int8, None), (torch.float8_e4m3fn, None),
                                               (torch.int8, 40), (torch.float8_e4m3fn, 40)])
def test_scores_of_a_text(pool_dtype, window):
    """The pass, the cache's type and the window, and the log probabilities, against float64;
    rows in more pieces than one."""
    from kvengine_amd import decode
    model = model_of(TINY, torch.float32, window, 4)
    ids = prompt(120)
    pool = PagedKVCache.for_model(model, 16, dtype=pool_dtype)
    seq = pool.new_sequence("a")
    was, decode.SCORE_ROWS = decode.SCORE_ROWS, 50
    try:
        lp, H, top_ids, top = score_tokens(model, ids.to(DEV), seq, top=5)
    finally:
        decode.SCORE_ROWS = was
    held = None if pool_dtype is None else lambda li: tuple(x[0].double().cpu() for x in seq._gather(li, 120))
    logits = reference(model, ids[0], held)
    w = torch.log_softmax(logits[:-1], -1)
    tol = 4 * TOL[torch.float32] * float(logits.abs().max())
    assert lp.shape == H.shape == (119,) and top_ids.shape == top.shape == (119, 5)
    assert float((lp.double().cpu() - w.gather(1, ids[0, 1:, None])[:, 0]).abs().max()) <= tol
    assert float((H.double().cpu() + (w.exp() * w).sum(-1)).abs().max()) <= tol * 2
    assert float((top.double().cpu() - w.topk(5, -1).values).abs().max()) <= tol
    assert seq.length == 120


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("pool_dtype,window", [(None, 30), (torch.int8, None), (torch.float8_e4m3fn, 30)])
def test_speculative_decoding(pool_dtype, window, dtype):
    """Drafts from the model itself, bf16 iterations as captured graphs, twice: the same tokens
    both times, the caches at the right length, all blocks given back."""
    model = model_of(TINY, dtype, window, 4)
    ids = prompt(45).to(DEV)
    runs = []
    tp, dp = (PagedKVCache.for_model(model, 32, dtype=pool_dtype) for _ in range(2))
    for _ in range(2):
        t, d = tp.new_sequence("t"), dp.new_sequence("d")
        r = speculative_greedy(model, model, ids, t, d, k=3, max_new_tokens=40, eos_token_id=None)
        assert len(r.new_token_ids) == 40
        runs.append(r.new_token_ids)
        t.free()
        d.free()
    assert tp.manager.num_free == dp.manager.num_free == 32
    if pool_dtype is None and dtype is torch.float32:
        g = greedy_paged(model, ids, tp, max_new_tokens=40, eos_token_id=None)
        assert g.new_token_ids[:40] == runs[0]
    assert runs[0] == runs[1]


def test_greedy_decoding_over_either_cache():
    model = model_of(TINY, torch.float32, 9, 2)
    ids = prompt(21).to(DEV)
    a = greedy_own_cache(model, ids, max_new_tokens=14, eos_token_id=None)
    b = greedy_paged(model, ids, PagedKVCache.for_model(model, 8), max_new_tokens=14, eos_token_id=None)
    assert len(a.new_token_ids) == 14 and a.new_token_ids == b.new_token_ids


def test_windows_set_between_calls_are_seen():
    """The same models and pools, other windows: captured iterations of the first call do not
    serve the second."""
    model = model_of(TINY, torch.bfloat16)
    ids = prompt(60).to(DEV)
    tp, dp = (PagedKVCache.for_model(model, 32) for _ in range(2))

    def run():
        t, d = tp.new_sequence("t"), dp.new_sequence("d")
        r = speculative_greedy(model, model, ids, t, d, k=3, max_new_tokens=30, eos_token_id=None)
        t.free()
        d.free()
        return r.new_token_ids

    plain = run()
    for layer in model.model.layers:
        layer.self_attn.sliding_window = 4
    short = run()
    assert short != plain
    tp, dp = (PagedKVCache.for_model(model, 32) for _ in range(2))
    assert run() == short


@pytest.mark.parametrize("pool_dtype", Q8)
def test_the_cache_protocol_over_8bit_blocks(pool_dtype):
    """write() takes rows of any layout and gives the history in their type."""
    pool = PagedKVCache(1, 2, 64, 4, 16, pool_dtype, DEV)
    seq = pool.new_sequence("a")
    g = torch.Generator().manual_seed(2)
    for n, start in ((5, 0), (1, 5), (20, 6)):
        seq.reserve(n)
        # (one row: the strides of dimensions of one differ between the two)
        k = torch.randn(1, 2, n, 64, generator=g).to(DEV, torch.bfloat16)
        v = torch.randn(1, n, 2, 64, generator=g).to(DEV, torch.bfloat16).transpose(1, 2)
        hk, hv = seq.write(0, k, v, start)
        seq.commit(n)
        assert hk.dtype == hv.dtype == torch.bfloat16 and hk.shape == (1, 2, start + n, 64)
        for h, x in ((hk, k), (hv, v)):
            # half a step of the largest, 2^-4 relative for e4m3 and 1 / 254 for int8, and bf16's own
            assert float((h[:, :, start:] - x).abs().max()) <= float(x.abs().max()) * (2 ** -4 + 2 ** -8)


def test_refusals():
    model = model_of(TINY, torch.bfloat16, 16)
    plain = model_of(TINY, torch.bfloat16)
    q8 = PagedKVCache.for_model(plain, 16, dtype=torch.int8)
    for m, pool in ((model, PagedKVCache.for_model(model, 16)), (plain, q8)):
        seq = pool.new_sequence("a")
        seq.reserve(4)
        kv, ids = seq.device_kv(), prompt(4).to(DEV)
        tree = kernels.tree_masks(torch.tensor([[-1, 0, 0, 1]], dtype=torch.int32, device=DEV))
        with pytest.raises(NotImplementedError):
            forward_hidden(m, ids, kv, seq.row_dev, 16, tree=tree)
        with pytest.raises((NotImplementedError, ValueError)):
            forward_hidden(m, ids, kv, seq.row_dev, 16, blocked_out=True)
        with pytest.raises(NotImplementedError):
            forward_packed(m, ids[0], torch.arange(4, device=DEV), 1, 4, kv, seq.row_dev, 16,
                           torch.tensor([4], dtype=torch.int32, device=DEV))
    from kvengine_amd.engine import SpecEngine
    for pair in ((model, plain), (plain, model)):
        with pytest.raises(NotImplementedError):
            SpecEngine(*pair, k=2, slots=2, t_blocks=16, d_blocks=16)
    with pytest.raises(ValueError):
        PagedKVCache.for_model(plain, 16, block_size=8, dtype=torch.int8)
    for ids in (prompt(1), prompt(8).view(2, 4), prompt(4)[0]):
        with pytest.raises(ValueError):
            score_tokens(plain, ids.to(DEV), PagedKVCache.for_model(plain, 4).new_sequence("s"))


@pytest.mark.parametrize("pool_dtype", Q8)
def test_captured_steps_replay(pool_dtype):
    """A decode step (write, attention with a window, scores) of two batches in two captured
    graphs, replayed in turn while eager steps run between: every replay gives what the eager
    step on a copy of the same state gives, bit for bit."""
    Hkv, G, D, bs, V, n = 2, 3, 64, 16, 777, 3
    g = torch.Generator().manual_seed(4)
    head = torch.randn(V, Hkv * G * D, generator=g).to(DEV, torch.bfloat16)

    def state():
        tables = torch.arange(n * 8, dtype=torch.int32).view(n, 8).to(DEV)
        return dict(k=torch.zeros(n * 8, Hkv, bs, D, dtype=pool_dtype, device=DEV),
                    v=torch.zeros(n * 8, Hkv, D, bs, dtype=pool_dtype, device=DEV),
                    ks=torch.zeros(n * 8, Hkv, device=DEV), vs=torch.zeros(n * 8, Hkv, device=DEV),
                    tables=tables, lens=torch.tensor([0, 17, 40], dtype=torch.int32, device=DEV),
                    x=torch.zeros(n, 1, (G + 2) * Hkv * D, dtype=torch.bfloat16, device=DEV),
                    ids=torch.zeros(n, dtype=torch.int32, device=DEV))

    def step(s):
        q, k, v = (t.view(n, 1, -1, D).contiguous()
                   for t in s["x"].split([G * Hkv * D, Hkv * D, Hkv * D], -1))
        kernels.kv_write_q8(k, v, s["k"], s["v"], s["ks"], s["vs"], s["tables"], s["lens"])
        o = kernels.paged_q8_attn(q, s["k"], s["v"], s["ks"], s["vs"], s["tables"], s["lens"], 128,
                                  window=24, sinks=2)
        out = kernels.token_logprobs(torch.nn.functional.linear(o.view(n, -1), head), s["ids"], top=4)
        s["lens"].add_(1)
        return (o, *out)

    live, copy = [state() for _ in range(2)], [state() for _ in range(2)]
    graphs, outs = [], []
    stream = torch.cuda.Stream()
    for s in live:
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            step(s)
        torch.cuda.current_stream().wait_stream(stream)
        fresh = state()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            out = step(s)
        torch.cuda.synchronize()
        for key in s:
            s[key].copy_(fresh[key])
        graphs.append(graph)
        outs.append(out)
    for t in range(20):
        for s, c in zip(live, copy):
            x = torch.randn(s["x"].shape, generator=g).to(DEV, torch.bfloat16) * 2.0 ** (t % 5)
            ids = torch.randint(0, V, (n,), generator=g).to(DEV, torch.int32)
            for d in (s, c):
                d["x"].copy_(x)
                d["ids"].copy_(ids)
        for graph in graphs:
            graph.replay()
        if t % 3 == 0:
            torch.cuda.synchronize()
        for s, c, out in zip(live, copy, outs):
            want = step(c)
            for a, b in zip(out, want):
                assert torch.equal(a, b), t
            for key in ("ks", "vs", "lens"):
                assert torch.equal(s[key], c[key])
            assert torch.equal(s["k"].view(torch.uint8), c["k"].view(torch.uint8))
            assert torch.equal(s["v"].view(torch.uint8), c["v"].view(torch.uint8))
