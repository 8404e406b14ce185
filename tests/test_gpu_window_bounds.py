"""A replayed iteration passes its bucket for max_ctx where an eager pass passes start + tokens:
windowed and 8-bit attention give the same bits under both. And whole speculative runs over windows
and 8-bit pools: captured iterations against eager ones and against the model in float64."""

import pytest
import torch

from kvengine_amd import kernels
from kvengine_amd.arch import TINY
from kvengine_amd.paged import PagedKVCache
from kvengine_amd.speculative import _IterationGraphs, speculative_greedy
from test_gpu_window import DEV, Case, i32
from test_gpu_window_model import TOL, model_of, prompt, reference

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("pool", ["bf16", "int8", "e4m3"])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("T", [1, 2, 5])
def test_the_same_bits_under_every_bound_of_a_bucket(T, D, pool):
    c = Case(80 + T, [2600], T, 14, 2, D, pool, "bf16")
    q, k, v = (t.to(DEV) for t in (c.q, c.k, c.v))
    s = [] if c.ks is None else [c.ks.to(DEV), c.vs.to(DEV)]
    fn = kernels.paged_window_attn if c.ks is None else kernels.paged_q8_attn
    for window, sinks in ((800, 300), (1000, 4), (10 ** 6, 0)):
        for end in (300, 860, 896, 897, 950, 1000, 1022, 1023, 1024, 1025, 1279, 1280, 1281, 2100):
            start = i32([end - T])
            bucket = 896 if end <= 896 else -(-end // 256) * 256
            got = [fn(q, k, v, *s, c.table(), start, m, window=window, sinks=sinks)
                   for m in {end, min(end + 1, bucket), bucket}]
            assert all(torch.equal(g, got[0]) for g in got), (window, end)


@pytest.mark.parametrize("n", [45, 995])
@pytest.mark.parametrize("pool_dtype,window", [(None, 30), (None, 900), (torch.int8, None),
                                               (torch.float8_e4m3fn, 30), (torch.int8, 900)])
def test_captured_iterations_give_the_eager_ones(pool_dtype, window, n, monkeypatch):
    """Prompts of which the second passes 1024 tokens while it decodes: as many tokens accepted
    and the same tokens, K/V pools included, with graphs, replayed graphs and without."""
    model = model_of(TINY, torch.bfloat16, window, 4)
    ids = prompt(n).to(DEV)

    def run(pools):
        t, d = (p.new_sequence("s") for p in pools)
        r = speculative_greedy(model, model, ids, t, d, k=3, max_new_tokens=60, eos_token_id=None)
        kept = [x[..., :t.length, :].clone() for i in range(2) for x in t._gather(i, t.length)]
        t.free()
        d.free()
        return r.new_token_ids, r.accepted_per_iter, kept

    pools = [PagedKVCache.for_model(model, 72, dtype=pool_dtype) for _ in range(2)]
    runs = [run(pools) for _ in range(2)]
    monkeypatch.setattr(_IterationGraphs, "usable", staticmethod(lambda *a: False))
    runs.append(run([PagedKVCache.for_model(model, 72, dtype=pool_dtype) for _ in range(2)]))
    for tokens, accepted, kept in runs[1:]:
        assert tokens == runs[0][0] and accepted == runs[0][1]
        assert all(torch.equal(a, b) for a, b in zip(kept, runs[0][2]))


@pytest.mark.parametrize("pool_dtype,window", [(None, 30), (None, 900), (torch.int8, None),
                                               (torch.float8_e4m3fn, 30), (torch.int8, 900)])
def test_captured_iterations_give_the_models_own_tokens(pool_dtype, window):
    """Every token of a run with graphs, fed to the model in float64, over an 8-bit pool to the rows
    that it holds in the end: its logit is the largest but for the passes' rounding (5e-2 of the
    largest logit each way, as in the passes' own test; a row that a growing int8 scale rounds
    again moves by 2^-8 of its block's largest value, one rounding more of some twenty a layer,
    and e4m3 scales, powers of two, move no code but the smallest)."""
    model = model_of(TINY, torch.bfloat16, window, 4)
    ids = prompt(1000)
    t, d = (PagedKVCache.for_model(model, 72, dtype=pool_dtype).new_sequence("s") for _ in range(2))
    r = speculative_greedy(model, model, ids.to(DEV), t, d, k=3, max_new_tokens=60, eos_token_id=None)
    assert len(r.new_token_ids) == 60
    n = min(t.length, 1060)
    text = torch.cat([ids[0], torch.tensor(r.new_token_ids)])[:n]
    held = None
    if pool_dtype is not None:
        held = lambda li: tuple(x[0].double().cpu() for x in t._gather(li, n))
    logits = reference(model, text, held)[999:]
    new = torch.tensor(r.new_token_ids)[:logits.shape[0]]
    assert len(new) >= 55
    own = logits[:len(new)].gather(1, new[:, None])[:, 0]
    best = logits[:len(new)].max(-1).values
    assert bool((best - own <= 2 * TOL[torch.bfloat16] * logits.abs().max()).all())
    # the draft is the target: what it proposes is what is verified, but for the same rounding
    assert r.tokens_accepted >= r.tokens_drafted // 2
