"""Windowed and 8-bit attention of so many rows that a wave takes two tiles of them (512
workgroups of 128 rows and more, bf16 queries), held to float64 at sampled rows.

Bound: every weight is off by a relative `rel` (the scores' error a, twice; exp2 and the sums, 2^-21 +
2 L 2^-24; what P keeps, 16 bits over bf16 pools and fp16's 11 over 8-bit ones, whose unit is rounded
three times more), which moves a channel by rel sum p_j |V_j| at most; over 8-bit pools a product has
steps of 2^-24 in units where the row's largest is 2^13 or more: 2^-38 of it, times a code, for each
key. The output is rounded by half a step, 2^-8.
"""

import random

import pytest
import torch

from test_gpu_window import DEV, Case, i32, poison

pytestmark = pytest.mark.gpu
POOLS = ["bf16", "int8", "e4m3"]


def bound_of(c, b, t, h, window, sinks):
    """(float64 output, its bound) of one row."""
    D, G = c.q.shape[3], c.q.shape[2] // c.k.shape[1]
    see = c.sees(b, t, window, sinks)
    K, V, _ = c.values(b, see, h // G)
    q, scale = c.q[b, t, h].double(), D ** -0.5
    s = K @ q * scale
    p = torch.softmax(s, 0)
    a = float((K.abs() @ q.abs()).max() * scale) * (D + 1) * 2.0 ** -24 + 8 * 2.0 ** -24 * float(s.abs().max())
    rel = 2 * a + 2.0 ** -21 + 2 * len(see) * 2.0 ** -24
    unit = 0.0
    if c.ks is not None:
        rel += 2.0 ** -11 + 3 * 2.0 ** -24
        blk = torch.tensor([c.tables[b][j // c.bs] for j in see])
        unit = float((p * c.vs[blk, h // G].double()).max()) * (127 if c.pool == "int8" else 448)
    else:
        rel += 2.0 ** -16
    want = p @ V
    bound = rel * (p @ V.abs()) + len(see) * 2.0 ** -38 * unit + 2.0 ** -8 * want.abs()
    return want, bound * (1 + 2.0 ** -8)


def check(c, got, rows, window, sinks):
    for b, t, h in rows:
        want, bound = bound_of(c, b, t, h, window, sinks)
        off = (got[b, t, h].double() - want).abs()
        assert bool((off <= bound).all()), (b, t, h, float((off / bound).max()))


def sample(c, n, seed):
    """The first and last rows of some sequences, and any."""
    r, B, Hq = random.Random(seed), len(c.starts), c.q.shape[2]
    rows = {(b, t, r.randrange(Hq)) for b in (0, B // 2, B - 1) for t in (0, c.counts[b] - 1) if c.counts[b]}
    while len(rows) < n:
        b = r.randrange(B)
        if c.counts[b]:
            rows.add((b, r.randrange(c.counts[b]), r.randrange(Hq)))
    return rows


def two_tiles(c):
    R = c.T * c.q.shape[2] // c.k.shape[1]
    return len(c.starts) * c.k.shape[1] * -(-R // 128) >= 512 and c.dtype == "bf16"


@pytest.mark.parametrize("pool", POOLS)
@pytest.mark.parametrize("D", [64, 128])
def test_prompts(D, pool):
    """Prompts behind histories, of a length that ends inside a wave's second tile, an odd window."""
    c = Case(70, [37, 0], 2100, 16, 2, D, pool, "bf16")
    assert two_tiles(c)
    check(c, c.run(333, 17), sample(c, 60, 1), 333, 17)
    if c.ks is not None:
        check(c, c.run(), sample(c, 25, 2), None, 0)


@pytest.mark.parametrize("pool", POOLS)
@pytest.mark.parametrize("D", [64, 128])
def test_many_sequences_of_few_tokens(D, pool):
    """260 sequences of up to 9 tokens, none at all among them, over four histories; rows past a
    sequence's last keep what is there."""
    c = Case(71, [700, 64, 3, 250], 9, 16, 2, D, pool, "bf16")
    g, r, n = torch.Generator().manual_seed(D), random.Random(D), 65
    c.starts, c.tables = c.starts * n, c.tables * n
    c.counts = [r.choice([9, 9, 8, 1, 0, 5]) for _ in c.starts]
    c.q = torch.randn(4 * n, 9, 16, D, generator=g).to(torch.bfloat16)
    assert two_tiles(c)
    out = torch.full(c.q.shape, 7.0, dtype=torch.bfloat16, device=DEV)
    got = c.run(100, 5, out=out)
    check(c, got, sample(c, 60, 3), 100, 5)
    for b, m in enumerate(c.counts):
        assert bool((got[b, m:] == 7.0).all())


@pytest.mark.parametrize("pool", POOLS)
@pytest.mark.parametrize("D", [64, 128])
def test_what_no_query_sees_may_hold_anything(D, pool):
    """NaN and infinities ahead of the window, behind the last token and in their scales."""
    c = Case(72, [500, 40], 31, 64, 8, D, pool, "bf16")
    poison(c, 70, 5)
    n = 17
    c.starts, c.tables, c.counts = c.starts * n, c.tables * n, c.counts * n
    c.q = torch.randn(2 * n, 31, 64, D, generator=torch.Generator().manual_seed(D)).to(torch.bfloat16)
    assert two_tiles(c)
    check(c, c.run(70, 5), sample(c, 60, 4), 70, 5)


@pytest.mark.parametrize("pool", ["bf16", "e4m3"])
@pytest.mark.parametrize("D", [64, 128])
def test_a_non_finite_value_reaches_the_rows_that_see_it_alone(D, pool):
    c = Case(73, [200], 2100, 32, 4, D, pool, "bf16")
    assert two_tiles(c)
    window, sinks = 60, 3
    bad = [150, 222, 1000, 1063, 2299]
    clean = c.v.clone()
    for j in bad:
        c.v[c.tables[0][j // 16], :, 5, j % 16] = float("nan") if pool == "e4m3" else float("inf")
    got = c.run(window, sinks)
    c.v = clean
    rows = {(0, t, t % 32) for j in bad for t in (j - 200 - 1, j - 200, j - 200 + window - 1, j - 200 + window)
            if 0 <= t < 2100}
    keep = torch.arange(D) != 5
    for b, t, h in rows:
        hit = any(j in c.sees(b, t, window, sinks) for j in bad)
        want, bound = bound_of(c, b, t, h, window, sinks)
        x = got[b, t, h].double()
        assert bool(torch.isfinite(x[5])) is not hit, (t, h)
        off = (x - want).abs() <= bound
        assert bool((off if not hit else off[keep]).all())


@pytest.mark.parametrize("pool", ["int8", "e4m3"])
def test_scales_of_any_size(pool):
    """Scales that differ by up to 1e9 from block to block, and 0."""
    c = Case(74, [90, 0], 2100, 16, 2, 64, pool, "bf16")
    assert two_tiles(c)
    for table in c.tables:
        for i, n in enumerate(table):
            c.vs[n] *= [1.0, 1e4, 1e-5, 0.0][i % 4]
            c.ks[n] *= [1.0, 1e-6, 0.0][i % 3]
    check(c, c.run(200, 9), sample(c, 60, 5), 200, 9)


@pytest.mark.parametrize("pool", POOLS)
def test_the_same_bits_again_and_as_a_captured_graph(pool):
    c = Case(75, [5, 90], 2080, 16, 2, 128, pool, "bf16")
    assert two_tiles(c)
    first = c.run(300, 4)
    q, k, v = (t.to(DEV) for t in (c.q, c.k, c.v))
    s = [] if c.ks is None else [c.ks.to(DEV), c.vs.to(DEV)]
    table, start, ctx = c.table(), i32(c.starts), max(c.starts) + c.T
    from kvengine_amd import kernels
    fn = kernels.paged_window_attn if c.ks is None else kernels.paged_q8_attn
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = fn(q, k, v, *s, table, start, ctx, window=300, sinks=4)
    for _ in range(3):
        out.zero_()
        g.replay()
        eager = c.run(300, 4)
        torch.cuda.synchronize()
        assert torch.equal(out.cpu(), first) and torch.equal(eager, first)
