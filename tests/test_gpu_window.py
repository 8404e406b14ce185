"""Attention with a sliding window and sinks, and attention over an 8-bit cache, held to
float64 attention over the same inputs, element by element, by a bound taken from the
inputs:

* a score is a sum of D products in fp32, off by at most (D + 1) 2^-24 sum|q k| scale (codes
  and bf16 multiply exactly), and by 2^-22 of the same where fp32 queries meet 8-bit codes (two
  fp16 of 11 bits), and is rounded a few times more on its way into the exponent (8
  roundings of values up to max|score|): =: a. A weight is then off by a relative 2 a
  (itself and the sum that divides it), exp2 and the sums over L keys add 2^-21 + 2 L 2^-24;
* a weight keeps 16 bits over a bf16 pool (2^-16; 8, 2^-8, in passes of more than 64 rows a
  kv head), and over 8-bit ones fp16's 11 (2^-11, bf16
  queries) or 22 (2^-22); in units of the largest scale that a walk has seen (less than
  twice it), 2^14 of them, it has steps of 2^-24 at the least: 2^-38 of that scale, over L keys,
  times a code;
* each relative error of a weight moves an output by at most that times max|v|, and the
  output is rounded by half a step (2^-8 bf16, 2^-24 fp32).
"""

import random

import pytest
import torch

from kvengine_amd import kernels

pytestmark = pytest.mark.gpu
DEV = "cuda"
DT = {"bf16": torch.bfloat16, "fp32": torch.float32, "int8": torch.int8, "e4m3": torch.float8_e4m3fn}


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


class Case:
    """Sequences over a paged pool in the kernel layout, on the CPU."""

    def __init__(self, seed, starts, T, Hq, Hkv, D, pool="bf16", dtype="bf16", bs=16, counts=None):
        g = torch.Generator().manual_seed(seed)
        self.starts, self.T, self.bs, self.pool, self.dtype = starts, T, bs, pool, dtype
        self.counts = counts or [T] * len(starts)
        need = [-(-(s + T) // bs) for s in starts]
        nb = sum(need) + 3
        ids = torch.randperm(nb, generator=g).tolist()
        self.tables = [[ids.pop() for _ in range(n)] for n in need]
        k, v = torch.randn(nb, Hkv, bs, D, generator=g), torch.randn(nb, Hkv, D, bs, generator=g)
        self.ks = self.vs = None
        if pool in ("int8", "e4m3"):
            # codes over the whole range, scales that differ by block
            self.ks, self.vs = (torch.exp(torch.randn(nb, Hkv, generator=g)) / 64 for _ in range(2))
            hi = 127 if pool == "int8" else 448
            k, v = ((32 * t).clamp(-hi, hi) for t in (k, v))
            k, v = (t.round() if pool == "int8" else t for t in (k, v))
        self.k, self.v = k.to(DT[pool]), v.to(DT[pool])
        self.q = torch.randn(len(starts), T, Hq, D, generator=g).to(DT[dtype])

    def table(self):
        w = max(len(t) for t in self.tables)
        return i32([t + [-1] * (w - len(t)) for t in self.tables])

    def run(self, window=None, sinks=0, out=None, **kw):
        q, k, v = (t.to(DEV) for t in (self.q, self.k, self.v))
        q_lens = None if self.counts == [self.T] * len(self.starts) else i32(self.counts)
        args = (self.table(), i32(self.starts), max(self.starts) + self.T)
        if self.ks is None:
            got = kernels.paged_window_attn(q, k, v, *args, window, sinks, q_lens=q_lens, out=out, **kw)
        else:
            got = kernels.paged_q8_attn(q, k, v, self.ks.to(DEV), self.vs.to(DEV), *args, window=window,
                                        sinks=sinks, q_lens=q_lens, out=out, **kw)
        torch.cuda.synchronize()
        return got.cpu()

    def sees(self, b, t, window, sinks):
        p = self.starts[b] + t
        return [j for j in range(p + 1) if window is None or j > p - window or j < sinks]

    def values(self, b, see, h):
        """K, V [L, D] of the keys in float64, their blocks' V scales (ones without any)."""
        blk = torch.tensor([self.tables[b][j // self.bs] for j in see])
        off = torch.tensor([j % self.bs for j in see])
        K, V = self.k[blk, h, off].double(), self.v[blk, h, :, off].double()
        if self.ks is None:
            return K, V, 0.0
        return (K * self.ks[blk, h].double()[:, None], V * self.vs[blk, h].double()[:, None],
                float(2 * self.vs[blk, h].max() * self.v[blk, h, :, off].float().abs().max()))

    def exact(self, b, t, h, window, sinks, scale=None):
        """(float64 output, its bound) of one row."""
        D, G = self.q.shape[3], self.q.shape[2] // self.k.shape[1]
        scale = D ** -0.5 if scale is None else scale
        see = self.sees(b, t, window, sinks)
        K, V, unit = self.values(b, see, h // G)
        q = self.q[b, t, h].double()
        s = K @ q * scale
        out = torch.softmax(s, 0) @ V
        e8 = self.ks is not None
        a = float((K.abs() @ q.abs()).max() * scale)
        a = a * ((D + 1) * 2.0 ** -24 + (2.0 ** -22 if e8 and self.dtype == "fp32" else 0.0))
        a += 8 * 2.0 ** -24 * float(s.abs().max())
        rel = 2 * a + 2.0 ** -21 + 2 * len(see) * 2.0 ** -24
        if e8:
            rel += 2.0 ** -11 if self.dtype == "bf16" else 2.0 ** -22
        elif self.dtype == "bf16":
            rel += 2.0 ** -16 if self.T * G <= 64 else 2.0 ** -8
        half = 2.0 ** -8 if self.dtype == "bf16" else 2.0 ** -24
        bound = rel * float(V.abs().max()) + half * out.abs() + len(see) * 2.0 ** -38 * unit
        return out, bound * (1 + half)

    def check(self, got, window, sinks, scale=None, rows=None):
        B, T, Hq, D = self.q.shape
        for b in range(B):
            for t in range(self.counts[b]):
                for h in range(Hq):
                    if rows is not None and (b, t, h) not in rows:
                        continue
                    want, bound = self.exact(b, t, h, window, sinks, scale)
                    off = (got[b, t, h].double() - want).abs()
                    assert bool((off <= bound).all()), (b, t, h, float((off / bound).max()))


SHAPES = [
    # starts, T, Hq, Hkv, D, bs, window, sinks
    ([0], 1, 2, 2, 64, 16, 1, 0),
    ([0, 1, 15, 16, 17], 1, 14, 2, 64, 16, 5, 2),
    ([33, 0, 700], 3, 16, 2, 128, 16, 40, 4),
    ([33, 90, 700], 5, 14, 2, 64, 16, 33, 33),
    ([50, 640], 4, 16, 1, 128, 32, 64, 1),     # 64 rows: two row waves at D = 128
    ([100, 7], 9, 14, 2, 64, 48, 100, 16),      # blocks that are no power of two
    ([0, 20], 70, 8, 2, 64, 16, 17, 3),         # 280 rows: several row groups
    ([3, 200], 41, 16, 2, 128, 64, 90, 0),      # 328 rows
    ([12], 40, 1, 1, 128, 16, 1000, 0),         # the window holds everything
    ([900], 2, 3, 1, 64, 16, 1, 1000),          # the sinks hold everything
    ([5000], 1, 14, 2, 64, 16, 4500, 5),        # chunks and their merge
    ([4000, 1], 6, 8, 1, 128, 16, 2500, 70),
]
POOLS = [("bf16", "bf16"), ("fp32", "fp32"), ("int8", "bf16"), ("e4m3", "bf16"), ("int8", "fp32"),
         ("e4m3", "fp32")]


@pytest.mark.parametrize("pool,dtype", POOLS)
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: f"{len(s[0])}x{s[1]}_{s[2]}h{s[4]}_w{s[6]}_{s[7]}")
def test_window(shape, pool, dtype):
    starts, T, Hq, Hkv, D, bs, window, sinks = shape
    c = Case(hash(shape[1:]) % 1000, starts, T, Hq, Hkv, D, pool, dtype, bs)
    rows = None
    if len(starts) * T * Hq > 300:  # some rows of each tile
        r = random.Random(1)
        rows = {(b, t, h) for b in range(len(starts)) for t in range(T) for h in range(Hq)
                if t in (0, T - 1) or r.random() < 200 / (len(starts) * T * Hq)}
    c.check(c.run(window, sinks), window, sinks, rows=rows)


@pytest.mark.parametrize("pool,dtype", [p for p in POOLS if p[0] in ("int8", "e4m3")])
@pytest.mark.parametrize("starts,T,Hq,Hkv,D,bs", [([0], 1, 4, 1, 64, 16), ([17, 300, 64], 2, 14, 2, 64, 16),
                                                  ([1100, 5], 5, 16, 2, 128, 32),
                                                  ([6000], 1, 8, 1, 128, 16), ([0, 9], 100, 4, 2, 128, 16)])
def test_q8_without_a_window(starts, T, Hq, Hkv, D, bs, pool, dtype):
    c = Case(T + D, starts, T, Hq, Hkv, D, pool, dtype, bs)
    rows = {(b, t, h) for b in range(len(starts)) for t in range(T) for h in range(Hq)
            if t < 3 or t >= T - 3 or t % 17 == 0}
    c.check(c.run(), None, 0, rows=rows)


@pytest.mark.parametrize("pool,dtype", POOLS)
@pytest.mark.parametrize("T,G,bs", [(1, 1, 16), (9, 2, 32)])
def test_walks_of_many_steps(T, G, bs, pool, dtype):
    """So many sequences that no walk is cut: 64 with one history (and block table), one of
    them shorter, over scales that grow along it."""
    c = Case(20 + T, [5000], T, 8 * G, 8, 64, pool, dtype, bs)
    if c.ks is not None:
        for i, n in enumerate(c.tables[0]):
            c.vs[n] *= 2.0 ** (i * 16 // (5000 // bs))
    c.starts, c.tables, c.counts = [5000] * 63 + [4990], c.tables * 64, [T] * 64
    g = torch.Generator().manual_seed(T)
    c.q = torch.randn(64, T, 8 * G, 64, generator=g).to(c.q.dtype)
    rows = {(b, t, (b + t) % (8 * G)) for b in (0, 17, 62, 63) for t in (0, T - 1)}
    c.check(c.run(4900, 33), 4900, 33, rows=rows)
    if c.ks is not None:
        c.check(c.run(), None, 0, rows=rows)


@pytest.mark.parametrize("pool,dtype", POOLS)
def test_ragged_rows_and_skipped_sequences_keep_what_is_there(pool, dtype):
    c = Case(3, [30, 5, 400, 64], 6, 14, 2, 64, pool, dtype, counts=[6, 0, 3, 1])
    out = torch.full((4, 6, 14, 64), 7.0, dtype=DT[dtype], device=DEV)
    got = c.run(50, 4, out=out)
    c.check(got, 50, 4)
    for b, n in enumerate(c.counts):
        assert bool((got[b, n:] == 7.0).all())
    # a row outside the tables, and a history past max_ctx
    q, k, v = (t.to(DEV) for t in (c.q, c.k, c.v))
    s = [] if c.ks is None else [c.ks.to(DEV), c.vs.to(DEV)]
    fn = kernels.paged_window_attn if c.ks is None else kernels.paged_q8_attn
    out.fill_(7.0)
    got = fn(q, k, v, *s, c.table(), i32([30, 5, 400, 64]), 100, window=50, sinks=4,
             seq_rows=i32([-1, 1, 2, 4]), out=out).cpu()
    assert bool((got[[0, 2, 3]] == 7.0).all()) and bool((got[1] != 7.0).any())


def poison(c, window, sinks):
    """NaN and infinities wherever no query of the pass looks, in K, V and scales; entries of
    blocks that none sees name no block."""
    big = {"bf16": float("inf"), "fp32": float("inf"), "e4m3": float("nan")}.get(c.pool)
    seen = set()
    for b in range(len(c.starts)):
        for t in range(c.counts[b]):
            seen |= {(c.tables[b][j // c.bs], j % c.bs) for j in c.sees(b, t, window, sinks)}
    blocks = {n for n, _ in seen}
    for n in range(c.k.shape[0]):
        for o in range(c.bs):
            if (n, o) not in seen and big is not None:
                c.k[n, :, o] = float("nan")
                c.v[n, :, :, o] = big
        if n not in blocks and c.ks is not None:
            c.ks[n] = float("nan")
            c.vs[n] = float("inf")
    for t in c.tables:
        for i, n in enumerate(t):
            if n not in blocks:
                t[i] = -1 if i % 2 else 1 << 30


@pytest.mark.parametrize("pool,dtype", POOLS)
def test_what_no_query_sees_may_hold_anything(pool, dtype):
    c = Case(5, [0, 37, 500, 1300], 4, 14, 2, 64, pool, dtype)
    poison(c, 70, 5)
    c.check(c.run(70, 5), 70, 5)


@pytest.mark.parametrize("pool,dtype", [p for p in POOLS if p[0] != "int8"])
@pytest.mark.parametrize("T,D", [(5, 64), (40, 128)])
def test_a_non_finite_value_reaches_the_rows_that_see_it_alone(pool, dtype, T, D):
    """K and V of a few keys at the window's and the sequence's edges: rows that see such a V
    are not finite in its channel, the others are as without it."""
    c = Case(6, [200, 0], T, 8, 2, D, pool, dtype)
    window, sinks = 60, 3
    bad = {0: [200 + T // 2, 200 - window + T // 2, 150], 1: [T - 1, 2]}
    clean = c.v.clone()
    value = float("nan") if pool == "e4m3" else float("inf")
    for b, keys in bad.items():
        for j in keys:
            c.v[c.tables[b][j // 16], :, 5, j % 16] = value
    got = c.run(window, sinks)
    c.v = clean
    for b in range(2):
        for t in range(T):
            hit = any(j in c.sees(b, t, window, sinks) for j in bad[b])
            for h in (0, 7):
                want, bound = c.exact(b, t, h, window, sinks)
                x = got[b, t, h].double()
                assert bool(torch.isfinite(x[5])) is not hit, (b, t, h)
                keep = torch.arange(D) != 5
                assert bool(((x - want).abs() <= bound)[keep].all())
                if not hit:
                    assert bool(((x - want).abs() <= bound).all())


@pytest.mark.parametrize("pool", ["int8", "e4m3"])
def test_a_scale_that_is_no_number_reaches_the_rows_that_see_its_block_alone(pool):
    c = Case(7, [64, 64], 20, 4, 2, 64, pool, "bf16")
    c.vs[c.tables[0][5]] = float("nan")  # keys 80 .. 95: rows from t = 16 on
    c.ks[c.tables[1][5]] = float("nan")
    got = c.run(30, 0)
    for b in range(2):
        for t in range(20):
            for h in range(4):
                if 64 + t >= 80:
                    assert bool(torch.isnan(got[b, t, h]).all())
                else:
                    want, bound = c.exact(b, t, h, 30, 0)
                    assert bool(((got[b, t, h].double() - want).abs() <= bound).all())


@pytest.mark.parametrize("pool,dtype", POOLS)
def test_scales_and_queries_of_any_size(pool, dtype):
    """Blocks a million times larger or smaller than others, zero blocks, large and tiny
    queries, a scale of the caller's."""
    c = Case(8, [300, 40], 3, 14, 2, 64, pool, dtype)
    if c.ks is not None:
        for i, n in enumerate(c.tables[0]):
            c.vs[n] *= [1.0, 1e6, 1e-6, 0.0][i % 4]
            c.ks[n] *= [1.0, 1e-6, 0.0][i % 3]
    c.q[:, 0] *= 1e4
    c.q[:, 1] *= 1e-30
    got = c.run(200, 17, scale=0.02)
    c.check(got, 200, 17, scale=0.02)


@pytest.mark.parametrize("pool,dtype", POOLS)
def test_a_window_of_everything_is_verify_attention(pool, dtype):
    """(and, over 8-bit pools, attention without a window)"""
    c = Case(9, [300, 40], 3, 14, 2, 64, pool, dtype)
    wide = c.run(10 ** 9, 0)
    c.check(wide, None, 0)
    if c.ks is not None:
        assert torch.equal(wide, c.run())
        return
    q, k, v = (t.to(DEV) for t in (c.q, c.k, c.v))
    other = kernels.paged_verify_attn(q, k, v, c.table(), i32(c.starts), 303).cpu()
    c.check(other, None, 0)


@pytest.mark.parametrize("pool,dtype", POOLS)
@pytest.mark.parametrize("T", [1, 40])
def test_scores_far_below_zero(T, pool, dtype):
    """Scores of -2^105 and lower: the first key's is the largest by more than 2^104, so the
    rows are its V."""
    c = Case(13, [60], T, 4, 2, 64, pool, dtype)
    c.q.zero_()
    c.q[..., 0] = 2.0 ** 52
    c.k.zero_()
    size = 2.0 ** 56
    if c.ks is not None:
        c.ks[:], c.vs[:] = 2.0 ** 50, 1.0
        size = 64.0
    c.k[:, :, :, 0] = -1.5 * size
    c.k[c.tables[0][0], :, 0, 0] = -size
    got = c.run(200, 0)
    want = c.v[c.tables[0][0], :, :, 0].float().repeat_interleave(2, 0).to(c.q.dtype)
    assert torch.equal(got, want.expand(1, T, 4, 64))


@pytest.mark.parametrize("pool,dtype", [("bf16", "bf16"), ("int8", "fp32")])
def test_prompts_of_more_than_2_16_rows(pool, dtype):
    c = Case(14, [3], 8300, 16, 2, 64, pool, dtype)
    r = random.Random(2)
    rows = {(0, t, h) for t in [0, 1, 4094, 4095, 4096, 8190, 8191, 8192, 8299] + r.sample(range(8300), 12)
            for h in (0, 7, 8, 15)}
    got = c.run(50, 3)
    for b, t, h in rows:
        want, bound = c.exact(b, t, h, 50, 3)
        assert bool(((got[b, t, h].double() - want).abs() <= bound).all()), (t, h)


def test_a_bf16_pool_past_32_bits():
    """More than 4 GiB of K and V each, the sequences in the last blocks; 16 rows and more."""
    nb, Hkv, D = 550_000, 2, 128
    for T in (2, 9):
        c = Case(15, [100, 70], T, 16, Hkv, D)
        n = c.k.shape[0]
        k, v = (torch.zeros(s, dtype=torch.bfloat16, device=DEV) for s in ((nb, Hkv, 16, D), (nb, Hkv, D, 16)))
        assert k.numel() * 2 > 1 << 32
        for big, small in ((k, c.k), (v, c.v)):
            big[nb - n:] = small.to(DEV)
        table = torch.where(c.table() < 0, -1, c.table() + (nb - n))
        got = kernels.paged_window_attn(c.q.to(DEV), k, v, table, i32(c.starts), 100 + T, 64, 5).cpu()
        c.check(got, 64, 5)


def test_offsets_past_32_bits():
    """A pool of more than 4 GiB of codes, the sequences in its last blocks."""
    nb, Hkv, D = 1_100_000, 2, 128
    c = Case(10, [100, 70], 2, 16, Hkv, D, "int8", "bf16")
    n = c.k.shape[0]
    k = torch.zeros(nb, Hkv, 16, D, dtype=torch.int8, device=DEV)
    v = torch.zeros(nb, Hkv, D, 16, dtype=torch.int8, device=DEV)
    ks, vs = torch.zeros(nb, Hkv, device=DEV), torch.zeros(nb, Hkv, device=DEV)
    assert k.numel() > 1 << 32
    for big, small in ((k, c.k), (v, c.v), (ks, c.ks), (vs, c.vs)):
        big[nb - n:] = small.to(DEV)
    table = torch.where(c.table() < 0, -1, c.table() + (nb - n))
    got = kernels.paged_q8_attn(c.q.to(DEV), k, v, ks, vs, table, i32(c.starts), 102).cpu()
    c.check(got, None, 0)


@pytest.mark.parametrize("pool,dtype", POOLS)
def test_the_same_bits_twice_and_on_another_stream(pool, dtype):
    c = Case(11, [2000, 31], 5, 16, 2, 128, pool, dtype)
    first = c.run(1500, 4)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = c.run(1500, 4)
    assert torch.equal(first, second)


def test_two_captured_calls_share_nothing():
    """Two graphs of calls that need a workspace, replayed in turn with eager calls between."""
    cases = [Case(12 + i, [3000 + i, 900], 2, 14, 2, 64, "int8", "bf16") for i in range(2)]
    want = [c.run() for c in cases]
    graphs = []
    for c in cases:
        ops = [t.to(DEV) for t in (c.q, c.k, c.v, c.ks, c.vs)]
        table, start, ctx = c.table(), i32(c.starts), max(c.starts) + 2
        torch.cuda.synchronize()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            kernels.paged_q8_attn(*ops, table, start, ctx)
        torch.cuda.current_stream().wait_stream(side)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = kernels.paged_q8_attn(*ops, table, start, ctx)
        graphs.append((g, out, ops, table, start))
    for i in range(6):
        for (g, out, *_), w in zip(graphs, want):
            out.fill_(0)
            g.replay()
        eager = cases[i % 2].run()
        torch.cuda.synchronize()
        for (g, out, *_), w in zip(graphs, want):
            assert torch.equal(out.cpu(), w)
        assert torch.equal(eager, want[i % 2])
