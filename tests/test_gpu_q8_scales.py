"""Attention over an 8-bit pool whose blocks have scales of very different size, held to float64
row by row: what a row does not see, or gives no weight, takes no bits from the rest.

Bound: every weight p_j is off by a relative `rel` (the scores' error a, twice, exp2 and sums; the
bits that P s_v keeps, 2^-11 for bf16 queries and 2^-22 for fp32; three roundings of the row's unit),
which moves a channel by rel sum p_j |V_j| at most. P s_v has steps of 2^-24 at the least, in units
where the row's largest product is 2^13 or more: off by half of one, 2^-38 of the largest product,
times a code, for each key. The output is rounded by half a step.
"""

import pytest
import torch

from test_gpu_window import Case

pytestmark = pytest.mark.gpu
Q8 = [(p, d) for p in ("int8", "e4m3") for d in ("bf16", "fp32")]


def check(c, got, window, sinks):
    B, T, Hq, D = c.q.shape
    G, scale = Hq // c.k.shape[1], D ** -0.5
    half = 2.0 ** -8 if c.dtype == "bf16" else 2.0 ** -24
    for b in range(B):
        for t in range(T):
            for h in range(Hq):
                see = c.sees(b, t, window, sinks)
                K, V, _ = c.values(b, see, h // G)
                q = c.q[b, t, h].double()
                s = K @ q * scale
                p = torch.softmax(s, 0)
                a = float((K.abs() @ q.abs()).max() * scale) * ((D + 1) * 2.0 ** -24 + 2.0 ** -22)
                a += 8 * 2.0 ** -24 * float(s.abs().max())
                rel = 2 * a + 2.0 ** -21 + 2 * len(see) * 2.0 ** -24 + 3 * 2.0 ** -24
                rel += 2.0 ** -11 if c.dtype == "bf16" else 2.0 ** -22
                blk = torch.tensor([c.tables[b][j // c.bs] for j in see])
                unit = float((p * c.vs[blk, h // G].double()).max()) * (127 if c.pool == "int8" else 448)
                want = p @ V
                bound = rel * (p @ V.abs()) + len(see) * 2.0 ** -38 * unit + half * want.abs()
                x = got[b, t, h].double()
                off = (x - want).abs()
                assert bool((off <= bound * (1 + half)).all()), (b, t, h, float((off / bound).max()))


@pytest.mark.parametrize("pool,dtype", Q8)
@pytest.mark.parametrize("T,Hq,D", [(2, 14, 64), (5, 14, 64), (40, 4, 128)])
@pytest.mark.parametrize("large", [1e9, 1e30])
def test_a_block_that_a_row_does_not_see(large, T, Hq, D, pool, dtype):
    """The newest blocks, which only the last rows see, and those on the window's edge, which only
    the first rows see, are larger by `large`."""
    c = Case(40 + T, [45 if T < 5 else 43, 200], T, Hq, 2, D, pool, dtype)
    last = (c.starts[0] + T - 1) // 16
    first = (200 - 60 + 1) // 16
    for blk in (c.tables[0][last], c.tables[1][first]):
        c.vs[blk] *= large
    check(c, c.run(60, 0), 60, 0)
    check(c, c.run(), None, 0)


@pytest.mark.parametrize("pool,dtype", Q8)
@pytest.mark.parametrize("T,n", [(1, 50), (1, 1500), (9, 700)])
def test_a_block_without_weight(T, n, pool, dtype):
    """Every third block is 1e12 or 1e30 times the others and its keys' scores lie so far below
    that their weight times it is nothing (2^-150 and, where exp2 gives 0, 0), or so far that it
    is as large as the rest (2^-40 times 2^40)."""
    for large, below in ((1e12, 150.0), (1e30, 2000.0), (2.0 ** 40, 40.0)):
        c = Case(50 + T, [n], T, 4, 2, 64, pool, dtype)
        c.q[..., 0] = 8.0
        c.k[:, :, :, 0] = 0
        one = c.k.clone()
        for i, blk in enumerate(c.tables[0][:-1]):
            if i % 3 == 1:
                # score = code * scale * 8 / 8 = -below ln 2
                one[blk, :, :, :] = 0
                one[blk, :, :, 0] = -64
                c.ks[blk] = below * 0.6931 / 64
                c.vs[blk] *= large
        c.k = one
        check(c, c.run(), None, 0)


@pytest.mark.parametrize("pool,dtype", Q8)
@pytest.mark.parametrize("T", [1, 9])
def test_scores_that_rise_along_the_history(T, pool, dtype):
    """From block to block scores rise by a half to 20 powers of two while scales of V fall as
    fast, faster and slower."""
    for rise, fall in ((0.5, 0.5), (2.0, 2.0), (6.0, 3.0), (3.0, 4.0), (20.0, 1.0), (9.0, 0.0)):
        c = Case(60 + T, [400], T, 4, 2, 64, pool, dtype)
        c.q[..., 0] = 8.0
        c.k[:, :, :, 0] = 64
        for i, blk in enumerate(c.tables[0]):
            c.ks[blk] = (i + 1) * rise * 0.6931 / 64
            c.vs[blk] = 2.0 ** (-fall * i) / 16
            c.k[blk, :, :, 1:] = 0
        check(c, c.run(), None, 0)
