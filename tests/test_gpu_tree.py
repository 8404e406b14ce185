"""Trees of drafted tokens on the GPU: masks and depths, attention over the paged cache,
the accept that moves the accepted path's K/V, and the whole of it driven by a model.

The attention is held to float64 attention over the same inputs, element by element, by
a bound taken from the inputs: a score is a sum of D products in fp32, off by at most
D 2^-24 sum|q k| scale =: a (a row's largest over its keys), and is rounded a few times
more on its way into the exponent (8 roundings of values up to max|score|); a weight is
then off by a relative 2 (a + ...) (itself and the sum that divides it), exp2 and the
sums over L keys add 2^-21 + 2 L 2^-24. In bf16 a weight keeps 16 significant bits (2^-16),
and the output is rounded by half a bf16 step (2^-8 of it). Each relative error of a weight
moves an output by at most that times max|v|.
"""

import dataclasses
import functools
import random

import pytest
import torch

from kvengine_amd import kernels
from kvengine_amd.layout import to_kernel_layout
from kvengine_amd.paged import DeviceKV

pytestmark = pytest.mark.gpu
DEV = "cuda"


def random_tree(n, r):
    return [-1] + [i - 1 if r.random() < 0.4 else r.randrange(i) for i in range(1, n)]


def way(parents, t):
    """Node t and those above it, by the documented reading of a parent."""
    out = []
    while 0 <= t:
        out.append(t)
        p = parents[t]
        t = p if 0 <= p < t else -1
    return out


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def mask_tensor(rows):
    return torch.tensor([[m - (1 << 64) if m >> 63 else m for m in row] for row in rows], device=DEV)


class Case:
    """Sequences with trees over a paged cache in the reference layout, on the CPU."""

    def __init__(self, seed, starts, T, Hq, Hkv, D, bs=16, dtype=torch.bfloat16, counts=None,
                 trees=None):
        r, g = random.Random(seed), torch.Generator().manual_seed(seed)
        self.starts, self.T, self.bs, self.dtype = starts, T, bs, dtype
        self.counts = counts or [T] * len(starts)
        need = [-(-(s + T) // bs) for s in starts]
        nb = sum(need) + 3
        ids = torch.randperm(nb, generator=g).tolist()
        self.tables = [[ids.pop() for _ in range(n)] for n in need]
        self.pool = torch.randn(2, nb, bs, Hkv, D, generator=g).to(dtype)
        self.q = torch.randn(len(starts), T, Hq, D, generator=g).to(dtype)
        self.parents = trees or [random_tree(T, r) for _ in starts]
        self.masks = [[sum(1 << j for j in way(p, t)) for t in range(T)] for p in self.parents]

    def table(self, width=None):
        w = width or max(len(t) for t in self.tables)
        return i32([t + [-1] * (w - len(t)) for t in self.tables])

    def slot(self, b, pos):
        return self.tables[b][pos // self.bs], pos % self.bs

    def run(self, order=(0, 0), plan=False, fn=kernels.paged_tree_attn, masks=None, out=None, **kw):
        k, v = (t.to(DEV) for t in to_kernel_layout(self.pool[0], self.pool[1]))
        tables, start = self.table(), i32(self.starts)
        q = self.q.to(DEV)
        B, T, Hq, D = q.shape
        ctx = max(self.starts) + T
        q_lens = None if self.counts == [T] * B else i32(self.counts)
        if plan:
            kw["plan"] = kernels.attn_plan(tables, start, B, T, Hq, k.shape[1], D, self.bs,
                                           k.shape[0], ctx, q.dtype, q_lens=q_lens,
                                           unit_blocks=order[0], key_waves=order[1])
        if fn is kernels.paged_tree_attn:
            kw["masks"] = mask_tensor(self.masks) if masks is None else masks
        got = fn(q, k, v, tables, start, ctx, q_lens=q_lens, unit_blocks=order[0],
                 key_waves=order[1], out=out, **kw)
        torch.cuda.synchronize()
        return got.cpu()

    def exact(self, b, t, h, scale=None):
        """(float64 output, its bound) of one row."""
        D, G = self.q.shape[3], self.q.shape[2] // self.pool.shape[3]
        scale = D ** -0.5 if scale is None else scale
        see = list(range(self.starts[b])) + [self.starts[b] + j for j in range(t + 1)
                                             if self.masks[b][t] >> j & 1]
        if not see:
            return torch.zeros(D, dtype=torch.float64), 0.0
        at = torch.tensor([self.slot(b, p) for p in see])
        K = self.pool[0][at[:, 0], at[:, 1], h // G].double()
        V = self.pool[1][at[:, 0], at[:, 1], h // G].double()
        q = self.q[b, t, h].double()
        s = K @ q * scale
        w = torch.softmax(s, 0)
        a = float((K.abs() @ q.abs()).max() * scale) * D * 2.0 ** -24
        a += 8 * 2.0 ** -24 * float(s.abs().max())
        rel = 2 * a + 2.0 ** -21 + 2 * len(see) * 2.0 ** -24
        if self.dtype == torch.bfloat16:
            rel += 2.0 ** -16
        out = (w[:, None] * V).sum(0)
        return out, rel * float(V.abs().max())

    def check(self, got):
        half = torch.finfo(self.dtype).eps / 2
        for b, n in enumerate(self.counts):
            for t in range(n):
                for h in range(self.q.shape[2]):
                    want, tol = self.exact(b, t, h)
                    off = (got[b, t, h].double() - want).abs() - half * want.abs()
                    assert float(off.max()) <= tol, (b, t, h, float(off.max()), tol)


# ---- masks ----------------------------------------------------------------------

@pytest.mark.parametrize("n", [1, 2, 5, 31, 32, 33, 63, 64])
def test_masks_and_depths(gpu_lib, n):
    r = random.Random(n)
    trees = [random_tree(n, r) for _ in range(5)] + [[i - 1 for i in range(n)], [-1] + [0] * (n - 1)]
    # parents that are none: below -1, the node itself, one behind it, far out
    trees.append([r.choice([-7, i, i + 1, 1 << 30, -(1 << 31), max(i - 1, 0)]) for i in range(n)])
    for counts in (None, [r.randrange(n + 1) for _ in trees]):
        masks, depths = kernels.tree_masks(i32(trees), None if counts is None else i32(counts))
        for b, p in enumerate(trees):
            m = n if counts is None else counts[b]
            ways = [way(p, t) if t < m else [] for t in range(n)]
            want = [sum(1 << j for j in w) for w in ways]
            assert [x & (2 ** 64 - 1) for x in masks[b].tolist()] == want
            assert depths[b].tolist() == [max(len(w) - 1, 0) for w in ways]


# ---- attention ------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("Hq,Hkv,D", [(14, 2, 64), (16, 2, 128), (2, 2, 64), (3, 1, 128)])
@pytest.mark.parametrize("T,order", [(1, (0, 0)), (7, (0, 0)), (13, (8, 2)), (33, (4, 1)),
                                     (64, (16, 2)), (64, (0, 0))])
def test_attention_against_float64(gpu_lib, dtype, Hq, Hkv, D, T, order):
    case = Case(T + D, [0, 1, 15, 16, 130, 311], T, Hq, Hkv, D, dtype=dtype)
    case.check(case.run(order))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("bs", [1, 3, 16, 17, 64])
def test_attention_any_block_size(gpu_lib, dtype, bs):
    case = Case(bs, [0, 5, 61, 200], 9, 4, 2, 64, bs=bs, dtype=dtype)
    case.check(case.run())
    case.check(case.run((2, 2)))


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("kw", [1, 2, 4, 8])
def test_attention_long_history_every_key_wave_count(gpu_lib, D, kw):
    """Several units a history, the tree across a unit's edge and across row groups."""
    for T, start in ((1, 1023), (5, 1022), (24, 1015), (64, 1000)):
        case = Case(T, [start, 40], T, 8, 1, D)
        case.check(case.run((8, kw)))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("order", [(0, 0), (8, 2), (4, 1), (16, 4)])
@pytest.mark.parametrize("T", [1, 2, 5, 16, 64])
def test_a_chain_gives_the_causal_kernels_bits(gpu_lib, dtype, order, T):
    counts = [T, max(T - 1, 1), 1, T]
    case = Case(T, [0, 77, 300, 1200], T, 14, 2, 64, dtype=dtype, counts=counts,
                trees=[[i - 1 for i in range(T)]] * 4)
    for plan in (False, True):
        out = [torch.full(case.q.shape, 7.0, dtype=dtype, device=DEV) for _ in range(2)]
        got = case.run(order, plan=plan, out=out[0])
        want = case.run(order, plan=plan, out=out[1], fn=kernels.paged_verify_attn)
        assert torch.equal(got, want)
    for b, n in enumerate(counts):
        assert (got[b, n:] == 7.0).all(), "rows past a sequence's nodes were written"


def test_blocked_output_is_the_same(gpu_lib):
    case = Case(3, [40, 200, 9], 11, 16, 2, 128)
    rows = case.run((8, 2)).view(33, -1)
    blk = case.run((8, 2), blocked=True)
    assert torch.equal(kernels.from_blocked(blk, 33), rows)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("D", [64, 128])
def test_rows_that_see_nothing_are_zeros(gpu_lib, dtype, D):
    """start 0 and an empty mask, in one unit and in a launch that merges units; a
    history with an empty mask is the history alone."""
    for order in ((0, 0), (1, 2), (2, 1)):
        case = Case(5, [0, 900, 0], 40, 4, 2, D, dtype=dtype)
        r = random.Random(1)
        case.masks = [[m if r.random() < 0.5 else 0 for m in row] for row in case.masks]
        got = case.run(order)
        case.check(got)
        for b in (0, 2):
            for t in range(40):
                if not case.masks[b][t]:
                    assert (got[b, t] == 0).all()


def test_bits_above_the_own_node_are_ignored(gpu_lib):
    case = Case(8, [33, 0], 20, 4, 2, 64)
    want = case.run()
    r = random.Random(2)
    noisy = [[m | (r.getrandbits(64) >> (t + 1) << (t + 1)) for t, m in enumerate(row)]
             for row in case.masks]
    assert torch.equal(case.run(masks=mask_tensor(noisy)), want)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("D,order", [(64, (0, 0)), (128, (0, 0)), (64, (2, 2)), (128, (8, 2)),
                                     (128, (4, 1))])
@pytest.mark.parametrize("bs", [16, 5])
def test_what_a_row_does_not_see_never_reaches_it(gpu_lib, dtype, D, order, bs):
    """NaN, infinities and the type's lowest value in unseen nodes, behind the tree and
    in other blocks leave a row's bits alone; a seen one reaches the rows that see it."""
    T = 21
    case = Case(D, [37, 0, 250], T, 6, 2, D, bs=bs, dtype=dtype, counts=[T, T - 4, T])
    clean = case.run(order)
    bad = {0: (9, float("nan")), 1: (4, float("inf")), 2: (17, torch.finfo(dtype).min)}
    for b, (node, x) in bad.items():
        blk, off = case.slot(b, case.starts[b] + node)
        case.pool[1, blk, off] = x
        case.pool[0, blk, off, :, ::2] = float("nan")
    blk, off = case.slot(1, case.starts[1] + T - 2)  # behind the tree's 17 nodes
    case.pool[:, blk, off] = float("nan")
    used = {i for t in case.tables for i in t}
    for i in range(case.pool.shape[1]):
        if i not in used:
            case.pool[:, i] = float("nan")
    got = case.run(order)
    for b, (node, _) in bad.items():
        for t in range(case.counts[b]):
            if case.masks[b][t] >> node & 1:
                assert torch.isnan(got[b, t]).all(), (b, t)
            else:
                assert torch.equal(got[b, t], clean[b, t]), (b, t)
    # infinities alone: a visible one gives the value itself, two signs NaN
    case = Case(D + 1, [37, 60], T, 6, 2, D, bs=bs, dtype=dtype)
    clean = case.run(order)
    nodes = {3: float("inf"), 11: float("-inf")}
    for node, x in nodes.items():
        blk, off = case.slot(0, 37 + node)
        case.pool[1, blk, off, 1, 5] = x
    got = case.run(order)
    for t in range(T):
        for h in range(6):
            seen = [x for node, x in nodes.items() if case.masks[0][t] >> node & 1]
            row, was = got[0, t, h].clone(), clean[0, t, h].clone()
            if h >= 3 and seen:
                assert torch.equal(row[5:6], torch.tensor([sum(seen)]).to(dtype)) \
                    or (len(seen) == 2 and row[5].isnan())
                row[5] = was[5] = 0
            assert torch.equal(row, was), (t, h)
    assert torch.equal(got[1], clean[1])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("kw", [1, 2, 4])
def test_a_seen_infinity_beside_unseen_ones_of_other_key_waves(gpu_lib, dtype, D, kw):
    """A row that sees one infinite node takes it whole, whatever the key waves hold in
    which the row sees no key, or only finite ones, and others are infinite."""
    T, far = 64, (20, 28, 36, 44, 52, 60)
    case = Case(D + kw, [96], T, 4, 2, D, dtype=dtype)
    case.masks[0] = [1 << 3 if t >= 3 else 0 for t in range(T)]
    for t in range(32, T, 2):
        case.masks[0][t] |= sum(1 << n for n in far if n < t)
    clean = case.run((10, kw))
    for node in (3,) + far:
        blk, off = case.slot(0, 96 + node)
        case.pool[1, blk, off, 1, 5] = float("inf")
    got = case.run((10, kw))
    for t in range(3, T):
        assert torch.equal(got[0, t, 2:, 5], torch.full((2,), float("inf"), dtype=dtype)), t
        got[0, t, 2:, 5] = clean[0, t, 2:, 5]
    assert torch.equal(got, clean)


def test_rows_of_a_table_and_a_skipped_sequence(gpu_lib):
    """seq_rows in any order, one row twice, one outside the table (left as it was)."""
    case = Case(4, [20, 90, 300], 6, 4, 2, 64)
    want = case.run((8, 2))
    k, v = (t.to(DEV) for t in to_kernel_layout(case.pool[0], case.pool[1]))
    order = [2, 0, 2, 9, 1]
    idx = [2, 0, 2, 0, 1]
    q, masks = case.q[idx].to(DEV), mask_tensor([case.masks[i] for i in idx])
    out = torch.full_like(q, 3.0)
    kernels.paged_tree_attn(q, k, v, case.table(), i32(case.starts), 306, masks,
                            seq_rows=i32(order), unit_blocks=8, key_waves=2, out=out)
    for i, b in enumerate(order):
        assert torch.equal(out[i].cpu(), want[b] if b < 3 else torch.full_like(want[0], 3.0))


def test_offsets_past_32_bits(gpu_lib):
    """Blocks at the end of a pool whose byte and element offsets pass 2^32."""
    T, Hq, Hkv, D, start = 6, 16, 2, 128, 45
    case = Case(11, [start], T, Hq, Hkv, D)
    want = case.run()
    NB = (1 << 32) // (Hkv * 16 * D) + 40
    k = torch.empty(NB, Hkv, 16, D, dtype=torch.bfloat16, device=DEV)
    v = torch.empty(NB, Hkv, D, 16, dtype=torch.bfloat16, device=DEV)
    kk, vv = to_kernel_layout(case.pool[0], case.pool[1])
    far = [NB - 1 - 7 * i for i in range(len(case.tables[0]))]
    for b, f in zip(case.tables[0], far):
        k[f], v[f] = kk[b].to(DEV), vv[b].to(DEV)
    got = kernels.paged_tree_attn(case.q.to(DEV), k, v, i32([far]), i32([start]), start + T,
                                  mask_tensor(case.masks))
    assert torch.equal(got.cpu(), want)


def test_streams_and_captured_graphs(gpu_lib):
    """The current stream is the one used; two graphs captured on one stream share no
    workspace, and replays follow their inputs with eager work in between."""
    cases = [Case(s, [900 + s, 40, 1000], 12, 16, 2, 128) for s in (1, 2)]
    want = [c.run((2, 2)) for c in cases]
    side, graphs, states = torch.cuda.Stream(), [], []
    for c in cases:
        k, v = (t.to(DEV) for t in to_kernel_layout(c.pool[0], c.pool[1]))
        st = {"q": c.q.to(DEV), "k": k, "v": v, "tab": c.table(), "s": i32(c.starts),
              "p": i32(c.parents)}

        def go(st=st, c=c):
            masks, _ = kernels.tree_masks(st["p"])
            return kernels.paged_tree_attn(st["q"], st["k"], st["v"], st["tab"], st["s"], 1012 + 2,
                                           masks, unit_blocks=2, key_waves=2)
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            eager = go()
        torch.cuda.current_stream().wait_stream(side)
        assert torch.equal(eager.cpu(), go().cpu())
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            st["out"] = go()
        graphs.append(g)
        states.append((st, go))
    eager = [go().clone() for _, go in states]
    other = torch.cuda.Stream()
    for i in range(4):
        for st, _ in states:
            st["out"].zero_()
        torch.cuda.synchronize()
        graphs[0].replay()
        with torch.cuda.stream(other):
            graphs[1].replay()
        torch.cuda.synchronize()
        for j, (st, go) in enumerate(states):
            assert torch.equal(st["out"], eager[j])
            st["q"].copy_(st["q"].flip(0) if i % 2 else st["q"] * 0.5)
            eager[j] = go().clone()
    assert all(torch.equal(w, c.run((2, 2))) for w, c in zip(want, cases))


# ---- accept ---------------------------------------------------------------------

def ref_accept(tokens, parents, preds, n):
    path, new = ([0] if n else []), []
    while path:
        want = preds[path[-1]]
        new.append(want)
        kids = [c for c in range(path[-1] + 1, n) if parents[c] == path[-1] and tokens[c] == want]
        if not kids:
            break
        path.append(kids[0])
    return path, new


def accept_case(seed, B, n, follow, vocab=9):
    """Trees whose picks follow a drafted child with probability `follow`; few tokens, so
    that brothers carry the same one at times."""
    r = random.Random(seed)
    trees = [random_tree(n, r) for _ in range(B)]
    tokens = [[r.randrange(vocab) for _ in range(n)] for _ in range(B)]
    preds = [[r.randrange(vocab) for _ in range(n)] for _ in range(B)]
    for b in range(B):
        for t in range(n):
            kids = [c for c in range(n) if trees[b][c] == t]
            if kids and r.random() < follow:
                preds[b][t] = tokens[b][r.choice(kids)]
    return trees, tokens, preds


@pytest.mark.parametrize("n", [1, 2, 8, 33, 64])
@pytest.mark.parametrize("follow", [0.0, 0.6, 1.0])
def test_accept_walks_the_tree(gpu_lib, n, follow):
    B = 19
    trees, tokens, preds = accept_case(n, B, n, follow)
    r = random.Random(n)
    for counts in (None, [r.randrange(n + 1) for _ in range(B)]):
        n_acc, emitted, path, keep = kernels.tree_accept(
            i32(tokens), i32(trees), i32(preds), q_lens=None if counts is None else i32(counts))
        assert keep is None
        for b in range(B):
            m = n if counts is None else counts[b]
            p, new = ref_accept(tokens[b], trees[b], preds[b], m)
            assert n_acc[b] == max(len(p) - 1, 0)
            assert path[b].tolist() == p + [-1] * (n - len(p))
            assert emitted[b].tolist() == new + [-1] * (n - len(new))


def test_accept_of_a_chain_is_kve_accept(gpu_lib):
    g = torch.Generator().manual_seed(0)
    B, k = 300, 7
    drafts = torch.randint(0, 2, (B, k), generator=g, dtype=torch.int32).to(DEV)
    preds = torch.randint(0, 2, (B, k + 1), generator=g, dtype=torch.int32).to(DEV)
    lens = torch.randint(k + 1, 400, (B,), generator=g, dtype=torch.int32).to(DEV)
    want = kernels.accept(drafts, preds, lens=lens)
    tokens = torch.cat([torch.full((B, 1), 5, dtype=torch.int32, device=DEV), drafts], 1)
    chain = torch.arange(-1, k, dtype=torch.int32, device=DEV).expand(B, k + 1).contiguous()
    nb = B * 25
    kv = DeviceKV(torch.zeros(1, nb, 1, 16, 64, device=DEV), torch.zeros(1, nb, 1, 64, 16, device=DEV),
                  torch.arange(nb, dtype=torch.int32, device=DEV).view(B, 25), lens, 16)
    n_acc, emitted, _, keep = kernels.tree_accept(tokens, chain, preds, kv=kv)
    assert torch.equal(n_acc, want[0]) and torch.equal(emitted, want[1])
    assert torch.equal(keep, want[2])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("bs,D,n", [(16, 64, 20), (16, 128, 64), (1, 64, 12), (7, 128, 33),
                                    (64, 64, 64), (16, 72, 9)])
def test_accept_moves_the_path(gpu_lib, dtype, bs, D, n):
    """Every pool byte as the definition leaves it: the path's rows consecutive, all else
    untouched; ragged counts, rows in any order, one row twice and one outside."""
    B, L, Hkv = 6, 3, 2
    r, g = random.Random(bs), torch.Generator().manual_seed(D)
    trees, tokens, preds = accept_case(bs + n, B, n, 0.85)
    counts = [n, n, max(n - 3, 1), n, n, n]
    rows = [4, 0, 2, 1, 4, 11]
    starts = [r.randrange(40) for _ in range(5)]
    lens = [0] * 5
    for b, row in enumerate(rows):
        if row < 5 and b != 4:
            lens[row] = starts[row] + counts[b]
    width = -(-(40 + n) // bs)
    nb = 5 * width + 2
    ids = torch.randperm(nb, generator=g)[:5 * width].view(5, width)
    k = torch.randn(L, nb, Hkv, bs, D, generator=g).to(dtype)
    v = torch.randn(L, nb, Hkv, D, bs, generator=g).to(dtype)
    want_k, want_v = k.clone(), v.clone()
    for b, row in enumerate(rows):
        if row > 4 or b == 4:
            continue
        p, _ = ref_accept(tokens[b], trees[b], preds[b], counts[b])
        for j, c in enumerate(p):
            (sb, so), (db, do) = ((int(ids[row, x // bs]), x % bs)
                                  for x in (starts[row] + c, starts[row] + j))
            want_k[:, db, :, do] = k[:, sb, :, so]
            want_v[:, db, :, :, do] = v[:, sb, :, :, so]
    kv = DeviceKV(k.to(DEV), v.to(DEV), ids.to(torch.int32).to(DEV), i32(lens), bs)
    n_acc, _, _, keep = kernels.tree_accept(i32(tokens), i32(trees), i32(preds), kv=kv,
                                            seq_rows=i32(rows), q_lens=i32(counts))
    assert torch.equal(kv.k.cpu(), want_k) and torch.equal(kv.v.cpu(), want_v)
    for b, row in enumerate(rows):
        assert keep[b] == (lens[row] - counts[b] + 1 + int(n_acc[b]) if row < 5 else 0)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("bs", [16, 5])
def test_accept_moves_any_number_of_nodes(gpu_lib, dtype, bs):
    """1 to 62 moves: node 1 hangs off the path 0, 2, 3, .., so that all behind it move by
    one slot, into slots that other moves read."""
    n, counts = 64, list(range(1, 63))
    B, D, g = len(counts), 72, torch.Generator().manual_seed(bs)
    trees = [[-1, 0, 0] + list(range(2, n - 1))] * B
    tokens = [[0, 1] + [5] * (n - 2)] * B
    preds = [[5 if t < m + 1 else 7 for t in range(n)] for m in counts]
    starts = [3 + 2 * b for b in range(B)]
    width = -(-(starts[-1] + n) // bs)
    ids = torch.randperm(B * width, generator=g).view(B, width)
    k = torch.randn(2, B * width, 3, bs, D, generator=g).to(dtype)
    v = torch.randn(2, B * width, 3, D, bs, generator=g).to(dtype)
    want_k, want_v = k.clone(), v.clone()
    for b, m in enumerate(counts):
        for j in range(1, m + 1):
            (sb, so), (db, do) = ((int(ids[b, x // bs]), x % bs)
                                  for x in (starts[b] + j + 1, starts[b] + j))
            want_k[:, db, :, do] = k[:, sb, :, so]
            want_v[:, db, :, :, do] = v[:, sb, :, :, so]
    kv = DeviceKV(k.to(DEV), v.to(DEV), ids.to(torch.int32).to(DEV), i32([s + n for s in starts]), bs)
    n_acc, _, _, keep = kernels.tree_accept(i32(tokens), i32(trees), i32(preds), kv=kv)
    assert n_acc.tolist() == counts
    assert keep.tolist() == [s + 1 + m for s, m in zip(starts, counts)]
    assert torch.equal(kv.k.cpu(), want_k) and torch.equal(kv.v.cpu(), want_v)


def test_accept_over_many_heads(gpu_lib):
    """More columns than one turn of the launch's workgroups takes: 2048 heads."""
    L, Hkv, D, bs, n, start = 64, 32, 128, 16, 12, 13
    g = torch.Generator(device=DEV).manual_seed(1)
    k = torch.randn(L, 3, Hkv, bs, D, generator=g, device=DEV, dtype=torch.bfloat16)
    v = torch.randn(L, 3, Hkv, D, bs, generator=g, device=DEV, dtype=torch.bfloat16)
    want_k, want_v = k.clone(), v.clone()
    path, table = [0, 3, 4, 8, 11], [2, 0]
    parents = [-1, 0, 0, 0, 3, 0, 1, 2, 4, 7, 9, 8]
    for j, c in enumerate(path):
        (sb, so), (db, do) = ((table[x // bs], x % bs) for x in (start + c, start + j))
        want_k[:, db, :, do] = k[:, sb, :, so]
        want_v[:, db, :, :, do] = v[:, sb, :, :, so]
    kv = DeviceKV(k, v, i32([table]), i32([start + n]), bs)
    tokens = i32([list(range(n))])
    preds = i32([[3, 0, 0, 4, 8, 0, 0, 0, 11, 0, 0, 2]])
    n_acc, emitted, got, _ = kernels.tree_accept(tokens, i32([parents]), preds, kv=kv)
    assert n_acc.tolist() == [4] and got[0, :5].tolist() == path
    assert emitted[0, :5].tolist() == [3, 4, 8, 11, 2]
    assert torch.equal(k, want_k) and torch.equal(v, want_v)


def test_accept_with_bad_blocks_and_lengths_moves_nothing_outside(gpu_lib):
    """Unallocated or out-of-range table entries and lengths are never followed."""
    n = 16
    tokens, preds = [[0] * n] * 4, [[0] * n] * 4
    trees = [[-1] + [max(i - 2, 0) for i in range(1, n)]] * 4
    k = torch.randn(2, 6, 1, 16, 64)
    v = torch.randn(2, 6, 1, 64, 16)
    tables = i32([[0, -1], [1, 1 << 20], [2, 3], [4, 5]])
    kv = DeviceKV(k.to(DEV), v.to(DEV), tables, i32([26, 30, 3, 1 << 30]), 16)
    kernels.tree_accept(i32(tokens), i32(trees), i32(preds), kv=kv)
    torch.cuda.synchronize()
    assert torch.equal(kv.k[:, 2:].cpu(), k[:, 2:]) and torch.equal(kv.v[:, 2:].cpu(), v[:, 2:])


# ---- the whole of it --------------------------------------------------------------

def tiny_model(name, dtype):
    from kvengine_amd.arch import PRESETS
    from kvengine_amd.model import build_model

    return build_model(PRESETS[name], seed=3, dtype=dtype, device=DEV)


@pytest.mark.parametrize("name,dtype,kw", [
    ("tiny-gqa7-d64", torch.float32, {"fused": False}), ("tiny-gqa7-d64", torch.float32, {}),
    ("tiny-gqa8-d128", torch.float32, {}), ("tiny-gqa8-d128", torch.bfloat16, {"fused": False}),
    ("tiny-gqa7-d64", torch.bfloat16, {}), ("tiny-gqa8-d128", torch.bfloat16, {}),
    ("tiny-gqa8-d128", torch.bfloat16, {"gemm_rows": 160, "attn_order": (8, 2)})])
@pytest.mark.parametrize("n", [1, 3, 13, 40])
def test_a_nodes_hidden_state_is_its_paths(gpu_lib, name, dtype, kw, n):
    """A tree pass gives each node what a plain pass over the history and the node's path
    gives its last token: fp32 within 1e-4 of its norm (two layers of sums in another
    order), bf16 within 2^-5: about twenty roundings of 2^-8 in random order, and a
    wrong mask or position moves a state of these models by its own size."""
    from kvengine_amd.forward import forward_hidden, forward_with_own_cache
    from kvengine_amd.paged import PagedKVCache

    model = tiny_model(name, dtype)
    r = random.Random(n)
    prompts = [[r.randrange(900) for _ in range(m)] for m in (3, 20, 45)]
    trees = [random_tree(n, r) for _ in prompts]
    ids = [[r.randrange(900) for _ in range(n)] for _ in prompts]
    counts = [n, max(n - 2, 1), n]
    pool = PagedKVCache.for_model(model, num_blocks=60, max_seqs=8)
    seqs = [pool.new_sequence(i) for i in range(3)]
    for s, p in zip(seqs, prompts):
        forward_with_own_cache(model, torch.tensor([p], device=DEV), s)
        s.reserve(n)
    tree = kernels.tree_masks(i32(trees), i32(counts))
    hid = forward_hidden(model, i32(ids).long(), pool.device_kv(), i32([s.row for s in seqs]), 45 + n,
                         q_lens=i32(counts), tree=tree, **kw)
    for b, p in enumerate(prompts):
        for t in range(counts[b]):
            text = p + [ids[b][j] for j in reversed(way(trees[b], t))]
            own = PagedKVCache.for_model(model, num_blocks=8).new_sequence("p")
            want = forward_with_own_cache(model, torch.tensor([text], device=DEV), own,
                                          return_hidden=True)[0, 0]
            off = float((hid[b, t].double() - want.double()).norm() / want.double().norm())
            assert off < (1e-4 if dtype == torch.float32 else 2.0 ** -5), (b, t, off)


@pytest.mark.parametrize("name,kw", [("tiny-gqa7-d64", {"fused": False}), ("tiny-gqa8-d128", {})])
def test_tree_decoding_gives_the_greedy_tokens(gpu_lib, name, kw):
    """Greedy decoding of three prompts through trees of eleven drafts that hold the model's
    own continuation on one path here and there: pass, picks, accept with the cache's
    compaction, rollback. The tokens are greedy's whatever the trees hold (fp32)."""
    from kvengine_amd.decode import greedy_paged
    from kvengine_amd.forward import forward_hidden, forward_with_own_cache
    from kvengine_amd.model import lm_head_weight
    from kvengine_amd.paged import PagedKVCache

    model = tiny_model(name, torch.float32)
    V, n, budget = model.arch.vocab, 11, 24
    r = random.Random(4)
    prompts = [[r.randrange(V) for _ in range(m)] for m in (5, 17, 40)]
    want = [greedy_paged(model, torch.tensor([p], device=DEV), PagedKVCache.for_model(model, 16),
                         max_new_tokens=budget + n, eos_token_id=None).new_token_ids
            for p in prompts]
    pool = PagedKVCache.for_model(model, num_blocks=60, max_seqs=8)
    seqs = [pool.new_sequence(i) for i in range(3)]
    for s, p in zip(seqs, prompts):
        forward_with_own_cache(model, torch.tensor([p[:-1]], device=DEV), s)
    got, accepted, passes = [[] for _ in prompts], 0, 0
    while min(len(g) for g in got) < budget:
        passes += 1
        trees, drafts = [], []
        for b, g in enumerate(got):
            parents, ids, depth, good = [-1], [(prompts[b] + g)[-1]], [0], [0]
            for t in range(1, n):
                p = r.choice([good[-1], r.randrange(t)])
                right = (want[b] + [0] * 40)[len(g) + depth[p]]
                if p == good[-1] and r.random() < 0.7:
                    good.append(t)
                    ids.append(right)
                else:
                    ids.append((right + 1 + r.randrange(V - 2)) % V)
                parents.append(p)
                depth.append(depth[p] + 1)
            trees.append(parents)
            drafts.append(ids)
        for s in seqs:
            s.reserve(n)
        kv, rows = pool.device_kv(), i32([s.row for s in seqs])
        parents, ids = i32(trees), i32(drafts)
        hid = forward_hidden(model, ids.long(), kv, rows, max(s.length for s in seqs) + n,
                             tree=kernels.tree_masks(parents), **kw)
        kernels.commit(kv.lens, 3, n, seq_rows=rows)
        preds = kernels.lmhead_argmax(hid.reshape(3 * n, -1), lm_head_weight(model)).view(3, n)
        n_acc, emitted, _, keep = kernels.tree_accept(ids, parents, preds, kv=kv, seq_rows=rows)
        kernels.rollback(kv.tables, kv.lens, keep, pool.block_size, seq_rows=rows)
        for b, s in enumerate(seqs):
            s.sync_committed(n)
            s.truncate(int(keep[b]), device_done=True)
            got[b] += emitted[b, :int(n_acc[b]) + 1].tolist()
            assert s.length == len(prompts[b]) + len(got[b]) - 1
        accepted += int(n_acc.sum())
    assert [g[:budget] for g in got] == [w[:budget] for w in want]
    assert accepted > 2 * passes
    assert kv.lens[rows.long()].tolist() == [s.length for s in seqs]


def test_sampled_tree_decoding_gives_the_sampled_tokens(gpu_lib):
    """The picks of a tree's nodes drawn by sample_verify (k = 0) with one uniform number per
    position of the text: the tokens are those that sampling one at a time gives."""
    from kvengine_amd.forward import forward_hidden, forward_with_own_cache
    from kvengine_amd.paged import PagedKVCache

    model = tiny_model("tiny-gqa7-d64", torch.float32)
    V, n, budget, T = model.arch.vocab, 9, 20, 0.5
    r = random.Random(6)
    prompt = [r.randrange(V) for _ in range(12)]
    u = torch.rand(200, generator=torch.Generator().manual_seed(1))

    def sample(logits, places):
        rows = logits.shape[0]
        none = torch.empty(rows, 0, device=DEV)
        return kernels.sample_verify(logits[:, None], none.int(), none, u[places].to(DEV),
                                     temperature=T)[1][:, 0]

    seq = PagedKVCache.for_model(model, 16).new_sequence("one")
    text = list(prompt)
    logits = forward_with_own_cache(model, torch.tensor([text], device=DEV), seq)[0]
    for _ in range(budget + n):
        text.append(int(sample(logits, torch.tensor([len(text)]))))
        logits = forward_with_own_cache(model, torch.tensor([text[-1:]], device=DEV), seq)[0]
    pool = PagedKVCache.for_model(model, 16)
    seq, got, accepted = pool.new_sequence("tree"), list(prompt), 0
    forward_with_own_cache(model, torch.tensor([got[:-1]], device=DEV), seq)
    while len(got) < len(prompt) + budget:
        parents = random_tree(n, r)
        depths = [len(way(parents, t)) - 1 for t in range(n)]
        ids = [got[-1]] + [text[min(len(got) + d - 1, len(text) - 1)] if r.random() < 0.6
                           else r.randrange(V) for d in depths[1:]]
        seq.reserve(n)
        kv = pool.device_kv()
        tree = kernels.tree_masks(i32([parents]))
        hid = forward_hidden(model, i32([ids]).long(), kv, seq.row_dev, seq.length + n, tree=tree)
        kernels.commit(kv.lens, 1, n, seq_rows=seq.row_dev)
        preds = sample(model.lm_head(hid)[0], torch.tensor([len(got) + d for d in depths]))
        n_acc, emitted, _, keep = kernels.tree_accept(i32([ids]), i32([parents]), preds.view(1, n),
                                                      kv=kv, seq_rows=seq.row_dev)
        kernels.rollback(kv.tables, kv.lens, keep, pool.block_size, seq_rows=seq.row_dev)
        seq.sync_committed(n)
        seq.truncate(int(keep[0]), device_done=True)
        got += emitted[0, :int(n_acc[0]) + 1].tolist()
        accepted += int(n_acc[0])
    assert got[:len(prompt) + budget] == text[:len(prompt) + budget]
    assert accepted > 3


@functools.lru_cache(maxsize=1)
def twelve_layers():
    from kvengine_amd.arch import QWEN25_0_5B
    from kvengine_amd.model import build_model

    arch = dataclasses.replace(QWEN25_0_5B, name="twelve layers", num_layers=12, vocab=1000)
    return build_model(arch, seed=3, dtype=torch.bfloat16, device=DEV)


@pytest.mark.parametrize("B,T", [(1, 1), (1, 2), (2, 2), (1, 4), (1, 5), (3, 6), (2, 16), (5, 13)])
@pytest.mark.parametrize("name", ["tiny-gqa7-d64", "tiny-gqa8-d128", None])
def test_a_chain_shaped_trees_pass_has_the_chains_bits(gpu_lib, name, B, T):
    """bf16: hidden states and the whole pool, at every layer the row count selects and at the
    wide layer that invariant_gemm_rows picks. (None: twelve layers of the 0.5B model's widths.
    Sums in another order change one bf16 value in some 2^14, a few of a pass of four rows.)"""
    from kvengine_amd.forward import forward_hidden, forward_with_own_cache, invariant_gemm_rows
    from kvengine_amd.paged import PagedKVCache

    model = tiny_model(name, torch.bfloat16) if name else twelve_layers()
    ok, rows = invariant_gemm_rows(model, 160)
    assert ok
    chain = kernels.tree_masks(i32([[t - 1 for t in range(T)]] * B))
    for seed in range(3):
        r = random.Random(seed)
        prompts = [[r.randrange(900) for _ in range(m)] for m in (3, 20, 45, 31, 16)[:B]]
        ids = torch.tensor([[r.randrange(900) for _ in range(T)] for _ in prompts], device=DEV)
        for kw in ({}, {"gemm_rows": rows}):
            out = []
            for tree in (None, chain):
                pool = PagedKVCache.for_model(model, num_blocks=60, max_seqs=8)
                seqs = [pool.new_sequence(i) for i in range(B)]
                for s, p in zip(seqs, prompts):
                    forward_with_own_cache(model, torch.tensor([p], device=DEV), s)
                    s.reserve(T)
                kv = pool.device_kv()
                hid = forward_hidden(model, ids, kv, i32([s.row for s in seqs]), 45 + T,
                                     attn_order=(8, 2), tree=tree, **kw)
                out.append((hid, kv.k.clone(), kv.v.clone()))
            for a, b in zip(*out):
                assert torch.equal(a, b), (seed, kw)


@pytest.mark.parametrize("name,dtype,kw", [
    ("tiny-gqa7-d64", torch.bfloat16, {}), ("tiny-gqa8-d128", torch.bfloat16, {"gemm_rows": 160}),
    ("tiny-gqa7-d64", torch.float32, {}), ("tiny-gqa8-d128", torch.float32, {"fused": False})])
@pytest.mark.parametrize("B,n", [(1, 3), (3, 11)])
def test_a_captured_step_of_tree_decoding(gpu_lib, name, dtype, kw, B, n):
    """Masks, pass, commit, picks, accept with compaction and rollback in one graph: replays
    with other tokens and trees, eager steps and a second graph in between, leave what the
    eager step leaves."""
    from kvengine_amd.capture import no_gc
    from kvengine_amd.forward import forward_hidden, forward_with_own_cache
    from kvengine_amd.model import lm_head_weight
    from kvengine_amd.paged import PagedKVCache

    model = tiny_model(name, dtype)
    r = random.Random(n)
    pool = PagedKVCache.for_model(model, num_blocks=60, max_seqs=8)
    seqs = [pool.new_sequence(i) for i in range(B)]
    for s, m in zip(seqs, (5, 30, 47)):
        forward_with_own_cache(model, torch.tensor([[r.randrange(900) for _ in range(m)]], device=DEV), s)
        s.reserve(n)
    kv, rows = pool.device_kv(), i32([s.row for s in seqs])
    weight = lm_head_weight(model)
    ids, parents = torch.zeros(B, n, dtype=torch.int32, device=DEV), i32([[-1] * n] * B)

    def step():
        hid = forward_hidden(model, ids.long(), kv, rows, 60, tree=kernels.tree_masks(parents), **kw)
        kernels.commit(kv.lens, B, n, seq_rows=rows)
        preds = kernels.lmhead_argmax(hid.reshape(B * n, -1), weight).view(B, n)
        got = kernels.tree_accept(ids, parents, preds, kv=kv, seq_rows=rows)
        kernels.rollback(kv.tables, kv.lens, got[3], pool.block_size, seq_rows=rows)
        return (hid, preds) + got

    start = [t.clone() for t in (kv.k, kv.v, kv.tables, kv.lens)]

    def inputs(seed):
        r = random.Random(seed)
        trees = [random_tree(n, r) for _ in range(B)]
        parents.copy_(i32(trees))
        ids.copy_(i32([[r.randrange(900) for _ in range(n)] for _ in range(B)]))
        back()
        # the picks of a few nodes put into their children, so that paths are accepted
        for _ in range(3):
            preds = step()[1].tolist()
            back()
            ids.copy_(i32([[t if not j or r.random() < 0.3 else preds[b][trees[b][j]]
                            for j, t in enumerate(row)] for b, row in enumerate(ids.tolist())]))

    def back():
        for t, was in zip((kv.k, kv.v, kv.tables, kv.lens), start):
            t.copy_(was)

    def state(got):
        return [t.clone() for t in got] + [t.clone() for t in (kv.k, kv.v, kv.tables, kv.lens)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        inputs(1)
        step()
        back()
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with no_gc(), torch.cuda.graph(g, stream=side):
            out = step()
        graphs.append((g, out))
    moved = 0
    for i in range(4):
        inputs(i)
        want = state(step())
        moved += int(want[2].sum())
        for g, out in graphs:
            back()
            g.replay()
            for a, b in zip(state(out), want):
                assert torch.equal(a, b), i
    assert moved > 0


@pytest.mark.parametrize("dtype,D,T,order", [
    (torch.bfloat16, 64, 8, (0, 0)), (torch.bfloat16, 128, 16, (0, 0)),
    (torch.bfloat16, 128, 13, (8, 2)), (torch.bfloat16, 128, 64, (16, 2)),
    (torch.float32, 64, 11, (0, 0)), (torch.float32, 128, 40, (4, 2))])
def test_the_same_call_gives_the_same_bits(gpu_lib, dtype, D, T, order):
    case = Case(T, [603, 0, 1500, 77], T, 14 if D == 64 else 16, 2, D, dtype=dtype)
    want = case.run(order)
    case.check(want)
    for _ in range(3):
        assert torch.equal(case.run(order), want)


@pytest.mark.parametrize("T,order", [(16, (2, 2)), (64, (2, 2)), (64, (4, 1))])
def test_offsets_past_32_bits_with_several_row_tiles(gpu_lib, T, order):
    """Blocks at the end of a pool of more than 2^32 elements for the kernel of several row
    tiles, with an infinity in a node, which it reads from the pool a second time."""
    Hq, Hkv, D, start = 16, 2, 128, 75
    case = Case(12, [start], T, Hq, Hkv, D)
    blk, off = case.slot(0, start + 2)
    case.pool[1, blk, off, 1, 7] = float("inf")
    want = case.run(order)
    assert want.isinf().any() and not want.isnan().any()
    NB = (1 << 32) // (Hkv * 16 * D) + 40
    k = torch.empty(NB, Hkv, 16, D, dtype=torch.bfloat16, device=DEV)
    v = torch.empty(NB, Hkv, D, 16, dtype=torch.bfloat16, device=DEV)
    kk, vv = to_kernel_layout(case.pool[0], case.pool[1])
    far = [NB - 1 - 3 * i for i in range(len(case.tables[0]))]
    for b, f in zip(case.tables[0], far):
        k[f], v[f] = kk[b].to(DEV), vv[b].to(DEV)
    got = kernels.paged_tree_attn(case.q.to(DEV), k, v, i32([far]), i32([start]), start + T,
                                  mask_tensor(case.masks), unit_blocks=order[0], key_waves=order[1])
    assert torch.equal(got.cpu(), want)


@pytest.mark.parametrize("layers", [1, 3])
def test_accept_moves_past_32_bits(gpu_lib, layers):
    """Blocks at the end of a pool of more than 2^32 elements, in one layer and over three."""
    Hkv, D, bs, n, start = 2, 128, 16, 40, 9
    NB = (1 << 32) // (layers * Hkv * bs * D) + 60
    k = torch.empty(layers, NB, Hkv, bs, D, dtype=torch.bfloat16, device=DEV)
    v = torch.empty(layers, NB, Hkv, D, bs, dtype=torch.bfloat16, device=DEV)
    table = [NB - 1, NB - 30, 2, NB - 2]
    g = torch.Generator(device=DEV).manual_seed(layers)
    for b in table:
        k[:, b] = torch.randn(layers, Hkv, bs, D, generator=g, device=DEV).bfloat16()
        v[:, b] = torch.randn(layers, Hkv, D, bs, generator=g, device=DEV).bfloat16()
    near_k, near_v = k[:, table].cpu(), v[:, table].cpu()
    path = [0, 5, 11, 12, 30, 39]
    parents = [-1] + [0] * (n - 1)
    for a, b in zip(path, path[1:]):
        parents[b] = a
    preds = [99] * n
    for a, b in zip(path, path[1:]):
        preds[a] = b
    want_k, want_v = near_k.clone(), near_v.clone()
    for j, c in enumerate(path):
        (sb, so), (db, do) = (divmod(start + x, bs) for x in (c, j))
        want_k[:, db, :, do] = near_k[:, sb, :, so]
        want_v[:, db, :, :, do] = near_v[:, sb, :, :, so]
    kv = DeviceKV(k, v, i32([table]), i32([start + n]), bs)
    n_acc, _, _, keep = kernels.tree_accept(i32([list(range(n))]), i32([parents]), i32([preds]), kv=kv)
    assert n_acc.tolist() == [5] and keep.tolist() == [start + 6]
    assert torch.equal(k[:, table].cpu(), want_k) and torch.equal(v[:, table].cpu(), want_v)
