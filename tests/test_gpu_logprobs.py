"""Log probabilities of given tokens, entropy and alternatives against float64.

Bounds: with y = (x - m) log2(e), a weight 2^y is off by a relative e = 2^-24 (3|y| + 2) (two
roundings of y and the constant's, the instruction's), sums of 32 weights by lane and the
wave's add 40 2^-24; the rest is in 64 bits. So log S is off by r = sum(p (e + 40 2^-24)),
log probabilities by r and half a step of themselves, the entropy log S - T / S by r, the
errors of T, sum(p |y| (e + 42 2^-24)) ln 2, r |T / S| ln 2 and half a step.
"""

import math

import pytest
import torch

from kvengine_amd import kernels

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = 2.0 ** -24


def exact(x, t):
    """(log probability of t, entropy, their bounds) of a row in float64."""
    x = x.double()
    w = torch.log_softmax(x, 0)
    p = w.exp()
    seen = p > 0
    y = ((x - x.max()) / math.log(2.0))[seen].abs()
    p, w = p[seen], w[seen]
    e = U * (3 * y + 42)
    r = float((p * e).sum())
    H = float(-(p * w).sum())
    T = float((p * y).sum())
    dH = r + math.log(2.0) * (float((p * y * (e + 2 * U)).sum()) + r * T) + U * abs(H)
    lp = float(torch.log_softmax(x, 0)[t]) if 0 <= t < x.numel() else math.nan
    return lp, H, r, dH


def to_range(w):
    """Float64 values past float32's range as it rounds them: from (2 - 2^-24) 2^127 on, half a
    step behind its largest number, they are infinite (a lowest logit beside a largest one
    has the log probability -6.8e38)."""
    return torch.where(w.abs() >= (2 - 2.0 ** -24) * 2.0 ** 127, w.sign() * math.inf, w)


def check(logits, tokens, top):
    got = kernels.token_logprobs(logits.to(DEV), tokens.to(DEV), top=top)
    torch.cuda.synchronize()
    lp, H, ids, tops = (g.cpu() for g in got)
    assert ids.shape == tops.shape == (logits.shape[0], top)
    for i, row in enumerate(logits):
        t = int(tokens[i])
        want, wH, r, dH = exact(row, t)
        want = float(to_range(torch.tensor(want, dtype=torch.float64)))
        if math.isnan(want):
            assert math.isnan(lp[i])
        elif math.isinf(want):
            assert float(lp[i]) == want
        else:
            assert abs(float(lp[i]) - want) <= r + U * abs(want) + 1e-45, (i, float(lp[i]), want)
        assert abs(float(H[i]) - wH) <= dH + 1e-45, (i, float(H[i]), wH, dH)
        order = torch.sort(row.double(), descending=True, stable=True).indices[:top]
        assert ids[i].tolist() == order.tolist(), i
        w = to_range(torch.log_softmax(row.double(), 0)[order])
        fin = torch.isfinite(w)
        assert torch.equal(torch.isfinite(tops[i]), fin)
        assert bool(((tops[i].double() - w).abs() <= r + U * w.abs())[fin].all())
    return lp, H, ids, tops


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("R,V,top", [(1, 1, 1), (1, 1, 0), (3, 2, 2), (2, 31, 31), (5, 63, 20), (4, 65, 32),
                                     (3, 129, 5), (2, 2047, 32), (2, 2049, 10), (3, 5000, 20),
                                     (7, 50257, 20), (2, 151936, 5), (40, 1000, 1), (1, 700001, 32)])
def test_logprobs(R, V, top, dtype):
    g = torch.Generator().manual_seed(V + R)
    x = (3 * torch.randn(R, V, generator=g)).to(dtype)
    t = torch.randint(0, V, (R,), generator=g).to(torch.int32)
    t[0] = int(x[0].float().argmax())
    check(x, t, top)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("V", [40, 3000, 151936])
def test_ties_go_to_the_lowest_id(dtype, V):
    x = torch.zeros(5, V, dtype=dtype)
    x[1, V // 2:] = 1.0
    x[2, ::7] = -0.0  # equal to 0
    x[3, [V - 1, 3, V // 3]] = 2.0
    x[4] = torch.arange(V).remainder(3).to(dtype)
    check(x, torch.zeros(5, dtype=torch.int32), 20)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("V", [37, 4100])
def test_masked_ids(dtype, V):
    """Masks of -inf and of the type's lowest value, all but one id masked, all of them at the
    lowest value, large logits."""
    lo = torch.finfo(dtype).min
    g = torch.Generator().manual_seed(V)
    x = torch.randn(7, V, generator=g).to(dtype)
    x[0, ::2] = -math.inf
    x[1, ::2] = lo
    x[2, :] = -math.inf
    x[2, V - 2] = -3.0
    x[3, :] = lo
    x[4] *= 1e30
    x[5, :] = torch.finfo(dtype).max
    x[6, :] = lo
    x[6, 5] = torch.finfo(dtype).max
    check(x, torch.tensor([1, 0, V - 2, 3, 4, 5, 6], dtype=torch.int32), 10)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_rows_without_a_distribution_and_ids_outside(dtype):
    g = torch.Generator().manual_seed(1)
    x = torch.randn(6, 3000, generator=g).to(dtype)
    x[0, 2500] = math.nan
    x[1, 7] = math.inf
    x[2, :] = -math.inf
    got = kernels.token_logprobs(x.to(DEV), torch.tensor([0, 7, 3, -1, 3000, 2 ** 31 - 1],
                                                         dtype=torch.int32, device=DEV), top=4)
    lp, H, ids, tops = (t.cpu() for t in got)
    assert bool(torch.isnan(lp).all())
    assert bool(torch.isnan(H[:3]).all()) and bool(torch.isfinite(H[3:]).all())
    assert int(ids[0, 0]) == 2500 and int(ids[1, 0]) == 7 and ids[2].tolist() == [0, 1, 2, 3]
    assert bool(torch.isnan(tops[:3]).all()) and bool(torch.isfinite(tops[3:]).all())
    check(x[3:], torch.tensor([5, 6, 7], dtype=torch.int32), 4)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("V", [151936, 700001])
def test_likely_ids_that_lie_together(dtype, V):
    """The likeliest ids spread evenly, in one place, ascending and descending, and in places
    that a selection by parts would find in one part: every 4th, 64th, 1024th, 32768th id."""
    g = torch.Generator().manual_seed(V)
    x = torch.randn(9, V, generator=g)
    i = torch.arange(V)
    x[0, V // 2:V // 2 + 100] += 10
    x[1] = i / V * 30
    x[2] = -i / V * 30
    for r, step in enumerate((4, 64, 1024, 32768), start=3):
        x[r, step - 1::step] += 8
    x[7] += 5.0 * (i // 128 % 1024 < 500)
    x[8] += 5.0 * (i // 64 % 256 < 128)
    check(x.to(dtype), torch.arange(9, dtype=torch.int32), 32)


def test_strided_and_unaligned_rows():
    g = torch.Generator().manual_seed(2)
    for dtype in (torch.bfloat16, torch.float32):
        big = (3 * torch.randn(5, 3, 2501, generator=g)).to(dtype)
        t = torch.randint(0, 2500, (5,), generator=g).to(torch.int32)
        dev = big.to(DEV)
        view = dev[:, 1, 1:]
        got = kernels.token_logprobs(view, t.to(DEV), top=3)
        want = kernels.token_logprobs(view.contiguous(), t.to(DEV), top=3)
        for a, b in zip(got, want):
            assert torch.equal(a, b)
        check(big[:, 1, 1:].contiguous(), t, 3)
        one = dev[0, 0].expand(4, 2501)  # the same row four times
        got = kernels.token_logprobs(one, t[:4].to(DEV), top=3)
        assert bool((got[2] == got[2][0]).all())


def test_captured_and_on_another_stream():
    g = torch.Generator().manual_seed(3)
    xs = [(3 * torch.randn(4, 30000, generator=g)).to(torch.bfloat16).to(DEV) for _ in range(2)]
    t = torch.tensor([1, 2, 3, 4], dtype=torch.int32, device=DEV)
    want = [kernels.token_logprobs(x, t, top=20) for x in xs]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = kernels.token_logprobs(xs[0], t, top=20)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want[0]))
    graphs = []
    for x in xs:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = kernels.token_logprobs(x, t, top=20)
        graphs.append((graph, out))
    for _ in range(4):
        for graph, out in graphs:
            for o in out:
                o.zero_()
            graph.replay()
        eager = kernels.token_logprobs(xs[1], t, top=20)
        torch.cuda.synchronize()
        for (_, out), w in zip(graphs, want):
            assert all(torch.equal(a, b) for a, b in zip(out, w))
        assert all(torch.equal(a, b) for a, b in zip(eager, want[1]))
