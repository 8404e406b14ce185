"""Verification of drafted tokens by rejection sampling against its definition in 64
bits. Every output is a whole number and has to be equal: the sums on both sides are off
by about 1e-13 of their size, so a draw could only turn where a uniform number lies that
near to one of V places, which happens once in some 10^7 draws of the largest vocabulary.
"""

import random

import pytest
import torch

from kvengine_amd import kernels

pytestmark = pytest.mark.gpu
DEV = "cuda"
INF = float("inf")


def reference(target, drafts, ua, us, draft=None, temps=1.0):
    """The definition, one sequence and position at a time, in float64 on the CPU."""
    B, k1, V = target.shape
    n_acc, emitted = [], []

    def softmax(row, T):
        e = torch.exp((row.double() - row.double().max()) / T)
        return e, e / e.sum()

    for b in range(B):
        T = float(temps[b]) if isinstance(temps, torch.Tensor) else temps
        new, token = [], -1
        for j in range(k1):
            if not 0.0 < T < INF:
                break
            e, p = softmax(target[b, j], T)
            if j == k1 - 1:
                w = e
            else:
                x = int(drafts[b, j])
                inside = 0 <= x < V
                q = softmax(draft[b, j], T)[1] if draft is not None else None
                qx = (float(q[x]) if q is not None else 1.0) if inside else 0.0
                if inside and float(ua[b, j]) * qx < float(p[x]):
                    new.append(x)
                    continue
                if q is not None:
                    w = torch.where(p - q < 0, 0.0, p - q)
                else:
                    w = e.clone()
                    if inside:
                        w[x] = 0.0
                if float(w.sum()) == 0.0:
                    w = e
            c = w.cumsum(0)
            if float(c[-1]) > 0.0:
                token = int((c <= float(us[b]) * c[-1]).sum())
                token = min(token, int(w.nonzero().max()))
            break
        n_acc.append(len(new))
        emitted.append(new + [token] + [-1] * (k1 - 1 - len(new)))
    return torch.tensor(n_acc, dtype=torch.int32), torch.tensor(emitted, dtype=torch.int32)


def draw_inputs(seed, B, k, V, dtype, near=0.7, spread=3.0, T=1.0):
    g = torch.Generator().manual_seed(seed)
    target = (spread * torch.randn(B, k + 1, V, generator=g)).to(dtype)
    draft = (target[:, :k] + near * torch.randn(B, k, V, generator=g)).to(dtype)
    u = torch.rand(B, k, V, generator=g).clamp_min(1e-30)
    drafts = (draft.float() / T - torch.log(-torch.log(u).clamp_min(1e-30))).argmax(-1) if k else \
        torch.zeros(B, 0)
    return (target, drafts.to(torch.int32), torch.rand(B, k, generator=g),
            torch.rand(B, generator=g), draft)


def run(target, drafts, ua, us, draft=None, temps=1.0, **kw):
    if isinstance(temps, torch.Tensor):
        temps = temps.to(DEV)
    out = kernels.sample_verify(target.to(DEV), drafts.to(DEV), ua.to(DEV), us.to(DEV),
                                draft_logits=None if draft is None else draft.to(DEV),
                                temperature=temps, **kw)
    return [None if t is None else t.cpu() for t in out]


def check(args, temps=1.0):
    n_acc, emitted, keep = run(*args, temps=temps)
    want = reference(*args, temps=temps)
    assert keep is None
    assert torch.equal(n_acc, want[0]) and torch.equal(emitted, want[1])
    return n_acc, emitted


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("B,k,V", [(1, 0, 1), (3, 2, 1), (5, 4, 2), (40, 3, 17), (7, 1, 1000),
                                   (9, 8, 2047), (6, 5, 2049), (4, 4, 8193), (3, 16, 16400),
                                   (2, 4, 50257), (1, 4, 151936), (64, 1, 5000)])
def test_against_the_definition(gpu_lib, dtype, B, k, V):
    T = 0.8
    target, drafts, ua, us, draft = draw_inputs(V + k, B, k, V, dtype, T=T)
    check((target, drafts, ua, us, draft), T)
    check((target, drafts, ua, us, None), T)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_many_rows_and_every_chunk_size(gpu_lib, dtype):
    """Row counts on both sides of the chunk rule's bounds, at one vocabulary."""
    for B in (1, 9, 20, 60, 130):
        args = draw_inputs(B, B, 1, 20011, dtype)
        check(args)


def test_a_temperature_per_sequence(gpu_lib):
    args = draw_inputs(1, 8, 3, 700, torch.float32)
    temps = torch.tensor([0.2, 1.0, 5.0, 1e-6, 1e4, 1.5, 1e-30, 1e30])
    check(args, temps)
    for T in (1e-38, 1e-3, 0.05, 30.0, 3e38):
        check(args, T)


def test_a_bad_temperature_has_no_answer(gpu_lib):
    args = draw_inputs(2, 5, 2, 300, torch.bfloat16)
    temps = torch.tensor([0.0, -1.0, INF, float("nan"), 1.0])
    n_acc, emitted, _ = run(*args, temps=temps)
    assert n_acc[:4].tolist() == [0] * 4 and (emitted[:4] == -1).all()
    want = reference(*args, temps=temps)
    assert torch.equal(emitted, want[1])
    for bad in (0.0, -2.0, INF, float("nan")):
        with pytest.raises(ValueError, match="temperature"):
            run(*args, temps=bad)


def test_greedy_at_a_vanishing_temperature(gpu_lib):
    """As T falls the draws become the greedy accept's."""
    target, drafts, ua, us, _ = draw_inputs(3, 50, 4, 400, torch.float32)
    preds = target.argmax(-1).to(torch.int32)
    drafts = torch.where(torch.rand(50, 4, generator=torch.Generator().manual_seed(1)) < 0.7,
                         preds[:, :4], drafts)
    n_acc, emitted, _ = run(target, drafts, ua.clamp_min(0.01), us, temps=1e-4)
    want = kernels.accept(drafts.to(DEV), preds.to(DEV))
    assert torch.equal(n_acc, want[0].cpu()) and torch.equal(emitted, want[1].cpu())


@pytest.mark.parametrize("offset,pad", [(0, 0), (1, 3), (3, 8), (5, 1)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_strides_and_alignment(gpu_lib, dtype, offset, pad):
    """Logits inside wider rows, at any element, positions before sequences."""
    B, k, V = 4, 3, 1234
    target, drafts, ua, us, draft = draw_inputs(5, B, k, V, dtype)
    want = reference(target, drafts, ua, us, draft)

    def laid(x, swap):
        n = x.shape[1]
        big = torch.full((n, B, offset + V + pad) if swap else (B, n, offset + V + pad),
                         float("nan"), dtype=dtype, device=DEV)
        view = big.transpose(0, 1) if swap else big
        view[..., offset:offset + V] = x.to(DEV)
        return view[..., offset:offset + V]
    for swap in (False, True):
        n_acc, emitted, _ = kernels.sample_verify(laid(target, swap), drafts.to(DEV), ua.to(DEV),
                                                  us.to(DEV), draft_logits=laid(draft, not swap))
        assert torch.equal(n_acc.cpu(), want[0]) and torch.equal(emitted.cpu(), want[1])
    one = laid(target[:1], False).expand(B, k + 1, V)  # one sequence's logits for all
    same = reference(target[:1].expand(B, -1, -1), drafts, ua, us, draft)
    got = kernels.sample_verify(one, drafts.to(DEV), ua.to(DEV), us.to(DEV),
                                draft_logits=draft.to(DEV)) if offset + pad == 0 else None
    if got is not None:
        assert torch.equal(got[1].cpu(), same[1])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("low", [-INF, None])
def test_filtered_vocabularies(gpu_lib, dtype, low):
    """Logits put out with -inf or the type's lowest value are never drawn: whole chunks of
    them, all but one, and drafts among them."""
    low = torch.finfo(dtype).min if low is None else low
    B, k, V = 24, 3, 30000
    target, drafts, ua, us, draft = draw_inputs(8, B, k, V, dtype)
    g = torch.Generator().manual_seed(2)
    for b in range(B):
        keep = torch.randperm(V, generator=g)[:(1, 2, 50, 4000)[b % 4]]
        for x in (target, draft) if b % 3 else (target,):
            row = x[b, :, keep].clone()
            x[b] = low
            x[b, :, keep] = row
    us[::5] = 0.0
    n_acc, emitted = check((target, drafts, ua, us, draft))
    check((target, drafts, ua, us, None))
    for b in range(B):
        last = emitted[b, n_acc[b]]
        assert target[b, n_acc[b], last] > low


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_rows_without_a_distribution(gpu_lib, dtype):
    """NaN, +inf and nothing but -inf: the draft falls and no token is drawn; what comes
    before it stands."""
    V, k = 9000, 3
    for where in range(k + 1):
        for bad in (float("nan"), INF, -INF):
            target, drafts, ua, us, draft = draw_inputs(where, 4, k, V, dtype)
            ua[:] = 0.0  # every draft of a sound row is accepted
            if bad == -INF:
                target[:2, where] = -INF
            else:
                target[:2, where, 8500] = bad
            if where < k:
                draft[2, where, 4] = float("nan")
            n_acc, emitted, _ = run(target, drafts, ua, us, draft)
            for b in range(2 if where == k else 3):
                assert n_acc[b] == where
                assert emitted[b].tolist() == drafts[b, :where].tolist() + [-1] * (k + 1 - where)
            assert n_acc[3] == k and emitted[3, k] >= 0
            n_acc, emitted, _ = run(target, drafts, ua, us, None)
            assert n_acc[:2].tolist() == [where] * 2 and (emitted[:2, where:] == -1).all()
            assert n_acc[2] == k


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("V", [1000, 1024, 8192, 12000])
def test_ties_and_ends(gpu_lib, dtype, V):
    """Equal logits make equal steps of the running sum: places that fall on a step go to the
    id behind it, 0 to the first id, the largest number below 1 to the last."""
    top = 1.0 - 2.0 ** -24
    us = torch.tensor([0.0, 0.25, 0.5, 0.75, top, 2.0 ** -24, 0.125, 0.3])
    B = len(us)
    none = torch.zeros(B, 0)
    for x in (0.0, -7.5, 100.0):
        target = torch.full((B, 1, V), x, dtype=dtype)
        n_acc, emitted, _ = run(target, none.int(), none, us)
        assert emitted[:, 0].tolist() == [min(int(float(u) * V), V - 1) for u in us]
    # an id of half the mass
    target = torch.full((B, 1, V), -INF, dtype=dtype)
    target[:, 0, V // 2:V // 2 + 2] = 1.0
    _, emitted, _ = run(target, none.int(), none, us)
    assert emitted[:, 0].tolist() == [V // 2 + (float(u) >= 0.5) for u in us]


def test_equal_distributions_accept_everything(gpu_lib):
    """p = q: the ratio is 1 and every uniform number lies below it."""
    target, drafts, ua, us, _ = draw_inputs(4, 30, 5, 3001, torch.bfloat16)
    ua[:] = 1.0 - 2.0 ** -24
    n_acc, emitted = check((target, drafts, ua, us, target[:, :5].clone()))
    assert (n_acc == 5).all()
    # a draft outside the vocabulary falls, and p - q leaves nothing: p itself is drawn from
    drafts[:10, 0], drafts[10:20, 2] = -1, 3001
    drafts[20:, 4] = 1 << 30
    n_acc, _ = check((target, drafts, ua, us, target[:, :5].clone()))
    assert n_acc.tolist() == [0] * 10 + [2] * 10 + [4] * 10
    check((target, drafts, ua, us, None))


def test_a_certain_token(gpu_lib):
    """All of p on one id: the draft of it is accepted at any number, any other falls to it."""
    target = torch.full((4, 2, 5000), -INF)
    target[:, :, 77] = 3.0
    ua = torch.full((4, 1), 1.0 - 2.0 ** -24)
    drafts = torch.tensor([[77], [78], [77], [0]], dtype=torch.int32)
    n_acc, emitted = check((target, drafts, ua, torch.rand(4), None))
    assert n_acc.tolist() == [1, 0, 1, 0] and (emitted[:, 0] == 77).all()


def test_keep_lens_and_rows(gpu_lib):
    args = draw_inputs(6, 5, 4, 500, torch.bfloat16)
    lens = torch.tensor([50, 60, 70, 80, 90, 100], dtype=torch.int32, device=DEV)
    n_acc, _, keep = run(*args, lens=lens)
    assert torch.equal(keep, lens[:5].cpu() - 4 + n_acc)
    rows = torch.tensor([5, 0, 7, -1, 2], dtype=torch.int32, device=DEV)
    _, _, keep = run(*args, lens=lens, seq_rows=rows)
    assert keep.tolist() == [100 - 4 + int(n_acc[0]), 50 - 4 + int(n_acc[1]), 0, 0,
                             70 - 4 + int(n_acc[4])]


def test_refusals(gpu_lib):
    target, drafts, ua, us, draft = (t.to(DEV) for t in draw_inputs(7, 3, 2, 64, torch.float32))
    ok = dict(draft_logits=draft)
    for change in (dict(drafts=drafts.long()), dict(drafts=drafts[:, :1]), dict(ua=ua.double()),
                   dict(us=us[:2]), dict(us=us.cpu()), dict(draft_logits=draft.bfloat16()),
                   dict(draft_logits=draft[:, :1]), dict(temperature=torch.ones(2, device=DEV)),
                   dict(target=target.transpose(1, 2)), dict(target=target[0]),
                   dict(lens=torch.zeros(2, dtype=torch.int32, device=DEV)),
                   dict(seq_rows=torch.zeros(2, dtype=torch.int32, device=DEV))):
        a = dict(target=target, drafts=drafts, ua=ua, us=us, **ok) | change
        pos = [a.pop(n) for n in ("target", "drafts", "ua", "us")]
        with pytest.raises(ValueError):
            kernels.sample_verify(*pos, **a)
    with pytest.raises(TypeError):
        kernels.sample_verify(target.half(), drafts, ua, us)


def test_calls_in_a_row_streams_and_graphs(gpu_lib):
    """Calls of other sizes between, on other streams at once, and replays of two graphs with
    new inputs: each equals the eager call."""
    sizes = [(2, 4, 3000), (30, 1, 151936), (1, 0, 17), (16, 8, 40000)]
    cases = [[t.to(DEV) for t in draw_inputs(i, B, k, V, torch.bfloat16)]
             for i, (B, k, V) in enumerate(sizes)]

    def call(c):
        return kernels.sample_verify(*c[:4], draft_logits=c[4], temperature=0.9)
    want = [call(c) for c in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    for _ in range(3):
        got = []
        for c, s in zip(cases, streams):
            with torch.cuda.stream(s):
                got.append(call(c))
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    graphs = []
    for c in (cases[0], cases[3]):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = call(c)
        graphs.append((g, c, out))
    for i in range(4):
        for s, (g, c, out) in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for g, c, out in graphs:
            eager = call(c)
            assert torch.equal(out[0], eager[0]) and torch.equal(out[1], eager[1])
            c[2].copy_(torch.rand_like(c[2]))
            c[3].copy_(torch.rand_like(c[3]))
            c[0].copy_(c[0].flip(-1))
        torch.cuda.synchronize()


def test_emitted_tokens_follow_the_target(gpu_lib):
    """Over many sequences with drafts drawn from q, the first emitted token is distributed as
    p whatever q is: with N = 2^17 draws each frequency lies within five standard deviations,
    sqrt(p (1 - p) / N), of its probability (the eight ids' joint odds are 5e-6)."""
    N, V = 1 << 17, 8
    g = torch.Generator().manual_seed(9)
    target = torch.randn(1, 2, V, generator=g) * 1.5
    draft = torch.randn(1, 1, V, generator=g) * 1.5
    q = torch.softmax(draft[0, 0].double(), 0)
    drafts = torch.multinomial(q, N, replacement=True, generator=g).to(torch.int32).view(N, 1)
    ua, us = torch.rand(N, 1, generator=g), torch.rand(N, generator=g)
    p = torch.softmax(target[0, 0].double(), 0)
    for d, x in ((draft, drafts), (None, torch.full((N, 1), 3, dtype=torch.int32))):
        got = kernels.sample_verify(target.to(DEV).expand(N, 2, V), x.to(DEV), ua.to(DEV), us.to(DEV),
                                    draft_logits=None if d is None else d.to(DEV).expand(N, 1, V))
        f = torch.bincount(got[1][:, 0].cpu().long(), minlength=V).double() / N
        assert ((f - p).abs() <= 5 * (p * (1 - p) / N).sqrt()).all(), (f, p)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("with_draft", [True, False])
def test_uniform_numbers_beside_a_test_s_edge(gpu_lib, dtype, with_draft):
    """u the fp32 numbers around p(x) / q(x): 32-bit sums do not decide these tests, and
    several of a sequence follow each other. An fp32 number lies some 1e-8 from the edge."""
    B, k, V = 24, 5, 4099
    target, drafts, ua, us, draft = draw_inputs(77, B, k, V, dtype, near=0.5)
    p = torch.softmax(target[:, :k].double(), -1).gather(2, drafts.long()[..., None])[..., 0]
    q = torch.softmax(draft.double(), -1).gather(2, drafts.long()[..., None])[..., 0]
    edge = (p / q if with_draft else p).float()
    for b in range(B):
        for j in range(k):
            if edge[b, j] >= 1 or (b + j) % 5 == 4:
                continue
            u = edge[b, j]
            for _ in range((b + 3 * j) % 4):
                u = torch.nextafter(u, torch.tensor(0.0 if (b + j) % 2 else 2.0))
            ua[b, j] = u
    n_acc, _ = check((target, drafts, ua, us, draft if with_draft else None))
    assert len(set(n_acc.tolist())) > 2


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_probabilities_that_differ_by_less_than_the_sums(gpu_lib, dtype):
    """Every id's p - q is a few millionths of p, all of one sign but the draft's."""
    B, V = 6, 30011
    g = torch.Generator().manual_seed(5)
    target = (0.25 * torch.randn(B, 2, V, generator=g)).to(dtype)
    draft = target[:, :1].clone()
    x = torch.randint(0, V, (B,), generator=g, dtype=torch.int32)
    for b in range(B):
        draft[b, 0, x[b]] += 0.125
    us = torch.rand(B, generator=g)
    n_acc, emitted = check((target, x[:, None], torch.full((B, 1), 1 - 2.0 ** -24), us, draft))
    assert n_acc.tolist() == [0] * B
    n_acc, emitted = check((target, x[:, None], torch.full((B, 1), 0.5), us, draft))
    assert n_acc.tolist() == [1] * B


def test_probabilities_that_differ_by_as_little_both_ways(gpu_lib):
    """Every id's p / q lies within some millionths of the ratio that decides its side."""
    B, V = 4, 5003
    g = torch.Generator().manual_seed(9)
    target = 0.25 * torch.randn(B, 2, V, generator=g)
    draft = target[:, :1] + 2e-6 * torch.randn(B, 1, V, generator=g)
    x = torch.randint(0, V, (B,), generator=g, dtype=torch.int32)
    for b in range(B):
        draft[b, 0, x[b]] += 0.125
    n_acc, _ = check((target, x[:, None], torch.full((B, 1), 0.99), torch.rand(B, generator=g), draft))
    assert n_acc.tolist() == [0] * B


@pytest.mark.parametrize("V", [2048, 30011])
def test_bf16_logits_with_few_differences(gpu_lib, V):
    """Target and draft differ by one of two values, so that nearly all ids have one of two
    p / q, and the deciding ratio may be either of them to any accuracy."""
    B = 8
    g = torch.Generator().manual_seed(V)
    target = torch.randint(-40, 40, (B, 2, V), generator=g).to(torch.bfloat16) / 16
    step = torch.zeros(B, 1, V)
    for b in range(B):
        step[b, 0, torch.randperm(V, generator=g)[:[0, 1, 2, 40, V // 2, V - 2, V - 1, V][b]]] = 0.25
    draft = (target[:, :1].float() + step).to(torch.bfloat16)
    x = torch.stack([(draft[b, 0].float() - target[b, 0].float()).argmax() for b in range(B)])
    u = torch.full((B, 1), 1 - 2.0 ** -24)
    check((target, x[:, None].to(torch.int32), u, torch.rand(B, generator=g), draft))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_more_chunks_than_threads(gpu_lib, dtype):
    args = draw_inputs(6, 3, 1, 700001, dtype)
    check(args)
    target, drafts, _, us, draft = args
    draft = target[:, :1].clone()
    drafts = torch.tensor([[3], [400000], [700000]], dtype=torch.int32)
    for b in range(3):
        draft[b, 0, drafts[b, 0]] += 4.0
    check((target, drafts, torch.full((3, 1), 0.99), us, draft))
    check((target[:, :1], torch.zeros(3, 0, dtype=torch.int32), torch.zeros(3, 0), us))


@pytest.mark.parametrize("with_draft", [True, False])
def test_as_many_drafts_as_a_call_takes(gpu_lib, with_draft):
    """256 drafts of a sequence, the sequences differing in the one that falls."""
    B, k, V = 5, 256, 61
    target, drafts, ua, us, draft = draw_inputs(8, B, k, V, torch.float32, near=0.05)
    ua = ua * 1e-6
    for b, j in enumerate((0, 1, 63, 255)):
        ua[b, j], target[b, j, drafts[b, j]] = 0.9, -30.0
    n_acc, _ = check((target, drafts, ua, us, draft if with_draft else None))
    if with_draft:  # (without one a draft of p(x) < u <= 1e-6 falls too)
        assert n_acc.tolist() == [0, 1, 63, 255, 256]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("T,top", [(0.8, 48.0), (0.7, 42.0), (0.3, 18.0), (1.3, 78.0)])
@pytest.mark.parametrize("V", [2, 5000])
def test_the_temperature_is_taken_in_64_bits(gpu_lib, dtype, T, top, V):
    """Id 0 has p = 1 / (1 + e^(top / T)), and rounding T to 32 bits moves it by up to 60 x
    3e-8 of it: u half way between the two values lies 2e-7 of it or more from either, ten
    times the spacing of fp32 numbers and far past the sums' errors (1e-13)."""
    logits = torch.full((1, 1, V), -INF, dtype=dtype)
    logits[..., 0], logits[..., V - 1] = 0.0, top
    p = [1.0 / (1.0 + torch.tensor(top / t, dtype=torch.float64).exp().item())
         for t in (T, torch.tensor(T, dtype=torch.float32).item())]
    u = torch.tensor([(p[0] + p[1]) / 2])
    assert min(abs(float(u) / x - 1) for x in p) > 1e-7
    none = torch.zeros(1, 0)
    check((logits, none.int(), none, u), T)
    two, first = logits.expand(1, 2, V).clone(), torch.zeros(1, 1, dtype=torch.int32)
    check((two, first, u[None], torch.tensor([0.5]), None), T)
    even = torch.full((1, 1, V), -INF, dtype=dtype)
    even[..., 0] = even[..., V - 1] = 1.0
    check((two, first, 2 * u[None], torch.tensor([0.5]), even), T)


def test_a_bad_temperature_costs_the_others_nothing(gpu_lib):
    """Sequences without an answer (a greedy request's T = 0 among sampled ones) are not
    tested in 64 bits draft by draft: the call is not slower for them (it was, 38 times; twice
    is the slack of short timings), with whole logits and with a filtered vocabulary."""
    B, k, V = 6, 12, 151936
    args = [t.to(DEV) for t in draw_inputs(12, B, k, V, torch.bfloat16)]
    good = torch.ones(B, device=DEV)
    bad = torch.tensor([1.0, 0.0, -1.0, INF, 0.0, 1.0], device=DEV)

    def call(temps):
        return kernels.sample_verify(*args[:4], draft_logits=args[4], temperature=temps)

    def cost(temps):
        a, b = (torch.cuda.Event(enable_timing=True) for _ in range(2))
        a.record()
        for _ in range(10):
            call(temps)
        b.record()
        b.synchronize()
        return a.elapsed_time(b)
    for filtered in (False, True):
        if filtered:
            for x in (args[0], args[4]):
                x[:, :, 7::3] = -INF
        want, got = call(good), call(bad)
        for b in range(B):
            if 0.0 < float(bad[b]) < INF:
                assert got[0][b] == want[0][b] and torch.equal(got[1][b], want[1][b])
            else:
                assert got[0][b] == 0 and (got[1][b] == -1).all()
        times = [(cost(good), cost(bad)) for _ in range(12)]
        assert min(t[1] for t in times) < 2 * min(t[0] for t in times)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_greedy_drafts_of_a_whole_vocabulary(gpu_lib, dtype):
    """Drafts without a distribution (the greedy draft's) at the models' vocabulary: sequences
    whose drafts are the target's likeliest tokens, accepted to different lengths."""
    B, k, V, T = 6, 4, 151936, 0.7
    target, _, ua, us, _ = draw_inputs(15, B, k, V, dtype)
    drafts = target[:, :k].argmax(-1).to(torch.int32)
    for b in range(B):
        target[b, torch.arange(min(b, k)), drafts[b, :min(b, k)].long()] += 20.0
    n_acc, _ = check((target, drafts, ua, us, None), T)
    assert n_acc.tolist() == sorted(n_acc.tolist()) and n_acc[0] < k and n_acc[-1] == k
