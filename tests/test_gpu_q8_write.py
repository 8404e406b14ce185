"""K/V rows into an 8-bit cache: codes and scales are exactly those of the definition in
64 bits (a quotient of two 32-bit numbers that is not a border of two codes is at least
2^-33 of it away from one, which 64 bits resolve)."""

import random
from fractions import Fraction

import pytest
import torch

from kvengine_amd import kernels

pytestmark = pytest.mark.gpu
DEV = "cuda"
POOLS = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}
DT = {"bf16": torch.bfloat16, "fp32": torch.float32}


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def scale_of(top, pool):
    """(top: the largest finite value, a Python float)"""
    if top == 0.0:
        return 0.0
    if pool == "int8":
        return max(float(torch.tensor(top / 127.0, dtype=torch.float64).float()), 2.0 ** -100)
    e = -100
    while top > 448 * 2.0 ** e:
        e += 1
    return 2.0 ** e


def code_of(x, s, pool):
    x = torch.where(torch.isnan(x), 0.0, x.double())
    if s == 0.0:
        return torch.zeros_like(x)
    if pool == "int8":
        return (x / s).round().clamp(-127, 127)
    q = (x / s).clamp(-448, 448)
    step = 2.0 ** (torch.floor(torch.log2(q.abs().clamp_min(2.0 ** -6))).clamp_min(-6) - 3)
    return (q / step).round() * step


def write(c, k_new, v_new, start, table, seq, T, pool):
    """The definition, on the CPU pools in c (codes as float64)."""
    bs = c["k"].shape[2]
    for lb in range(start // bs, (start + T - 1) // bs + 1):
        blk = table[lb]
        lo, hi = max(start, lb * bs), min(start + T, (lb + 1) * bs)
        o, n = lo - lb * bs, hi - lo
        for name, rows in (("k", k_new), ("v", v_new)):
            for h in range(rows.shape[2]):
                r = rows[seq, lo - start:hi - start, h].double()
                fin = r[torch.isfinite(r)].abs()
                s = scale_of(float(fin.max()) if fin.numel() else 0.0, pool)
                tile = c[name][blk, h] if name == "k" else c[name][blk, h].t()  # [bs, D]
                if o:
                    was = float(c[name + "s"][blk, h])
                    s = max(s, was)
                    if s != was:
                        tile[:o] = code_of(tile[:o] * was, s, pool)
                tile[o:o + n] = code_of(r, s, pool)
                c[name + "s"][blk, h] = s


def pools(seed, nb, Hkv, bs, D, pool):
    g = torch.Generator().manual_seed(seed)
    hi = 127 if pool == "int8" else 448
    mk = lambda *s: (40 * torch.randn(*s, generator=g)).clamp(-hi, hi).round().to(POOLS[pool])
    sc = lambda: 2.0 ** torch.randint(-6, 2, (nb, Hkv), generator=g).float()
    return {"k": mk(nb, Hkv, bs, D), "v": mk(nb, Hkv, D, bs), "ks": sc(), "vs": sc()}


def same(p, c):
    for n in ("k", "v", "ks", "vs"):
        got = p[n].cpu().double()
        assert torch.equal(got, c[n].double()), (n, (got != c[n].double()).nonzero()[:4].tolist())


@pytest.mark.parametrize("pool", list(POOLS))
@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("starts,T,Hkv,D,bs,counts", [
    ([0], 1, 1, 64, 16, None), ([5, 15, 16, 31], 1, 2, 128, 16, None),
    ([0, 3, 14, 40], 5, 2, 64, 16, [5, 0, 3, 1]), ([7, 100], 33, 2, 128, 32, None),
    ([1, 47, 48], 50, 1, 64, 48, [50, 49, 2]), ([9], 200, 3, 64, 16, None), ([130], 90, 1, 128, 64, None), ([3, 40], 9, 2, 64, 32, None)])
def test_write(starts, T, Hkv, D, bs, counts, dtype, pool):
    r, g = random.Random(T), torch.Generator().manual_seed(D + T)
    B = len(starts)
    need = [-(-(s + T) // bs) for s in starts]
    nb = sum(need) + 2
    ids = list(range(nb))
    r.shuffle(ids)
    tables = [[ids.pop() for _ in range(n)] for n in need]
    p = pools(D, nb, Hkv, bs, D, pool)
    c = {n: t.double() for n, t in p.items()}
    k, v = (torch.randn(B, T, Hkv, D, generator=g) * torch.exp(2 * torch.randn(B, T, Hkv, 1, generator=g))
            for _ in range(2))
    k, v = k.to(DT[dtype]), v.to(DT[dtype])
    w = max(need)
    table = i32([t + [-1] * (w - len(t)) for t in tables])
    p = {n: t.to(DEV) for n, t in p.items()}
    n = counts or [T] * B
    # a second pass behind the first, one row a sequence, and the first again in its place
    # after a rollback: scales stay
    for again in range(3):
        kernels.kv_write_q8(k.to(DEV), v.to(DEV), p["k"], p["v"], p["ks"], p["vs"], table, i32(starts),
                            q_lens=None if counts is None else i32(counts))
        for b in range(B):
            if n[b]:
                write(c, k, v, starts[b], tables[b], b, n[b], pool)
        same(p, c)
        if again == 0:
            k, v = k * 3, v / 5


@pytest.mark.parametrize("pool", list(POOLS))
def test_values_on_the_borders_of_two_codes(pool):
    """bf16 values that are odd multiples of half a step, and fp32 neighbours of the borders."""
    s = 2.0 ** -3 if pool == "e4m3" else float(torch.tensor(127 * 0.1).float() / 127)
    if pool == "int8":
        top = torch.tensor(12.7)
        s = float((top.double() / 127).float())
        mid = torch.tensor([float(Fraction(2 * n + 1, 2) * Fraction(s)) for n in range(-63, 63)],
                           dtype=torch.float64).float()
        row = torch.cat([mid, top[None], -top[None]])
    else:
        grid = torch.tensor([i / 512 for i in range(9)] + [(8 + i) * 2.0 ** e for e in range(-9, 5) for i in range(9)])
        mid = ((grid[1:] + grid[:-1]) / 2 * s)[:125]
        row = torch.cat([mid, torch.tensor([448 * s, -448 * s, 0.0])])
    rows = [row, torch.nextafter(row, torch.full_like(row, 1e9)),
            torch.nextafter(row, torch.full_like(row, -1e9)), -row]
    x = torch.stack(rows)
    # the neighbours of the largest value would move the scale
    x = x.clamp(float(row.min()), float(row.max()))
    x = x[None, :, None, :].contiguous()
    assert x.shape[-1] == 128
    p = {n: t.to(DEV) for n, t in pools(1, 1, 1, 16, 128, pool).items()}
    c = {n: t.cpu().double() for n, t in p.items()}
    write(c, x, x, 0, [0], 0, 4, pool)
    kernels.kv_write_q8(x.to(DEV), x.to(DEV), p["k"], p["v"], p["ks"], p["vs"], i32([[0]]), i32([0]))
    same(p, c)
    assert float(p["ks"][0, 0]) == (s if pool == "int8" else float(c["ks"][0, 0]))


@pytest.mark.parametrize("pool", list(POOLS))
def test_zeros_tiny_large_and_non_finite_values(pool):
    inf, nan = float("inf"), float("nan")
    base = torch.linspace(-1, 1, 64)
    rows = [torch.zeros(64), base * 1e-37, base * 3e38, base, torch.full((64,), inf)]
    rows[3] = rows[3].clone()
    rows[3][:4] = torch.tensor([inf, -inf, nan, 0.5])
    for row in rows:
        for o in (0, 6):
            p = {n: t.to(DEV) for n, t in pools(2, 2, 1, 16, 64, pool).items()}
            p["ks"].fill_(2.0 ** -90)
            p["vs"].fill_(2.0 ** -90)
            c = {n: t.cpu().double() for n, t in p.items()}
            x = row[None, None, None].expand(1, 2, 1, 64).contiguous()
            write(c, x, x, o, [1], 0, 2, pool)
            kernels.kv_write_q8(x.to(DEV), x.to(DEV), p["k"], p["v"], p["ks"], p["vs"], i32([[1]]), i32([o]))
            same(p, c)
    assert float(p["ks"][1, 0]) == 2.0 ** -90  # infinities do not count for a scale


def test_bad_rows_blocks_and_lengths_write_nothing():
    p = {n: t.to(DEV) for n, t in pools(3, 4, 2, 16, 64, "int8").items()}
    was = {n: t.clone() for n, t in p.items()}
    x = torch.randn(4, 3, 2, 64, device=DEV)
    table = i32([[9, 9], [-1, -1], [0, 1], [2, 3]])
    kernels.kv_write_q8(x, x, p["k"], p["v"], p["ks"], p["vs"], table, i32([0, 5, -1, 32]))
    kernels.kv_write_q8(x, x, p["k"], p["v"], p["ks"], p["vs"], table, i32([0, 0, 0, 2 ** 31 - 2]),
                        seq_rows=i32([-1, 4, 3, 3]), q_lens=i32([3, 3, -2, 0]))
    kernels.kv_write_q8(x, x, p["k"], p["v"], p["ks"], p["vs"], table, i32([0, 0, 0, 2 ** 31 - 2]),
                        seq_rows=i32([3, 3, 3, 3]))
    for n in p:
        assert torch.equal(p[n].view(torch.uint8), was[n].view(torch.uint8))


@pytest.mark.parametrize("pool", list(POOLS))
def test_strided_rows_and_another_stream(pool):
    """Rows as views of a fused projection's output, as forward passes hand them over."""
    g = torch.Generator().manual_seed(4)
    qkv = torch.randn(2, 20, 3 * 2 * 128, generator=g).to(torch.bfloat16)
    k, v = qkv[..., 256:512].view(2, 20, 2, 128), qkv[..., 512:].view(2, 20, 2, 128)
    p = {n: t.to(DEV) for n, t in pools(5, 6, 2, 16, 128, pool).items()}
    c = {n: t.cpu().double() for n, t in p.items()}
    dev = qkv.to(DEV)
    kd, vd = dev[..., 256:512].view(2, 20, 2, 128), dev[..., 512:].view(2, 20, 2, 128)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        kernels.kv_write_q8(kd, vd, p["k"], p["v"], p["ks"], p["vs"], i32([[0, 2], [5, 4]]), i32([3, 0]),
                            seq_rows=i32([1, 0]))
    torch.cuda.synchronize()
    write(c, k, v, 0, [5, 4], 0, 20, pool)
    write(c, k, v, 3, [0, 2], 1, 20, pool)
    same(p, c)


def test_offsets_past_32_bits():
    """Pools of more than 4 GiB of codes, the sequence in the last blocks."""
    nb, Hkv, D = 1_100_000, 2, 128
    p = dict(k=torch.zeros(nb, Hkv, 16, D, dtype=torch.int8, device=DEV),
             v=torch.zeros(nb, Hkv, D, 16, dtype=torch.int8, device=DEV),
             ks=torch.zeros(nb, Hkv, device=DEV), vs=torch.zeros(nb, Hkv, device=DEV))
    assert p["k"].numel() > 1 << 32
    c = {n: t[:4].cpu().double() for n, t in p.items()}
    x = torch.randn(1, 40, Hkv, D, generator=torch.Generator().manual_seed(6)).to(torch.bfloat16)
    kernels.kv_write_q8(x.to(DEV), x.to(DEV), p["k"], p["v"], p["ks"], p["vs"],
                        i32([[nb - 1, nb - 3, nb - 2]]), i32([0]))
    write(c, x, x, 0, [3, 1, 2], 0, 40, "int8")
    same({n: t[nb - 4:] for n, t in p.items()}, c)
    assert not any(bool(t[:nb - 4].any()) for t in p.values())


@pytest.mark.parametrize("B,T,Hkv", [(1, 1, 2), (3, 1, 2), (1, 5, 1), (2, 1, 1), (1, 1, 1)])
def test_strides_of_dimensions_of_one_do_not_matter(B, T, Hkv):
    """K and V rows whose strides differ in dimensions of one element only."""
    g = torch.Generator().manual_seed(7)
    x = torch.randn(B, T, Hkv, 64, generator=g)
    p = {n: t.to(DEV) for n, t in pools(8, 6, Hkv, 16, 64, "e4m3").items()}
    c = {n: t.cpu().double() for n, t in p.items()}
    k = x.to(DEV)
    odd = [s if n > 1 else s + 8 * (i + 1) for i, (n, s) in enumerate(zip(x.shape, x.stride()))]
    v = k.as_strided(x.shape, odd)
    kernels.kv_write_q8(k, v, p["k"], p["v"], p["ks"], p["vs"], i32([[1, 0], [3, 2], [5, 4]]),
                        i32([15, 0, 3]))
    for b, (start, table) in enumerate([(15, [1, 0]), (0, [3, 2]), (3, [5, 4])][:B]):
        write(c, x, x, start, table, b, T, "e4m3")
    same(p, c)
