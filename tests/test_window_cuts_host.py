"""Where the walks of windowed and 8-bit attention are cut: read off the workspace, which holds a
state for each row tile and cut. Nothing is launched."""

import types

import pytest

from kvengine_amd import _lib
from kvengine_amd.speculative import CTX_STEP, _IterationGraphs

I8, BF16, F32 = _lib.DTYPE_I8, _lib.DTYPE_BF16, _lib.DTYPE_F32


def cuts(ctx, T=1, Hq=14, Hkv=2, D=64, window=0, sinks=0, dtype=BF16, pool=I8):
    n = _lib.lib().kve_window_workspace_bytes(1, T, Hq, Hkv, D, ctx, window, sinks, dtype, pool)
    R = Hq // Hkv * T
    rows = 16 if R <= 16 else -(-R // 64) * 64
    per = Hkv * rows * (D + 2) * 4
    assert n % per == 0
    return n // per or 1


def lengths(ctx, T, dtype, **kw):
    """The chunk lengths (in steps) that the number of cuts under this bound allows."""
    n, steps = cuts(ctx, T, dtype=dtype, **kw), -(-ctx // 64)
    return {c for c in range(1, steps + 64) if -(-steps // c) == n}


@pytest.mark.parametrize("T", [1, 5])
def test_one_order_between_multiples_of_256(T):
    """Some chunk length fits all bounds of a bucket: the first and last rows of its range, and those
    between."""
    for end in list(range(1280, 2600, 256)) + list(range(4096, 9000, 256)) + [65536, 65792, 66048, 81920, 82176]:
        common = None
        for ctx in (end - 255, end - 200, end - 65, end - 64, end - 1, end):
            got = lengths(ctx, T, BF16)
            common = got if common is None else common & got
        assert common, (T, end)


@pytest.mark.parametrize("T,Hkv", [(5, 2), (40, 8), (101, 8), (201, 8)])
def test_one_order_under_every_bound_up_to_1024(T, Hkv):
    """Also where so many rows share a walk that it is cut in few chunks."""
    common = None
    for ctx in (T, 256, 300, 512, 600, 700, 896, 1000, 1024):
        got = lengths(max(ctx, T), T, BF16, Hq=8 * Hkv, Hkv=Hkv, pool=BF16)
        common = got if common is None else common & got
    assert common


@pytest.mark.parametrize("window,sinks", [(0, 0), (800, 300), (1000, 0), (5000, 4)])
def test_one_token_in_one_piece_up_to_1024(window, sinks):
    for ctx in (1, 64, 500, 896, 897, 960, 1000, 1023, 1024):
        assert cuts(ctx, window=window, sinks=sinks) == 1, ctx
    # the window's own walk is short enough, or not
    assert (cuts(1025, window=window, sinks=sinks) == 1) is (window == 1000)


def test_a_bound_does_not_make_sinks_longer_than_the_history():
    for ctx in (700, 3000, 9000):
        assert cuts(ctx, window=10, sinks=2 ** 31 - 1) == cuts(ctx)


def graphs(by_step, t, d, k=4):
    g = _IterationGraphs.__new__(_IterationGraphs)
    pool = types.SimpleNamespace(max_blocks=1000)
    g.k, g.by_step = k, by_step
    g.t, g.d = (types.SimpleNamespace(length=n, pool=pool, block_size=16) for n in (t, d))
    return g


def test_buckets_of_replayed_iterations():
    """A bucket's bound cuts as each pass's own does, or the iteration runs eagerly."""
    for n in range(1, 2500):
        for u in (1, 2):
            d = n + 1 - u
            exact = [d + u + j for j in range(4)] + [n + 1 + 4]
            b = graphs(True, n, d).bucket(u)
            if b is None:
                assert any(lo < m <= max(exact) for m in [897] + list(range(1025, 2600, 256)) for lo in exact)
                continue
            assert b >= max(exact)
            for c in exact:
                assert (c <= 1024) == (b <= 1024)
                assert b <= 1024 or -(-c // CTX_STEP) == b // CTX_STEP
            assert b == graphs(False, n, d).bucket(u)
