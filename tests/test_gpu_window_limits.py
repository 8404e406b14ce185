"""Windowed and 8-bit attention at the ends of what its arguments may be."""

import pytest
import torch

from kvengine_amd import _lib
from test_gpu_window import DEV, POOLS, Case, i32

pytestmark = pytest.mark.gpu
CODES = {"fp32": _lib.DTYPE_F32, "bf16": _lib.DTYPE_BF16, "int8": _lib.DTYPE_I8, "e4m3": _lib.DTYPE_E4M3}


def call(c, window, sinks):
    """The C entry on a case, without the wrapper's limits; out holds 7 before it."""
    B, T, Hq, D = c.q.shape
    NB, Hkv, bs, _ = c.k.shape
    q, k, v = (t.to(DEV) for t in (c.q, c.k, c.v))
    ks, vs = (None if t is None else t.to(DEV) for t in (c.ks, c.vs))
    table, start, max_ctx = c.table(), i32(c.starts), max(c.starts) + T
    out = torch.full_like(q, 7.0)
    lib, dtype, pool = _lib.lib(), CODES[c.dtype], CODES[c.pool]
    n = lib.kve_window_workspace_bytes(B, T, Hq, Hkv, D, max_ctx, window, sinks, dtype, pool)
    ws = torch.empty(n, dtype=torch.uint8, device=DEV)
    rc = lib.kve_paged_window_attn(q.data_ptr(), k.data_ptr(), v.data_ptr(), None if ks is None else ks.data_ptr(),
                                   None if vs is None else vs.data_ptr(), table.data_ptr(), None, start.data_ptr(),
                                   None, B, T, Hq, Hkv, D, bs, table.shape[1], B, NB, max_ctx, window, sinks,
                                   D ** -0.5, dtype, pool, out.data_ptr(), ws.data_ptr() if n else None, n,
                                   torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    assert rc == 0, lib.kve_last_error()
    return out.cpu()


@pytest.mark.parametrize("pool,dtype", POOLS)
@pytest.mark.parametrize("T,start", [(1, 90), (9, 700), (1, 3000)])
def test_as_many_sinks_as_there_are_numbers(T, start, pool, dtype):
    """Sinks up to the largest 32-bit number are all keys, beside a window and without one."""
    c = Case(30 + T, [start, 3], T, 8, 2, 64, pool, dtype)
    for sinks in (2 ** 31 - 1, 2 ** 31 - 33, 2 ** 30 + 1, start + T):
        for window in (0, 5):
            c.check(call(c, window, sinks), None, 0)
