"""Infinities among K and V rows on their way into an 8-bit block."""

import math

import pytest
import torch

from kvengine_amd import kernels

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("pool,top", [(torch.int8, 127.0), (torch.float8_e4m3fn, 448.0)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_infinities(dtype, pool, top):
    """The largest code beside finite values, which alone make the scale; beside zeros alone the
    scale is 0, and so is what the infinity stands for."""
    x = torch.zeros(1, 2, 2, 64)
    x[..., 3], x[..., 7], x[..., 9] = math.inf, -math.inf, math.nan
    x[:, :, 0, 20] = -2.0
    p = [torch.zeros(s, device="cuda").to(pool) for s in ((1, 2, 16, 64), (1, 2, 64, 16))]
    s = [torch.full((1, 2), math.nan, device="cuda") for _ in range(2)]
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")
    d = x.to("cuda", dtype)
    kernels.kv_write_q8(d, d, *p, *s, i32([[0]]), i32([0]))
    k, v = p[0][0, :, :2].float().cpu(), p[1][0, :, :, :2].float().cpu().transpose(1, 2)
    scale = float(torch.tensor(2.0 / 127)) if pool is torch.int8 else 2.0 ** -7  # 2 = 256 2^-7
    for c, sc in zip((k, v), s):
        assert sc.tolist() == [[scale, 0.0]]
        assert bool((c[0, :, 3] == top).all()) and bool((c[0, :, 7] == -top).all())
        assert bool((c[0, :, 9] == 0).all())
        assert bool((c[0, :, 20] == (-127 if pool is torch.int8 else -256)).all())
        assert not bool(c[1].any())
