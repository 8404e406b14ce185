"""A block that holds a NaN already (codes from elsewhere; the write makes none) keeps it when a new
row raises the block's scale."""

import pytest
import torch

from kvengine_amd import kernels

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("start", [1, 5, 15])
def test_a_held_nan_stays(start, D):
    codes = torch.randint(0, 120, (1, 1, 16, D), generator=torch.Generator().manual_seed(start)).to(torch.uint8)
    codes[0, 0, 0, 3], codes[0, 0, start - 1, D - 1] = 0x7f, 0xff
    k = codes.view(torch.float8_e4m3fn).cuda()
    v = codes.transpose(2, 3).contiguous().view(torch.float8_e4m3fn).cuda()
    ks, vs = (torch.full((1, 1), 2.0 ** -6, device="cuda") for _ in range(2))
    before = k.float().cpu()[0, 0]
    x = torch.full((1, 1, 1, D), 448.0, device="cuda")
    i32 = lambda n: torch.tensor(n, dtype=torch.int32, device="cuda")
    kernels.kv_write_q8(x, x, k, v, ks, vs, i32([[0]]), i32([start]))
    assert float(ks) == float(vs) == 1.0
    for got in (k.float().cpu()[0, 0], v.float().cpu()[0, 0].t()):
        assert torch.equal(torch.isnan(got), torch.isnan(before))
        want = (before[:start] * 2.0 ** -6).to(torch.float8_e4m3fn).float()
        assert torch.equal(got[:start].nan_to_num(0.0), want.nan_to_num(0.0))
        assert bool((got[start] == 448.0).all())
        assert torch.equal(got[start + 1:].nan_to_num(0.0), before[start + 1:].nan_to_num(0.0))
