"""Alternatives of rows with a NaN, wherever the likeliest ids lie."""

import math

import pytest
import torch

from kvengine_amd import kernels

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("at", [0, 1, 127, 350001])
def test_a_nan_ranks_first_where_the_likely_ids_lie_together(at, dtype):
    """Likely ids in so few of the selection's 64 sets that their n-th maximum bounds nothing, and
    too many for its list: the n largest are then taken one after another."""
    V = 700001
    g = torch.Generator().manual_seed(at)
    i = torch.arange(V)
    x = torch.randn(3, V, generator=g)
    group = 128 if dtype is torch.bfloat16 else 64
    x += 5.0 * (i // group % 1024 < 496)
    x[2] = 1.0  # equal logits
    x = x.to(dtype)
    x[0, at] = x[2, at] = math.nan
    ids = kernels.token_logprobs(x.cuda(), torch.zeros(3, dtype=torch.int32, device="cuda"), top=32)[2].cpu()
    want = torch.sort(x.double(), dim=-1, descending=True, stable=True).indices[:, :32]
    assert int(want[0, 0]) == at
    assert ids.tolist() == want.tolist()
