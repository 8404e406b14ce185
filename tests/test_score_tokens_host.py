"""What score_tokens refuses, it refuses before the cache takes the text."""

import pytest
import torch

from kvengine_amd import decode
from kvengine_amd.arch import TINY
from kvengine_amd.model import build_model


class Untouched:
    length = 0

    def __getattr__(self, name):
        raise AssertionError(f"the cache was asked for {name}")


@pytest.mark.parametrize("top", [-1, 33, 1 << 20])
@pytest.mark.parametrize("head", ["plain", "other"])
def test_alternatives(top, head):
    model = build_model(TINY, seed=3, dtype=torch.float32, device="cpu")
    if head == "other":
        model.lm_head = torch.nn.Sequential(model.lm_head)
    with pytest.raises(ValueError, match="alternatives"):
        decode.score_tokens(model, torch.zeros(1, 4, dtype=torch.long), Untouched(), top=top)


def test_more_alternatives_than_ids():
    model = build_model(TINY, seed=3, dtype=torch.float32, device="cpu")
    model.lm_head = torch.nn.Linear(TINY.hidden, 5, bias=False)
    with pytest.raises(ValueError, match="6 alternatives, at most 5"):
        decode.score_tokens(model, torch.zeros(1, 4, dtype=torch.long), Untouched(), top=6)
