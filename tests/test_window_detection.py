"""Models of any make are asked for their windows: ones without layers, with layers in wrappers."""

import types

import pytest
import torch

from kvengine_amd.arch import TINY
from kvengine_amd.forward import forward_with_own_cache, windowed, windows
from kvengine_amd.model import build_model
from kvengine_amd.paged import ContiguousKVCache, PagedKVCache


class Wrapped(torch.nn.Module):
    """A layer in a module that forwards its attributes."""

    def __init__(self, layer):
        super().__init__()
        self.inner = layer

    def __getattr__(self, name):
        if name == "inner":
            return super().__getattr__(name)
        return getattr(self.inner, name)


class ConfigOnly(torch.nn.Module):
    """What a cache's sizes are read from, and nothing else."""

    def __init__(self):
        super().__init__()
        self.config = types.SimpleNamespace(num_hidden_layers=2, num_attention_heads=4, num_key_value_heads=2,
                                            hidden_size=256, head_dim=64)
        self.weight = torch.nn.Parameter(torch.zeros(1))


def test_a_model_without_layers_has_no_window():
    m = ConfigOnly()
    assert not windowed(m) and windows(m) == ()
    cache = ContiguousKVCache.for_model(m, 21)
    assert cache.k.shape == (2, 1, 2, 21, 64) and cache.room == 21
    assert PagedKVCache.for_model(m, 4).k.shape == (2, 4, 2, 16, 64)


def test_layers_in_wrappers():
    m = build_model(TINY, seed=3, dtype=torch.float32, device="cpu")
    layers = m.model.layers
    m.model.layers = torch.nn.ModuleList([Wrapped(layer) for layer in layers])
    assert not windowed(m) and windows(m) == ((None, 0),) * len(layers)
    assert ContiguousKVCache.for_model(m, 21).room == 21
    m.model.layers[1].self_attn.sliding_window = 7
    m.model.layers[1].self_attn.window_sinks = 3
    assert windowed(m) and windows(m)[:2] == ((None, 0), (7, 3))
    assert ContiguousKVCache.for_model(m, 21).room == 32


@pytest.mark.gpu
@pytest.mark.parametrize("window", [None, 9])
def test_a_pass_over_layers_in_wrappers(window):
    """Module calls: the same bits as without the wrappers."""
    ids = torch.randint(0, 1000, (1, 40), generator=torch.Generator().manual_seed(1)).cuda()
    m = build_model(TINY, seed=3, dtype=torch.float32, device="cuda")
    for layer in m.model.layers:
        layer.self_attn.sliding_window = window
        del layer.self_attn.qkv_weight
    want = forward_with_own_cache(m, ids, PagedKVCache.for_model(m, 8).new_sequence("a"), all_logits=True)
    m.model.layers = torch.nn.ModuleList([Wrapped(layer) for layer in m.model.layers])
    got = forward_with_own_cache(m, ids, PagedKVCache.for_model(m, 8).new_sequence("a"), all_logits=True)
    assert torch.equal(got, want)
