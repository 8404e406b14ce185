"""Refusals of the windowed and 8-bit attention, the 8-bit write and the log probabilities:
nothing is launched, so none of it needs a GPU."""

import pytest
import torch

from kvengine_amd import _lib, kernels


def call_attn(**kw):
    a = dict(q=16, k=16, v=16, ks=None, vs=None, tables=16, rows=None, start=16, q_lens=None, B=1,
             T=5, Hq=14, Hkv=2, D=64, bs=16, max_blocks=8, num_rows=1, num_blocks=8, max_ctx=128,
             window=64, sinks=4, scale=0.125, dtype=1, pool=1, out=16, ws=16, wsb=1 << 30)
    a.update(kw)
    rc = _lib.lib().kve_paged_window_attn(*a.values(), None)
    return rc, _lib.lib().kve_last_error().decode()


@pytest.mark.parametrize("change,text", [
    (dict(q=None), "null pointer"), (dict(out=None), "null pointer"), (dict(tables=None), "null pointer"),
    (dict(T=0), "tokens"), (dict(B=-1), "tokens"), (dict(Hq=15), "heads"), (dict(D=96), "heads"),
    (dict(Hkv=0), "heads"), (dict(window=-1), "window"), (dict(sinks=-1), "sinks"),
    (dict(T=1 << 28), "tokens"), (dict(max_blocks=1 << 27, max_ctx=(1 << 30) + 1), "max_ctx"),
    (dict(B=1 << 22, T=1), "too large"), (dict(bs=24), "block_size"), (dict(bs=0), "block_size"),
    (dict(bs=1 << 21), "block_size"), (dict(max_ctx=129), "max_ctx"), (dict(max_ctx=0), "max_ctx"),
    (dict(num_blocks=0), "blocks"), (dict(num_blocks=1 << 30), "too large"),
    (dict(scale=0.0), "scale"), (dict(scale=float("nan")), "scale"), (dict(scale=float("inf")), "scale"),
    (dict(dtype=2, pool=2), "dtype"), (dict(dtype=0), "dtype"), (dict(pool=0), "dtype"),
    (dict(pool=4), "dtype"), (dict(pool=2), "scales"), (dict(pool=3, ks=16), "scales"),
    (dict(q=8), "16-byte"), (dict(k=8), "16-byte"), (dict(out=24), "16-byte"),
])
def test_attention_refuses(change, text):
    rc, msg = call_attn(**change)
    assert rc == -1 and text in msg and "kve_paged_window_attn" in msg


def test_attention_workspace():
    need = _lib.lib().kve_window_workspace_bytes(1, 1, 14, 2, 64, 8000, 0, 0, 1, 1)
    assert need > 0
    long = dict(T=1, max_blocks=500, max_ctx=8000, window=0)
    assert call_attn(**long, wsb=need - 1)[0] == -2
    assert call_attn(**long, ws=None)[0] == -2
    rc, msg = call_attn(**long, ws=8, wsb=need)
    assert rc == -1 and "16-byte" in msg
    size = _lib.lib().kve_window_workspace_bytes
    assert size(0, 1, 14, 2, 64, 8000, 0, 0, 1, 1) == size(1, 1, 14, 2, 96, 8000, 0, 0, 1, 1) == 0
    assert call_attn(B=0)[0] == 0


def call_write(**kw):
    a = dict(k=16, v=16, stride=128, kp=16, vp=16, ks=16, vs=16, tables=16, rows=None, start=16,
             q_lens=None, B=1, T=5, Hkv=2, D=64, bs=16, max_blocks=8, num_rows=1, num_blocks=8,
             dtype=1, pool=2)
    a.update(kw)
    rc = _lib.lib().kve_kv_write_q8(*a.values(), None)
    return rc, _lib.lib().kve_last_error().decode()


@pytest.mark.parametrize("change,text", [
    (dict(k=None), "null pointer"), (dict(vs=None), "null pointer"), (dict(start=None), "null pointer"),
    (dict(T=0), "bad sizes"), (dict(B=-1), "bad sizes"), (dict(num_blocks=0), "bad sizes"),
    (dict(bs=8), "block_size"), (dict(bs=0), "block_size"), (dict(D=60), "head_dim"),
    (dict(D=256), "head_dim"), (dict(dtype=2), "dtype"), (dict(pool=1), "pool dtype"),
    (dict(stride=120), "stride"), (dict(stride=132), "stride"), (dict(k=8), "aligned"),
    (dict(vp=20), "aligned"), (dict(B=1 << 28, T=1 << 10), "too large"),
    (dict(B=1 << 24, T=1), "too large"),
])
def test_write_refuses(change, text):
    rc, msg = call_write(**change)
    assert rc == -1 and text in msg and "kve_kv_write_q8" in msg


def test_write_of_no_sequences_is_nothing():
    assert call_write(B=0)[0] == 0


def call_logprobs(**kw):
    a = dict(x=16, stride=1000, tokens=16, rows=4, V=1000, top=5, dtype=1, lp=16, H=16, ids=16, tops=16,
             ws=16, wsb=1 << 20)
    a.update(kw)
    rc = _lib.lib().kve_token_logprobs(*a.values(), None)
    return rc, _lib.lib().kve_last_error().decode()


@pytest.mark.parametrize("change,rc,text", [
    (dict(x=None), -1, "null pointer"), (dict(tokens=None), -1, "null pointer"),
    (dict(ids=None), -1, "null pointer"), (dict(tops=None), -1, "null pointer"),
    (dict(rows=-1), -1, "rows"), (dict(V=0), -1, "rows"), (dict(top=33), -1, "alternatives"),
    (dict(top=-1), -1, "alternatives"), (dict(V=4), -1, "alternatives"), (dict(dtype=2), -1, "dtype"),
    (dict(x=17), -1, "aligned"), (dict(x=18, dtype=0), -1, "aligned"), (dict(ws=None), -1, "workspace"),
    (dict(ws=8), -1, "16-byte"), (dict(wsb=8), -2, "workspace"),
    (dict(rows=1 << 24, V=1 << 20), -1, "too large"),
    (dict(rows=1 << 22, wsb=1 << 40), -1, "too large"),
])
def test_logprobs_refuses(change, rc, text):
    got, msg = call_logprobs(**change)
    assert got == rc and text in msg and "kve_token_logprobs" in msg


def test_logprobs_of_no_rows_is_nothing():
    assert call_logprobs(rows=0)[0] == 0


def test_wrappers_refuse_before_anything_runs():
    q = torch.zeros(1, 1, 4, 64)
    with pytest.raises(ValueError, match="on the GPU|contiguous"):
        kernels.paged_window_attn(q, *[None] * 4, 16, 4)
    with pytest.raises(ValueError, match="on the GPU|contiguous"):
        kernels.paged_q8_attn(q, *[None] * 6, 16)
    with pytest.raises(ValueError, match="on the GPU"):
        kernels.kv_write_q8(q, q, *[None] * 6)
    with pytest.raises(ValueError, match="on the GPU"):
        kernels.token_logprobs(torch.zeros(2, 8), torch.zeros(2, dtype=torch.int32))
