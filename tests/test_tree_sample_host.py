"""Refusals of the tree and sampled verification entry points, and forward_hidden's tree
argument checks: nothing is launched, so none of it needs a GPU."""

import os
import subprocess
import sys

import pytest
import torch

from kvengine_amd import _lib, kernels


def call_tree_attn(**kw):
    a = dict(q=16, k=16, v=16, masks=16, tables=16, rows=None, start=16, q_lens=None, B=1, T=5,
             Hq=14, Hkv=2, D=64, bs=16, max_blocks=8, num_rows=1, num_blocks=8, max_ctx=128,
             unit=0, kw=0, scale=0.125, dtype=1, plan=None, out=16, ws=None, wsb=0, layout=0)
    a.update(kw)
    rc = _lib.lib().kve_paged_tree_attn(*a.values(), None)
    return rc, _lib.lib().kve_last_error().decode()


@pytest.mark.parametrize("change,text", [
    (dict(masks=None), "masks"), (dict(masks=12), "masks"), (dict(T=65), "65 nodes"),
    (dict(scale=0.0), "scale"), (dict(scale=float("nan")), "scale"), (dict(q=None), "null pointer"),
    (dict(q=8), "16-byte"), (dict(D=96), "head_dim"), (dict(Hq=15), "multiple"),
    (dict(dtype=3), "dtype"), (dict(max_ctx=129), "max_ctx"), (dict(T=0), "q_len"),
    (dict(kw=3), "key_waves"), (dict(layout=2), "workspace"), (dict(B=-1), "num_seqs"),
])
def test_tree_attention_refuses(change, text):
    rc, msg = call_tree_attn(**change)
    assert rc in (-1, -2) and text in msg and "kve_paged_tree_attn" in msg


def test_tree_attention_of_no_sequences_is_nothing():
    assert call_tree_attn(B=0)[0] == 0


@pytest.mark.parametrize("args,text", [
    ((None, None, 1, 4, 16, 16), "null pointer"), ((16, None, 1, 4, None, None), "null pointer"),
    ((16, None, 1, 65, 16, 16), "65 nodes"), ((16, None, 1, 0, 16, 16), "0 nodes"),
    ((16, None, -1, 4, 16, 16), "-1 sequences"),
])
def test_tree_masks_refuses(args, text):
    assert _lib.lib().kve_tree_masks(*args, None) == -1
    assert text in _lib.lib().kve_last_error().decode()


def call_accept(**kw):
    a = dict(tokens=16, parents=16, preds=16, counts=None, lens=16, num_rows=4, rows=None, B=2, n=8,
             n_acc=16, emitted=16, path=16, keep=16, k=16, v=16, tables=16, L=2, Hkv=2, D=64, bs=16,
             max_blocks=8, num_blocks=8, dtype=1)
    a.update(kw)
    rc = _lib.lib().kve_tree_accept(*a.values(), None)
    return rc, _lib.lib().kve_last_error().decode()


@pytest.mark.parametrize("change,text", [
    (dict(tokens=None), "null pointer"), (dict(path=None), "null pointer"), (dict(n=65), "65 nodes"),
    (dict(n=0), "0 nodes"), (dict(lens=None), "need lens"), (dict(num_rows=0), "need lens"),
    (dict(k=None), "go together"), (dict(v=None), "go together"), (dict(tables=None), "bad sizes"),
    (dict(L=0), "bad sizes"), (dict(bs=0), "bad sizes"), (dict(dtype=2), "dtype"),
    (dict(D=60), "head_dim"), (dict(k=8), "16-byte"), (dict(max_blocks=1 << 27), "too large"),
])
def test_tree_accept_refuses(change, text):
    rc, msg = call_accept(**change)
    assert rc == -1 and text in msg


def call_sample(**kw):
    a = dict(target=16, ts=5000, tp=1000, draft=16, ds=4000, dp=1000, drafts=16, ua=16, us=16,
             temps=None, temp=1.0, lens=None, num_rows=0, rows=None, B=2, k=4, V=1000, dtype=1,
             n_acc=16, emitted=16, keep=None, ws=16, wsb=1 << 20)
    a.update(kw)
    rc = _lib.lib().kve_sample_verify(*a.values(), None)
    return rc, _lib.lib().kve_last_error().decode()


@pytest.mark.parametrize("change,rc,text", [
    (dict(target=None), -1, "null pointer"), (dict(drafts=None), -1, "null pointer"),
    (dict(ua=None), -1, "null pointer"), (dict(us=None), -1, "null pointer"),
    (dict(k=-1), -1, "k = -1"), (dict(k=257), -1, "k = 257"), (dict(V=0), -1, "vocabulary 0"),
    (dict(dtype=7), -1, "dtype"), (dict(temp=0.0), -1, "temperature"),
    (dict(temp=float("inf")), -1, "temperature"), (dict(temp=float("nan")), -1, "temperature"),
    (dict(temp=-1.0), -1, "temperature"), (dict(keep=16), -1, "needs lens"),
    (dict(target=17), -1, "aligned"), (dict(draft=18, dtype=0), -1, "aligned"),
    (dict(ws=None), -1, "workspace"), (dict(ws=8), -1, "16-byte"), (dict(wsb=8), -2, "workspace"),
    (dict(B=1 << 24, k=128, V=1 << 20), -1, "too large"),
    (dict(B=1 << 20, k=0, V=2048 * 1024), -1, "too large"),
])
def test_sample_verify_refuses(change, rc, text):
    got, msg = call_sample(**change)
    assert got == rc and text in msg


def test_sample_workspace_sizes():
    ws = _lib.lib().kve_sample_workspace_bytes
    assert ws(0, 4, 1000, 1) == ws(1, -1, 1000, 1) == ws(1, 4, 0, 1) == ws(1, 4, 1000, 9) == 0
    # every row's chunks have a maximum and a sum
    assert ws(32, 4, 151936, 1) >= 32 * 9 * (151936 // 8192) * 12
    assert call_sample(B=0)[0] == 0


def test_wrappers_refuse_before_anything_runs():
    i32 = torch.zeros(2, 4, dtype=torch.int32)
    with pytest.raises(ValueError, match="on the GPU"):
        kernels.tree_masks(i32)
    with pytest.raises(ValueError, match="on the GPU"):
        kernels.tree_accept(i32, i32, i32)
    with pytest.raises(ValueError, match=r"\[B, k\+1, V\]"):
        kernels.sample_verify(torch.zeros(2, 1, 8), i32[:, :0], torch.zeros(2, 0), torch.zeros(2))
    with pytest.raises(ValueError, match="contiguous"):
        kernels.paged_tree_attn(torch.zeros(1, 2, 4, 64), *[None] * 6)


def test_forward_hidden_checks_the_trees_shape():
    from kvengine_amd.forward import forward_hidden

    ids = torch.zeros(2, 4, dtype=torch.long)
    tree = torch.zeros(2, 5, dtype=torch.int64), torch.zeros(2, 5, dtype=torch.int32)
    with pytest.raises(ValueError, match="tree masks"):
        forward_hidden(None, ids, None, None, 16, fused=False, tree=tree)


@pytest.mark.parametrize("T", [1e-46, 3.5e38, 1e300, 5e-324, -0.8])
def test_sample_verify_refuses_temperatures_past_the_floats(T):
    """(nothing is launched for them: the workspace is refused next)"""
    rc, msg = call_sample(temp=T, wsb=8)
    assert rc == -1 and "temperature" in msg
    assert call_sample(temp=1e-45, wsb=8)[0] == call_sample(temp=3.4e38, wsb=8)[0] == -2


def test_an_lds_refusal_names_the_trees_call():
    """Without a device (hidden from the child, so that nothing can be launched) the first
    thing an order of several row tiles asks for is refused."""
    code = """if True:
        from kvengine_amd import _lib
        args = dict(q=16, k=16, v=16, masks=16, tables=16, rows=None, start=16, q_lens=None, B=2,
                    T=16, Hq=16, Hkv=2, D=128, bs=16, max_blocks=16, num_rows=2, num_blocks=32,
                    max_ctx=128, unit=8, kw=2, scale=0.125, dtype=1, plan=16, out=16, ws=256,
                    wsb=1 << 30, layout=0)
        rc = _lib.lib().kve_paged_tree_attn(*args.values(), None)
        print(rc, _lib.lib().kve_last_error().decode())
    """
    env = dict(os.environ, HIP_VISIBLE_DEVICES="-1", ROCR_VISIBLE_DEVICES="-1")
    out = subprocess.run([sys.executable, "-c", code], env=env, capture_output=True, text=True,
                         cwd=os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
    assert out.returncode == 0, out.stderr
    assert "LDS refused" in out.stdout and "kve_paged_tree_attn" in out.stdout, out.stdout


def test_sample_workspace_holds_every_chunk():
    """A sum (8 bytes) and a maximum (4) per row and chunk of 2048 logits, and 64 bytes of the
    deciding position's sums per sequence and chunk, for 2k + 1 rows with a draft's logits."""
    ws = _lib.lib().kve_sample_workspace_bytes
    for B, k, V in ((32, 4, 151936), (1, 1, 2049), (3, 0, 50257), (2, 256, 4096)):
        chunks = -(-V // 2048)
        need = B * (2 * k + 1) * chunks * 12 + (B * chunks * 64 if k else 0)
        assert ws(B, k, V, 1) >= need and ws(B, k, V, 0) >= need
        rc, msg = call_sample(B=B, k=k, V=V, ts=(k + 1) * V, tp=V, ds=k * V, dp=V, wsb=need - 1)
        assert rc == -2 and "workspace" in msg
