"""The measured work of the tree and sampled verification operators.

A case is one pass of one of three kinds, as a serving program with tree drafts
or sampled decoding issues it on one GPU:

  tree    attention of a tree of drafted tokens over the paged cache: the
          trees' masks and one plan, then the launch of every layer
  accept  the walk of the trees by the target's picks, with the accepted
          paths' K/V moved to consecutive slots in every layer
  sample  verification of drafted tokens against the target's and the draft's
          probabilities from given uniform numbers (k = 0: one token a row)

`own` false computes the same in elementary torch operations.
"""

import math
import random

import torch

own = False

# (layers, query heads, kv heads, head dim) of the framework's two models
HEADS = {"0.5b": (24, 14, 2, 64), "3b": (36, 16, 2, 128)}
DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}
VOCAB = 151936
BS = 16  # tokens per block


def listed():
    return [
        # One live request with a small tree, the draft-sized model's heads:
        # the launches a single user waits for.
        {"name": "tree_1x8", "kind": "tree", "arch": "0.5b", "dtype": "bf16", "layers": 2,
         "seqs": 1, "nodes": 8, "ctx_lo": 603, "ctx_hi": 603, "unit": 0, "kw": 0, "spread": 1},
        # A full batch of the target with 16 nodes each over ragged histories.
        {"name": "tree_32x16", "kind": "tree", "arch": "3b", "dtype": "bf16", "layers": 2,
         "seqs": 32, "nodes": 16, "ctx_lo": 64, "ctx_hi": 4096, "unit": 0, "kw": 0, "spread": 2},
        # The same batch in the batched engine's fixed summation order, an odd
        # number of nodes.
        {"name": "tree_32x13_fixed", "kind": "tree", "arch": "3b", "dtype": "bf16", "layers": 2,
         "seqs": 32, "nodes": 13, "ctx_lo": 48, "ctx_hi": 860, "unit": 8, "kw": 2, "spread": 3},
        # The widest trees over long histories.
        {"name": "tree_16x64_long", "kind": "tree", "arch": "3b", "dtype": "bf16", "layers": 2,
         "seqs": 16, "nodes": 64, "ctx_lo": 7000, "ctx_hi": 8128, "unit": 16, "kw": 2, "spread": 4},
        # The parity configuration: fp32, a few requests.
        {"name": "tree_fp32", "kind": "tree", "arch": "0.5b", "dtype": "fp32", "layers": 2,
         "seqs": 4, "nodes": 11, "ctx_lo": 200, "ctx_hi": 1500, "unit": 0, "kw": 0, "spread": 5},
        # Accept of one request: a whole model's cache rows move by one launch.
        {"name": "accept_1x8", "kind": "accept", "arch": "0.5b", "dtype": "bf16", "seqs": 1,
         "nodes": 8, "ctx_lo": 40, "ctx_hi": 40, "spread": 26},
        # Accept of a full batch of the target's trees.
        {"name": "accept_32x16", "kind": "accept", "arch": "3b", "dtype": "bf16", "seqs": 32,
         "nodes": 16, "ctx_lo": 16, "ctx_hi": 120, "spread": 7},
        # Accept of wide trees in fp32.
        {"name": "accept_64x64_fp32", "kind": "accept", "arch": "0.5b", "dtype": "fp32", "seqs": 64,
         "nodes": 64, "ctx_lo": 16, "ctx_hi": 60, "spread": 8},
        # One sampled request, k = 4.
        {"name": "sample_1x4", "kind": "sample", "dtype": "bf16", "seqs": 1, "k": 4,
         "vocab": VOCAB, "draft": True, "temperature": 0.8},
        # A full batch of sampled requests in the models' type.
        {"name": "sample_32x4", "kind": "sample", "dtype": "bf16", "seqs": 32, "k": 4,
         "vocab": VOCAB, "draft": True, "temperature": 1.0},
        # fp32 logits, eight drafts each: the largest call.
        {"name": "sample_32x8_fp32", "kind": "sample", "dtype": "fp32", "seqs": 32, "k": 8,
         "vocab": VOCAB, "draft": True, "temperature": 0.7},
        # A token for every node of eight trees (no drafts: the walk follows),
        # from a vocabulary whose rows are not 16-byte aligned.
        {"name": "sample_rows_104", "kind": "sample", "dtype": "bf16", "seqs": 104, "k": 0,
         "vocab": 50257, "draft": False, "temperature": 1.0},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["tree", "tree", "accept", "sample", "sample"])
    arch = rng.choice(["0.5b", "3b"])
    dtype = rng.choice(["bf16", "bf16", "bf16", "fp32"])
    spread = rng.randrange(100000)
    if kind == "tree":
        nodes = _log_int(rng, 1, 64)
        hi = _log_int(rng, 16, 8128)
        fixed = rng.random() < 0.5
        # at most the longest listed case's keys times nodes
        seqs = _log_int(rng, 1, max(1, min(64, 100000 // hi, 1 + 4000000 // (hi * nodes))))
        return {"kind": "tree", "arch": arch, "dtype": dtype, "layers": 2, "seqs": seqs,
                "nodes": nodes, "ctx_lo": max(1, hi // rng.choice([1, 4, 16])), "ctx_hi": hi,
                "unit": (16 if hi > 4096 else 8) if fixed else 0, "kw": 2 if fixed else 0,
                "spread": spread}
    if kind == "accept":
        hi = _log_int(rng, 1, 100)
        return {"kind": "accept", "arch": arch, "dtype": dtype, "seqs": _log_int(rng, 1, 40),
                "nodes": _log_int(rng, 1, 64), "ctx_lo": max(1, hi // 4), "ctx_hi": hi,
                "spread": spread}
    k = rng.choice([0, 1, 2, 3, 4, 5, 7, 8])
    vocab = rng.choice([VOCAB, _log_int(rng, 1000, 160000), 8 * _log_int(rng, 100, 19000)])
    rows = 32 * 9 * VOCAB // (vocab * (k + 1))
    return {"kind": "sample", "dtype": dtype, "seqs": _log_int(rng, 1, max(1, min(256, rows))),
            "k": k, "vocab": vocab, "draft": k > 0 and rng.random() < 0.7,
            "temperature": round(rng.uniform(0.3, 1.5), 2)}


# ---- inputs -------------------------------------------------------------------

def _trees(case):
    """Each sequence's committed length and its tree: parents[0] = -1 (the last
    emitted token), parents[i] < i; about half the nodes continue the one before
    them, the others branch anywhere."""
    r = random.Random(case["spread"])
    starts = [_log_int(r, case["ctx_lo"], case["ctx_hi"]) for _ in range(case["seqs"])]
    trees = [[-1] + [i - 1 if r.random() < 0.5 else r.randrange(i) for i in range(1, case["nodes"])]
             for _ in range(case["seqs"])]
    return starts, trees


def _walks(case):
    """Per sequence the nodes that the target's picks will follow, root first:
    the way to a node anywhere in the tree."""
    r = random.Random(case["spread"] + 1)
    out = []
    for parents in _trees(case)[1]:
        i, way = r.randrange(len(parents)), []
        while i >= 0:
            way.append(i)
            i = parents[i]
        out.append(way[::-1])
    return out


def _tables(starts, nodes, seed):
    """Block tables over a shuffled pool with a quarter to spare."""
    need = [-(-(n + nodes) // BS) for n in starts]
    nb = sum(need) + sum(need) // 4 + 1
    ids = list(range(nb))
    random.Random(seed).shuffle(ids)
    t = torch.full((len(need), max(need)), -1, dtype=torch.int32)
    at = 0
    for i, n in enumerate(need):
        t[i, :n] = torch.tensor(ids[at:at + n], dtype=torch.int32)
        at += n
    return t.cuda(), nb


def _inputs(case, seed):
    """Everything a pass reads, from the case and the seed alone."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype = DTYPES[case["dtype"]]

    def normal(*shape):
        return torch.randn(shape, generator=g, device="cuda")

    if case["kind"] == "sample":
        B, k, V, T = case["seqs"], case["k"], case["vocab"], case["temperature"]
        # logits of spread 3, the draft's close to the target's
        x = {"target": (3.0 * normal(B, k + 1, V)).to(dtype), "draft": None, "temperature": T}
        draft = (x["target"][:, :k] + 0.7 * normal(B, k, V)).to(dtype)
        u = torch.rand(B, k, V, generator=g, device="cuda").clamp_min_(1e-30)
        gumbel = -torch.log(-torch.log(u).clamp_min_(1e-30))
        noisy = draft.float() / T + (gumbel if case["draft"] else 0.0)
        x["drafts"] = (noisy.argmax(-1) if k else torch.zeros(B, 0, device="cuda")).to(torch.int32)
        if case["draft"]:
            x["draft"] = draft
        x["u_accept"] = torch.rand(B, k, generator=g, device="cuda")
        x["u_sample"] = torch.rand(B, generator=g, device="cuda")
        return x
    starts, trees = _trees(case)
    L, Hq, Hkv, D = HEADS[case["arch"]]
    L = case.get("layers", L)
    tables, nb = _tables(starts, case["nodes"], seed)
    x = {"parents": torch.tensor(trees, dtype=torch.int32, device="cuda"), "tables": tables,
         "k": normal(L, nb, Hkv, BS, D).to(dtype), "v": normal(L, nb, Hkv, D, BS).to(dtype)}
    start = torch.tensor(starts, dtype=torch.int32, device="cuda")
    if case["kind"] == "tree":
        x.update(start=start, max_ctx=max(starts) + case["nodes"], order=(case["unit"], case["kw"]),
                 q=normal(L, case["seqs"], case["nodes"], Hq, D).to(dtype))
        return x
    shape = (case["seqs"], case["nodes"])
    tokens = torch.randint(0, VOCAB, shape, generator=g, device="cuda", dtype=torch.int32)
    preds = torch.randint(0, VOCAB, shape, generator=g, device="cuda", dtype=torch.int32)
    walks = _walks(case)
    at = torch.tensor([(b, i, j) for b, w in enumerate(walks) for i, j in zip(w, w[1:])],
                      device="cuda").view(-1, 3)
    preds[at[:, 0], at[:, 1]] = tokens[at[:, 0], at[:, 2]]
    # the cache holds the tree: lengths after the pass's commit
    x.update(tokens=tokens, preds=preds, lens=start + case["nodes"])
    return x


def prepare(case, seed):
    return {"kind": case["kind"], **_inputs(case, seed)}


# ---- the passes ---------------------------------------------------------------

def run(s):
    if own:
        return {"tree": _own_tree, "accept": _own_accept, "sample": _own_sample}[s["kind"]](s)
    return {"tree": _plain_tree, "accept": _plain_accept, "sample": _plain_sample}[s["kind"]](s)


def _own_tree(s):
    from kvengine_amd import kernels

    q, k, v, tables, start, ctx = s["q"], s["k"], s["v"], s["tables"], s["start"], s["max_ctx"]
    L, B, n, Hq, D = q.shape
    unit, kw = s["order"]
    masks, depths = kernels.tree_masks(s["parents"])
    plan = kernels.attn_plan(tables, start, B, n, Hq, k.shape[2], D, BS, k.shape[1], ctx, q.dtype,
                             unit_blocks=unit, key_waves=kw)
    out = [kernels.paged_tree_attn(q[i], k[i], v[i], tables, start, ctx, masks, unit_blocks=unit,
                                   key_waves=kw, plan=plan) for i in range(L)]
    return {"masks": masks, "depths": depths, "out": out}


def _own_accept(s):
    from kvengine_amd import kernels
    from kvengine_amd.paged import DeviceKV

    kv = DeviceKV(s["k"], s["v"], s["tables"], s["lens"], BS)
    n_acc, emitted, path, keep = kernels.tree_accept(s["tokens"], s["parents"], s["preds"], kv=kv)
    return {"n_acc": n_acc, "emitted": emitted, "path": path, "keep": keep, "k": s["k"], "v": s["v"]}


def _own_sample(s):
    from kvengine_amd import kernels

    n_acc, emitted, _ = kernels.sample_verify(s["target"], s["drafts"], s["u_accept"],
                                              s["u_sample"], draft_logits=s["draft"],
                                              temperature=s["temperature"])
    return {"n_acc": n_acc, "emitted": emitted}


def _ancestors(parents):
    """[B, n, n] bool: node j is node i or above it. With P the parent relation,
    the closure of I + P, squared until paths of 64 steps are covered."""
    n = parents.shape[1]
    node = torch.arange(n, device=parents.device)
    a = ((parents[:, :, None] == node) | torch.eye(n, dtype=torch.bool, device=parents.device)).float()
    for _ in range(6):
        a = ((a @ a) > 0).float()
    return a > 0


def _plain_tree(s):
    q, k, v, start = s["q"], s["k"], s["v"], s["start"].long()
    L, B, n, Hq, D = q.shape
    Hkv = k.shape[2]
    anc = _ancestors(s["parents"])
    node = torch.arange(n, device=q.device)
    masks = torch.where(anc, torch.ones_like(node) << node, 0).sum(-1)
    depths = (anc.sum(-1) - 1).to(torch.int32)
    blocks = s["tables"].long().clamp_min(0)
    C = blocks.shape[1] * BS
    # the histories gathered from their blocks: [L, B, Hkv, C, D]
    kg = k[:, blocks].float().permute(0, 1, 3, 2, 4, 5).reshape(L, B, Hkv, C, D)
    vg = v[:, blocks].float().permute(0, 1, 3, 2, 5, 4).reshape(L, B, Hkv, C, D)
    rel = torch.arange(C, device=q.device) - start[:, None]  # [B, C]
    inside = (rel >= 0) & (rel < n)
    seen = anc.gather(2, rel.clamp(0, n - 1)[:, None].expand(B, n, C)) & inside[:, None]
    seen |= (rel < 0)[:, None]  # [B, n, C]
    qg = q.float().view(L, B, n, Hkv, Hq // Hkv, D).permute(0, 1, 3, 4, 2, 5)
    scores = qg.reshape(L, B, Hkv, -1, D) @ kg.transpose(-1, -2).contiguous() * D ** -0.5
    scores = scores.view(L, B, Hkv, -1, n, C).masked_fill(~seen[None, :, None, None], -math.inf)
    p = torch.exp(scores - scores.amax(-1, keepdim=True))
    p = p / p.sum(-1, keepdim=True)
    out = (p.view(L, B, Hkv, -1, C) @ vg).view(L, B, Hkv, -1, n, D).permute(0, 1, 4, 2, 3, 5)
    out = out.reshape(L, B, n, Hq, D).to(q.dtype)
    return {"masks": masks, "depths": depths, "out": list(out.unbind(0))}


def _plain_accept(s):
    tokens, parents, preds = s["tokens"], s["parents"].long(), s["preds"]
    B, n = tokens.shape
    node = torch.arange(n, device=tokens.device)
    anc = _ancestors(s["parents"])
    match = (tokens == preds.gather(1, parents.clamp_min(0))) & (parents >= 0)
    # of equal tokens under one parent the lowest node is the child that counts
    twin = (parents[:, :, None] == parents[:, None]) & (tokens[:, :, None] == tokens[:, None])
    match &= ~(twin & (node[:, None] > node)).any(-1)
    match |= node == 0
    taken = (match[:, None] | ~anc).all(-1)  # a node is accepted with all above it
    n_acc = (taken.sum(-1) - 1).to(torch.int32)
    path = torch.where(taken, node, n).sort(-1).values
    there = path < n
    last = torch.where(taken, node, 0).amax(-1, keepdim=True)
    shifted = torch.cat([path[:, 1:], torch.full_like(path[:, :1], n)], 1)
    emitted = torch.where(shifted < n, tokens.gather(1, shifted.clamp_max(n - 1)),
                          torch.where(node == n_acc[:, None], preds.gather(1, last), -1))
    path = torch.where(there, path, -1)
    start = s["lens"].long() - n
    keep = (start + 1 + n_acc).to(torch.int32)
    # rows of the accepted nodes, all read before any is written
    b, j = there.nonzero(as_tuple=True)
    src, dst = start[b] + path[b, j], start[b] + j
    sb, db = (s["tables"][b, x // BS].long() for x in (src, dst))
    k, v = s["k"], s["v"]
    k[:, db, :, dst % BS] = k[:, sb, :, src % BS]
    v[:, db, :, :, dst % BS] = v[:, sb, :, :, src % BS]
    return {"n_acc": n_acc, "emitted": emitted.to(torch.int32), "path": path.to(torch.int32),
            "keep": keep, "k": k, "v": v}


def _plain_sample(s):
    # 64 bits: a token is a place among up to 160000 running sums
    target, drafts, T = s["target"].double(), s["drafts"].long(), s["temperature"]
    B, k = drafts.shape
    e = torch.exp((target - target.amax(-1, keepdim=True)) / T)
    p = e / e.sum(-1, keepdim=True)
    at = drafts[..., None]
    if s["draft"] is not None:
        d = s["draft"].double()
        d = torch.exp((d - d.amax(-1, keepdim=True)) / T)
        q = d / d.sum(-1, keepdim=True)
    else:
        q = torch.zeros_like(p[:, :k]).scatter_(2, at, 1.0)
    ok = s["u_accept"].double() * q.gather(2, at)[..., 0] < p[:, :k].gather(2, at)[..., 0]
    n_acc = ok.long().cumprod(1).sum(1)
    pick = n_acc[:, None, None].expand(B, 1, p.shape[-1])
    q = torch.cat([q, torch.zeros_like(p[:, :1])], 1).gather(1, pick)[:, 0]
    rest = (p.gather(1, pick)[:, 0] - q).clamp_min(0.0)
    if s["draft"] is None:  # the rejected token leaves the others as they are
        rest = torch.where(q > 0, 0.0, e.gather(1, pick)[:, 0])
    run_sum = rest.cumsum(-1)
    token = (run_sum <= s["u_sample"].double()[:, None] * run_sum[:, -1:]).sum(-1)
    j = torch.arange(k + 1, device=drafts.device)
    padded = torch.cat([drafts, token[:, None]], 1)
    emitted = torch.where(j < n_acc[:, None], padded, torch.where(j == n_acc[:, None], token[:, None], -1))
    return {"n_acc": n_acc.to(torch.int32), "emitted": emitted.to(torch.int32)}


# ---- what a pass cannot do without ----------------------------------------------

def work(case):
    e = 4 if case["dtype"] == "fp32" else 2
    if case["kind"] == "sample":
        rows = case["seqs"] * (2 * case["k"] + 1 if case["draft"] else case["k"] + 1)
        # each logit read once; a subtraction, an exponential and an addition of it
        return {"bytes": rows * case["vocab"] * e, "flops": 3 * rows * case["vocab"]}
    L, Hq, Hkv, D = HEADS[case["arch"]]
    starts, trees = _trees(case)
    n = case["nodes"]
    if case["kind"] == "tree":
        keys = sum(starts) + n * len(starts)
        pairs = n * sum(starts) + sum(_depth_sum(p) for p in trees)
        return {"bytes": case["layers"] * (keys * Hkv * D * 2 + 2 * len(starts) * n * Hq * D) * e,
                "flops": case["layers"] * 4 * Hq * D * pairs}
    moved = sum(i != j for w in _walks(case) for j, i in enumerate(w))
    return {"bytes": moved * L * Hkv * D * 2 * e * 2 + 20 * n * len(starts), "flops": 0}


def _depth_sum(parents):
    """Nodes that a tree's nodes see in it, themselves included."""
    seen = []
    for p in parents:
        seen.append(1 + (seen[p] if p >= 0 else 0))
    return sum(seen)


# ---- the same in 64 bits, from the definition -----------------------------------

def exact(case, seed):
    x = _inputs(case, seed)
    if case["kind"] == "sample":
        return _exact_sample(x)
    if case["kind"] == "accept":
        return _exact_accept(case, x)
    starts, trees = _trees(case)
    n, (_, Hq, Hkv, D) = case["nodes"], HEADS[case["arch"]]
    ways = []
    for parents in trees:
        w = []
        for i, p in enumerate(parents):
            w.append(([] if p < 0 else w[p]) + [i])
        ways.append(w)
    masks = [[sum(1 << j for j in w) for w in ws] for ws in ways]
    masks = [[m - (1 << 64) if m >> 63 else m for m in row] for row in masks]
    out = torch.zeros(x["q"].shape, dtype=torch.float64, device="cuda")
    for b, (start, ws) in enumerate(zip(starts, ways)):
        hide = torch.zeros(n, start + n, dtype=torch.bool)
        hide[:, start:] = True
        for t, w in enumerate(ws):
            hide[t, [start + j for j in w]] = False
        hide = hide.cuda()
        ids = x["tables"][b, :-(-(start + n) // BS)].long()
        for i in range(case["layers"]):
            k = x["k"][i][ids].permute(1, 0, 2, 3).flatten(1, 2)[:, :start + n].double()
            v = x["v"][i][ids].permute(1, 0, 3, 2).flatten(1, 2)[:, :start + n].double()
            for h in range(Hq):
                kh, vh = k[h // (Hq // Hkv)], v[h // (Hq // Hkv)]
                z = x["q"][i, b, :, h].double() @ kh.t().contiguous() / math.sqrt(D)
                out[i, b, :, h] = torch.softmax(z.masked_fill(hide, -math.inf), -1) @ vh
    return {"masks": torch.tensor(masks), "out": list(out.unbind(0)),
            "depths": torch.tensor([[len(w) - 1 for w in ws] for ws in ways], dtype=torch.int32)}


def _exact_accept(case, x):
    n = case["nodes"]
    tokens, preds, parents = (x[t].tolist() for t in ("tokens", "preds", "parents"))
    lens, tables = x["lens"].tolist(), x["tables"].tolist()
    k, v = x["k"].clone(), x["v"].clone()
    n_acc, emitted, paths, keep = [], [], [], []
    for b in range(case["seqs"]):
        way, new = [0], []
        while True:
            want = preds[b][way[-1]]
            new.append(want)
            kids = [c for c in range(n) if parents[b][c] == way[-1] and tokens[b][c] == want]
            if not kids:
                break
            way.append(kids[0])
        n_acc.append(len(way) - 1)
        emitted.append(new + [-1] * (n - len(new)))
        paths.append(way + [-1] * (n - len(way)))
        start = lens[b] - n
        keep.append(start + len(way))
        for j, c in enumerate(way):
            (sb, so), (db, do) = ((tables[b][p // BS], p % BS) for p in (start + c, start + j))
            k[:, db, :, do] = x["k"][:, sb, :, so]
            v[:, db, :, :, do] = x["v"][:, sb, :, :, so]

    def ints(t):
        return torch.tensor(t, dtype=torch.int32)

    return {"n_acc": ints(n_acc), "emitted": ints(emitted), "path": ints(paths), "keep": ints(keep),
            "k": k, "v": v}


def _exact_sample(x):
    T = x["temperature"]
    B, k = x["drafts"].shape
    drafts, u, us = x["drafts"].tolist(), x["u_accept"].tolist(), x["u_sample"].tolist()

    def weights(logits):
        z = logits.double() / T
        return torch.exp(z - z.max())

    n_acc, emitted = [], []
    for b in range(B):
        new = []
        for j in range(k + 1):
            w = weights(x["target"][b, j])
            p = w / w.sum()
            if j == k:
                break
            c = drafts[b][j]
            if x["draft"] is None:
                if u[b][j] < float(p[c]):
                    new.append(c)
                    continue
                w[c] = 0.0
            else:
                q = weights(x["draft"][b, j])
                q = q / q.sum()
                if u[b][j] * float(q[c]) < float(p[c]):
                    new.append(c)
                    continue
                w = (p - q).clamp(min=0.0)
            break
        n_acc.append(len(new))
        c = torch.cumsum(w, 0)
        new.append(int(torch.searchsorted(c, us[b] * c[-1:], right=True)))
        emitted.append(new + [-1] * (k + 1 - len(new)))
    return {"n_acc": torch.tensor(n_acc, dtype=torch.int32),
            "emitted": torch.tensor(emitted, dtype=torch.int32)}
