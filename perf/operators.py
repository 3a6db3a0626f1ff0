"""Cases of the KV-cache operators: attention of drafted token trees over a paged cache, acceptance of a drafted
path, attention weights accumulated per cached row, and eviction by them.

The cache is the batch engine's: bf16 pages of 16 rows, [layer][page][K | V][16][kv_heads][hdim], behind a page table
[slot][page].  Slot s holds rows 0 .. lens[s] - 1; its drafted nodes are tokens offsets[s] .. offsets[s + 1] - 1, and
node i of a slot has its K and V in row lens[s] + i.  parent[t] is the node's parent within its tree (-1: none, -2: a
padding node, which sees nothing).

  tree     q of every node over the cached rows, its ancestors and itself -> attention output, log-sum-exp
  commit   the longest path from node 0 whose every token is the one chosen after its parent; its rows move up to
           follow the cache in every layer
  weights  probabilities of the accepted queries, summed per layer, KV head and row into the accumulated weights
  evict    the first `sinks` and last `recent` rows and the heaviest of the others, `budget` in all, per layer and KV
           head, copied in order into another cache
"""
import math
import random

import numpy as np
import torch

own = False  # True: the framework's operators; False: their plain form

PAGE = 16
DEV = "cuda"


# ---------------------------------------------------------------- cases

def listed():
    return [
        # one sequence of the 32-layer model at a short context: a plain decode step, all latency
        dict(name="tree_decode_short", op="tree", slots=1, rows=55, nodes=1, kv_heads=4, group=4, hd=128, type="f32", ragged=0, pad=0),
        # the same model at a 4096-row context with a small drafted tree
        dict(name="tree_one_4k", op="tree", slots=1, rows=4096, nodes=16, kv_heads=4, group=4, hd=128, type="f32", ragged=0, pad=0),
        # the server's 256 slots of up to 192 rows, a few drafted tokens each
        dict(name="tree_serve_256", op="tree", slots=256, rows=176, nodes=5, kv_heads=4, group=4, hd=128, type="f32", ragged=60, pad=0),
        # medium batch, trees of 30 nodes, lengths far apart
        dict(name="tree_batch_32", op="tree", slots=32, rows=3001, nodes=30, kv_heads=4, group=4, hd=128, type="f32", ragged=90, pad=0),
        # long contexts with the widest trees, bf16 queries
        dict(name="tree_long_wide", op="tree", slots=12, rows=16500, nodes=64, kv_heads=4, group=4, hd=128, type="bf16", ragged=30, pad=0),
        # narrow heads, wide groups, odd sizes, padded trees
        dict(name="tree_odd_hd64", op="tree", slots=7, rows=1237, nodes=13, kv_heads=3, group=8, hd=64, type="bf16", ragged=95, pad=3),
        # one sequence's step: 32 layers, a path of a few nodes
        dict(name="commit_one", op="commit", slots=1, rows=4096, nodes=25, kv_heads=4, hd=128, layers=32, ragged=0),
        # every slot of a serving batch
        dict(name="commit_batch", op="commit", slots=128, rows=170, nodes=22, kv_heads=4, hd=128, layers=32, ragged=60),
        # a step's three accepted tokens over all 32 layers
        dict(name="weights_one_4k", op="weights", slots=1, rows=4096, nodes=3, kv_heads=4, group=4, hd=128, layers=32, type="f32", ragged=0),
        # the last 31 prompt tokens of a batch of prompts, four layers
        dict(name="weights_window", op="weights", slots=16, rows=6007, nodes=31, kv_heads=4, group=4, hd=128, layers=4, type="bf16", ragged=50),
        # one sequence over its bound: 32 layers
        dict(name="evict_one_4k", op="evict", slots=1, rows=4096, budget=1024, sinks=4, recent=256, kv_heads=4, hd=128, layers=32, ragged=0),
        # a batch of long prompts cut to a quarter, some of them short enough to stay whole
        dict(name="evict_batch", op="evict", slots=24, rows=6100, budget=1500, sinks=8, recent=333, kv_heads=4, hd=128, layers=8, ragged=85),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng: random.Random):
    op = rng.choice(["tree", "tree", "tree", "commit", "weights", "evict"])
    hd, kvh = rng.choice([64, 128, 128]), rng.choice([1, 2, 3, 4, 4, 8])
    c = dict(op=op, slots=_log(rng, 1, 256), rows=_log(rng, 1, 16000), kv_heads=kvh, hd=hd, ragged=rng.randrange(0, 96))
    width = kvh * hd / 512.0
    if op == "tree":
        c.update(nodes=_log(rng, 1, 64), group=rng.choice([1, 2, 4, 4, 8]), type=rng.choice(["f32", "bf16"]))
        c["pad"] = rng.randrange(0, c["nodes"]) if rng.random() < 0.3 else 0
        most = min(150000 / width, 12 * 16500 * 64 * 16 / (kvh * c["group"] * c["nodes"]))
    elif op == "commit":
        c.update(nodes=_log(rng, 2, 64), layers=_log(rng, 1, 32))
        most = 700000 / width / c["layers"]
    elif op == "weights":
        c.update(nodes=_log(rng, 1, 64), group=rng.choice([1, 2, 4, 4, 8]), layers=_log(rng, 1, 32), type=rng.choice(["f32", "bf16"]))
        most = min(300000 / width / c["layers"], 16 * 6007 * 4 * 31 * 16 / (c["layers"] * c["nodes"] * kvh * c["group"]))
    else:
        c.update(layers=_log(rng, 1, 32))
        c["budget"] = _log(rng, max(1, c["rows"] // 16), max(2, int(c["rows"] * 1.1)))
        c["sinks"] = rng.randrange(0, min(9, c["budget"] + 1))
        c["recent"] = rng.randrange(0, (c["budget"] - c["sinks"]) // 2 + 1)
        most = 900000 / width / c["layers"]
    c["rows"] = max(1, min(c["rows"], int(most)))
    c["slots"] = max(1, min(c["slots"], int(most / c["rows"])))
    if op == "evict":
        c["budget"] = max(c["sinks"] + c["recent"], min(c["budget"], 2 * c["rows"]), 1)
    return c


# ---------------------------------------------------------------- what follows from the case alone

def _lens(c):
    """Cached rows of each slot: spread over ragged % of `rows` below it."""
    s = np.arange(c["slots"], dtype=np.int64)
    return c["rows"] - (c["rows"] * c["ragged"] // 100) * ((s * 7919 + 13) % 101) // 100


def _counts(c):
    """Nodes of each slot: `nodes` for the first, one to three fewer for some others."""
    s = np.arange(c["slots"], dtype=np.int64)
    return np.maximum(1, c["nodes"] - (s * 5 % 4))


def _trees(c):
    """(offsets, parents, paths): trees where a node hangs from one of the eight before it; a path down each."""
    counts = _counts(c)
    rng = np.random.default_rng([c["slots"], c["nodes"], c["rows"]])
    parents, paths = [], []
    for n in counts.tolist():
        back = rng.integers(1, 9, n)
        par = np.maximum(np.arange(n) - back, 0)
        par[0] = -1
        path, u = [0], rng.random(n)
        for i in range(1, n):
            if par[i] == path[-1] and u[i] < 0.4:
                path.append(i)
        parents.append(par)
        paths.append(path)
    off = np.concatenate([[0], np.cumsum(counts)])
    return off, parents, paths


def work(case):
    c = case
    lens = _lens(c)
    cnt = _counts(c) if "nodes" in c else None
    row = c["kv_heads"] * c["hd"]  # elements of one K or V row
    qb = 2 if c.get("type") == "bf16" else 4
    if c["op"] == "tree":
        nt, heads = int(cnt.sum()), c["kv_heads"] * c["group"]
        live = int((lens + np.maximum(cnt - c["pad"], 0)).sum())
        pairs = int((lens * np.maximum(cnt - c["pad"], 0)).sum())
        return dict(bytes=live * row * 4 + nt * heads * (c["hd"] * 2 * qb + 4) + nt * 4, flops=4.0 * pairs * heads * c["hd"])
    if c["op"] == "commit":
        _, _, paths = _trees(c)
        moved = sum(sum(1 for j, p in enumerate(x) if p != j) for x in paths)
        return dict(bytes=moved * row * 2 * 2 * 2 * c["layers"] + int(cnt.sum()) * 12, flops=0)
    if c["op"] == "weights":
        heads = c["kv_heads"] * c["group"]
        rows, pairs = int((lens + cnt).sum()), int(((lens + cnt) * cnt).sum())
        return dict(bytes=c["layers"] * (rows * row * 2 + int(cnt.sum()) * heads * (c["hd"] * qb + 4) + int(lens.sum() * 2 + cnt.sum()) * c["kv_heads"] * 4),
                    flops=2.0 * c["layers"] * pairs * heads * c["hd"])
    kept = np.minimum(lens, c["budget"])
    return dict(bytes=c["layers"] * c["kv_heads"] * (int(lens.sum()) * 4 + int(kept.sum()) * (c["hd"] * 8 + 8)), flops=0)


# ---------------------------------------------------------------- inputs

def _pool(c, g, layers, page_max):
    """Random pages for every slot, a few spare ones, in an order of their own; every row filled."""
    slots = c["slots"]
    npages = slots * page_max + 3
    kv = torch.empty((layers, npages, 2, PAGE, c["kv_heads"], c["hd"]), dtype=torch.bfloat16, device=DEV)
    for l in range(layers):
        kv[l] = torch.randn(kv[l].shape, generator=g, device=DEV, dtype=torch.float32).to(torch.bfloat16)
    perm = torch.randperm(npages, generator=g, device=DEV)[:slots * page_max]
    return kv, perm.to(torch.int32).view(slots, page_max).contiguous()


def _dev(a, dtype=torch.int32):
    return torch.as_tensor(np.ascontiguousarray(a), device=DEV).to(dtype)


def prepare(case, seed):
    c = dict(case)
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    s = dict(case=c)
    lens, layers = _lens(c), c.get("layers", 1)
    dt = torch.bfloat16 if c.get("type") == "bf16" else torch.float32
    s["lens"] = _dev(lens)
    if c["op"] == "evict":
        page_max = -(-int(lens.max()) // PAGE)
        s["kv"], s["pages"] = _pool(c, g, layers, page_max)
        # accumulated weights: heavy first rows, a long tail, exact zeros among them
        shape = (layers, c["slots"], c["kv_heads"], page_max * PAGE)
        acc = torch.exp(2.0 * torch.randn(shape, generator=g, device=DEV))
        acc[..., :2] *= 50.0
        s["acc"] = torch.where(torch.rand(shape, generator=g, device=DEV) < 0.05, torch.zeros_like(acc), acc)
        dmax = -(-c["budget"] // PAGE)
        n = c["slots"] * dmax + 2
        s["dst"] = torch.zeros((layers, n, 2, PAGE, c["kv_heads"], c["hd"]), dtype=torch.bfloat16, device=DEV)
        s["dst_pages"] = torch.randperm(n, generator=g, device=DEV)[:c["slots"] * dmax].to(torch.int32).view(c["slots"], dmax).contiguous()
        return s
    off, parents, paths = _trees(c)
    nt, cnt = int(off[-1]), np.diff(off)
    page_max = -(-int((lens + cnt).max()) // PAGE)
    s["kv"], s["pages"] = _pool(c, g, layers, page_max)
    s["offsets"] = _dev(off)
    if c["op"] == "weights":
        # the queries and their log-sum-exp as the attention left them (here of rows of about these lengths)
        heads = c["kv_heads"] * c["group"]
        s["q"] = torch.randn((layers, nt, heads, c["hd"]), generator=g, device=DEV).to(dt)
        at = np.repeat(lens, cnt) + np.arange(nt) - np.repeat(off[:-1], cnt) + 1
        s["lse"] = torch.log(torch.as_tensor(at, device=DEV).float())[None, :, None] + 0.5 + 0.1 * torch.randn((layers, nt, heads), generator=g, device=DEV)
        s["n_query"] = _dev(cnt)
        s["sel"] = _dev(np.minimum(off[:-1, None] + np.arange(c["nodes"])[None], nt - 1))
        s["acc"] = torch.rand((layers, c["slots"], c["kv_heads"], page_max * PAGE), generator=g, device=DEV) * 4.0
        return s
    par = np.concatenate(parents)
    if c["op"] == "commit":
        vocab = 120818
        tok = torch.randint(0, vocab, (nt,), generator=g, device=DEV)
        nxt = torch.randint(0, vocab, (nt,), generator=g, device=DEV)
        # the model agrees with the draft along the path
        a = np.concatenate([off[k] + np.asarray(p[:-1], dtype=np.int64) for k, p in enumerate(paths)])
        b = np.concatenate([off[k] + np.asarray(p[1:], dtype=np.int64) for k, p in enumerate(paths)])
        nxt[_dev(a, torch.int64)] = tok[_dev(b, torch.int64)]
        s["parent"], s["tokens"], s["next"] = _dev(par), tok.to(torch.int32), nxt.to(torch.int32)
        return s
    node = np.arange(nt) - np.repeat(off[:-1], cnt)
    par = np.where(node >= np.repeat(cnt, cnt) - c["pad"], -2, par)  # the tail of a padded tree
    s["parent"] = _dev(par)
    # q as the fused q | k | v projection leaves it: rows of a wider buffer
    heads = c["kv_heads"] * c["group"]
    wide = torch.randn((nt, (heads + 2 * c["kv_heads"]) * c["hd"]), generator=g, device=DEV).to(dt)
    s["q"] = wide[:, :heads * c["hd"]].view(nt, heads, c["hd"])
    return s


# ---------------------------------------------------------------- the operators

def run(state):
    return _own(state) if own else _PLAIN[state["case"]["op"]](state)


def _own(s):
    from hymt2_b200.kvcache import PagedKV
    c = s["case"]
    if "handle" not in s:  # a program keeps its caches' handles
        s["handle"] = PagedKV(s["kv"], s["pages"])
        s["dst_handle"] = PagedKV(s["dst"], s["dst_pages"]) if c["op"] == "evict" else None
    kv = s["handle"]
    if c["op"] == "tree":
        out, lse = kv.tree_attention(s["q"], s["lens"], s["offsets"], s["parent"], c["nodes"])
        return dict(out=out, lse=lse)
    if c["op"] == "commit":
        lens, n, path, bonus = kv.tree_commit(s["lens"], s["offsets"], s["parent"], s["tokens"], s["next"], c["nodes"])
        return dict(kv=s["kv"], lens=lens, accepted=n, path=path, bonus=bonus)
    if c["op"] == "weights":
        kv.add_weights(s["acc"], s["q"], s["lse"], s["lens"], s["n_query"], s["sel"])
        return dict(acc=s["acc"])
    lens, kept, acc = kv.evict(s["dst_handle"], s["lens"], s["acc"], c["budget"], c["sinks"], c["recent"])
    return dict(kv=s["dst"], lens=lens, kept=kept, acc=acc)


# ---------------------------------------------------------------- plain forms

def _rows(s, n):
    """K and V of rows 0 .. n - 1 of every slot, [L][slots][n][kv_heads][hd] in 32 bits."""
    r = torch.arange(n, device=DEV)
    page = s["pages"].long()[:, r >> 4]  # [slots][n]
    kv = s["kv"][:, page, :, (r & 15)[None].expand_as(page)].permute(2, 0, 1, 3, 4, 5)  # [L][slots][n][2][kv_heads][hd]
    return kv[:, :, :, 0].float(), kv[:, :, :, 1].float()


def _reach(link, n):
    """link[s][i]: the node above i, or a negative number.  [s][i][j]: j is i or reached from i."""
    step = (link[:, :, None] == torch.arange(n, device=DEV)) | torch.eye(n, device=DEV, dtype=torch.bool)
    return torch.linalg.matrix_power(step.float(), 64) > 0


def _nodes(s, n):
    """Token of node i of each slot [slots][n] (0 past its tree) and whether it is one."""
    off = s["offsets"].long()
    i = torch.arange(n, device=DEV)
    ok = i[None] < (off[1:] - off[:-1])[:, None]
    return torch.where(ok, off[:-1, None] + i[None], torch.zeros_like(off[:-1, None])), ok


def _plain_tree(s):
    c = s["case"]
    n, H, G, hd = c["nodes"], c["kv_heads"], c["group"], c["hd"]
    R = s["pages"].shape[1] * PAGE
    t, ok = _nodes(s, n)
    par = torch.where(ok, s["parent"].long()[t], torch.full_like(t, -2))
    lens = s["lens"].long()
    k, v = _rows(s, R)
    q = s["q"].float()[t].view(-1, n, H, G, hd)
    sc = torch.einsum("snhgd,srhd->shgnr", q, k[0]) * (1.0 / math.sqrt(hd))
    r = torch.arange(R, device=DEV)[None] - lens[:, None]  # the row's node, negative for cached rows
    node = torch.gather(_reach(par, n), 2, r.clamp(0, n - 1)[:, None].expand(-1, n, -1))
    see = ((r < 0)[:, None] | (node & (r >= 0)[:, None] & (r < n)[:, None])) & (par != -2)[:, :, None]
    sc = torch.where(see[:, None, None], sc, torch.full_like(sc[:1, :1, :1, :1, :1], -math.inf))
    m = sc.amax(-1, keepdim=True)
    p = torch.exp(sc - torch.where(torch.isinf(m), torch.zeros_like(m), m))
    l = p.sum(-1, keepdim=True)
    o = torch.einsum("shgnr,srhd->snhgd", p / torch.where(l > 0, l, torch.ones_like(l)), v[0])
    lse = (m + torch.log(l)).squeeze(-1).permute(0, 3, 1, 2)
    return dict(out=o.reshape(-1, n, H * G, hd)[ok].to(s["q"].dtype), lse=lse.reshape(-1, n, H * G)[ok])


def _plain_commit(s):
    c = s["case"]
    n = c["nodes"]
    t, ok = _nodes(s, n)
    par = torch.where(ok, s["parent"].long()[t], torch.full_like(t, -2))
    tok, nxt = s["tokens"].long()[t], s["next"].long()[t]
    hit = ok & (par >= 0) & (tok == torch.gather(nxt, 1, par.clamp_min(0)))
    i = torch.arange(n, device=DEV)
    # of the children that match, the first
    twin = hit[:, :, None] & hit[:, None] & (par[:, :, None] == par[:, None]) & (i[None, None] < i[None, :, None])
    link = torch.where(hit & ~twin.any(-1), par, torch.full_like(par, -1))
    took = _reach(link, n)[:, :, 0] & ok
    count = took.sum(1)
    path = torch.sort(torch.where(took, i[None], torch.full_like(t, n)), dim=1).values
    valid = path < n
    last = torch.gather(path, 1, (count - 1)[:, None])
    bonus = torch.gather(nxt, 1, last).squeeze(1)
    lens = s["lens"].long()
    src, dst = (lens[:, None] + path)[valid], (lens[:, None] + i[None])[valid]
    slot = torch.arange(c["slots"], device=DEV)[:, None].expand_as(path)[valid]
    pages = s["pages"].long()
    moved = s["kv"][:, pages[slot, src >> 4], :, src & 15]
    s["kv"][:, pages[slot, dst >> 4], :, dst & 15] = moved
    return dict(kv=s["kv"], lens=(lens + count).int(), accepted=count.int(),
                path=torch.where(valid, s["offsets"].long()[:-1, None] + path, torch.full_like(path, -1)).int(), bonus=bonus.int())


def _plain_weights(s):
    c = s["case"]
    H, G, hd, n = c["kv_heads"], c["group"], c["hd"], c["nodes"]
    R = s["pages"].shape[1] * PAGE
    lens, nq = s["lens"].long(), s["n_query"].long()
    k, _ = _rows(s, R)
    sel = s["sel"].long()
    q = s["q"].float()[:, sel].view(-1, c["slots"], n, H, G, hd)
    lse = s["lse"][:, sel].view(-1, c["slots"], n, H, G)
    p = torch.exp(torch.einsum("lsnhgd,lsrhd->lshgnr", q, k) * (1.0 / math.sqrt(hd)) - lse.permute(0, 1, 3, 4, 2)[..., None])
    i, r = torch.arange(n, device=DEV), torch.arange(R, device=DEV)
    see = (r[None, None] <= (lens[:, None] + i[None])[:, :, None]) & (i[None] < nq[:, None])[:, :, None]
    w = torch.where(see[None, :, None, None], p, torch.zeros_like(p[:1, :1, :1, :1, :1, :1])).sum((3, 4))
    old, new = r[None] < lens[:, None], r[None] < (lens + nq)[:, None]
    s["acc"].copy_(torch.where(old[None, :, None], s["acc"] + w, torch.where(new[None, :, None], w, s["acc"])))
    return dict(acc=s["acc"])


def _plain_evict(s):
    c = s["case"]
    B, H = c["budget"], c["kv_heads"]
    L, R = s["acc"].shape[0], s["acc"].shape[-1]
    lens = s["lens"].long()
    r = torch.arange(R, device=DEV)
    must = (r[None] < c["sinks"]) | (r[None] >= (lens - c["recent"])[:, None])
    key = torch.nan_to_num(s["acc"], nan=-math.inf, posinf=math.inf, neginf=-math.inf)
    key = torch.where(must[None, :, None], torch.full_like(key[:1, :1, :1, :1], math.inf), key)
    # heaviest first, ties to the lowest row; forced rows before all, rows past the end after all
    rank = torch.where(r[None] >= lens[:, None], 2, torch.where(must, 0, 1))
    order = torch.sort(key, dim=-1, descending=True, stable=True).indices
    by = torch.sort(torch.gather(rank[None, :, None].expand_as(order), -1, order), dim=-1, stable=True).indices
    top = torch.gather(order, -1, by)[..., :B]
    top = torch.nn.functional.pad(top, (0, B - top.shape[-1]), value=R)
    live = torch.arange(B, device=DEV)[None] < lens[:, None]
    kept = torch.sort(torch.where(live[None, :, None], top, torch.full_like(top, R)), dim=-1).values
    ok = kept < R
    at = kept.clamp_max(R - 1)
    acc = torch.where(ok, torch.gather(s["acc"], -1, at), torch.zeros_like(s["acc"][..., :1]))
    l, sl, h, j = torch.nonzero(ok, as_tuple=True)
    src = kept[ok]
    sp, dp = s["pages"].long()[sl, src >> 4], s["dst_pages"].long()[sl, j >> 4]
    s["dst"][l, dp, :, j & 15, h] = s["kv"][l, sp, :, src & 15, h]
    return dict(kv=s["dst"], lens=lens.clamp_max(B).int(), kept=torch.where(ok, kept, torch.full_like(kept, -1)).int(), acc=acc)


_PLAIN = dict(tree=_plain_tree, commit=_plain_commit, weights=_plain_weights, evict=_plain_evict)


# ---------------------------------------------------------------- 64 bits, slot by slot

def exact(case, seed):
    s = prepare(case, seed)
    return dict(tree=_exact_tree, commit=_exact_commit, weights=_exact_weights, evict=_exact_evict)[case["op"]](s)


def _slot(s, layer, sl, n):
    """K and V of the first n rows of a slot in 64 bits, [n][kv_heads][hd]."""
    pg = s["pages"][sl, :-(-n // PAGE)].long()
    x = s["kv"][layer, pg].double()  # [pages][2][16][kv_heads][hd]
    return x[:, 0].flatten(0, 1)[:n], x[:, 1].flatten(0, 1)[:n]


def _exact_tree(s):
    c = s["case"]
    H, G, hd = c["kv_heads"], c["group"], c["hd"]
    off, lens, par = s["offsets"].tolist(), s["lens"].tolist(), s["parent"].tolist()
    out = torch.zeros((off[-1], H * G, hd), dtype=torch.float64, device=DEV)
    lse = torch.full((off[-1], H * G), -math.inf, dtype=torch.float64, device=DEV)
    for sl in range(c["slots"]):
        n, t0, L = off[sl + 1] - off[sl], off[sl], lens[sl]
        see = torch.zeros((n, L + n), dtype=torch.bool)
        for i in range(n):
            if par[t0 + i] == -2:
                continue
            see[i, :L] = True
            j = i
            while j >= 0:
                see[i, L + j] = True
                j = par[t0 + j]
        k, v = _slot(s, 0, sl, L + n)
        rows = [i for i in range(n) if par[t0 + i] != -2]
        if not rows:
            continue
        see = see[rows].to(DEV)
        q = s["q"][t0:t0 + n].double()[rows].view(len(rows), H, G, hd)
        at = torch.tensor(rows, device=DEV) + t0
        for h in range(H):
            x = torch.einsum("ngd,rd->gnr", q[:, h], k[:, h]) / math.sqrt(hd)
            x = x.masked_fill(~see[None], -math.inf)
            lse[at, h * G:(h + 1) * G] = torch.logsumexp(x, -1).T
            out[at, h * G:(h + 1) * G] = torch.einsum("gnr,rd->ngd", torch.softmax(x, -1), v[:, h])
    return dict(out=out, lse=lse)


def _exact_commit(s):
    """Rows are moved, not computed: the moved cache is the whole answer."""
    c = s["case"]
    off, lens, par, tok, nxt = (s[k].tolist() for k in ("offsets", "lens", "parent", "tokens", "next"))
    pages = s["pages"].tolist()
    for sl in range(c["slots"]):
        t0, n, cur, path = off[sl], off[sl + 1] - off[sl], 0, [0]
        for i in range(1, n):
            if par[t0 + i] == cur and tok[t0 + i] == nxt[t0 + cur]:
                path.append(i)
                cur = i
        for j, i in enumerate(path):
            a, b = lens[sl] + i, lens[sl] + j
            if a != b:
                s["kv"][:, pages[sl][b // PAGE], :, b % PAGE] = s["kv"][:, pages[sl][a // PAGE], :, a % PAGE]
    return dict(kv=s["kv"], lens=None, accepted=None, path=None, bonus=None)


def _exact_weights(s):
    c = s["case"]
    H, G, hd = c["kv_heads"], c["group"], c["hd"]
    lens, nq, sel = s["lens"].tolist(), s["n_query"].tolist(), s["sel"].long()
    acc = s["acc"].double()
    for l in range(c["layers"]):
        for sl in range(c["slots"]):
            n, L = nq[sl], lens[sl]
            k, _ = _slot(s, l, sl, L + n)
            q = s["q"][l, sel[sl, :n]].double().view(n, H, G, hd)
            e = s["lse"][l, sel[sl, :n]].double().view(n, H, G)
            p = torch.exp(torch.einsum("nhgd,rhd->hgnr", q, k) / math.sqrt(hd) - e.permute(1, 2, 0)[..., None])
            p = p.tril(diagonal=L).sum((1, 2))
            acc[l, sl, :, :L] += p[:, :L]
            acc[l, sl, :, L:L + n] = p[:, L:]
    return dict(acc=acc)


def _exact_evict(s):
    c = s["case"]
    B, S0, W = c["budget"], c["sinks"], c["recent"]
    lens, pages, dpages = s["lens"].tolist(), s["pages"].cpu().numpy(), s["dst_pages"].cpu().numpy()
    acc = s["acc"].cpu().numpy()
    out = np.zeros(acc.shape[:3] + (B,))
    for l in range(acc.shape[0]):
        for sl in range(acc.shape[1]):
            n = lens[sl]
            for h in range(acc.shape[2]):
                if n <= B:
                    keep = np.arange(n)
                else:
                    a = acc[l, sl, h, S0:n - W].astype(np.float64)
                    a = np.where(np.isnan(a), -np.inf, a)
                    mid = np.argsort(-a, kind="stable")[:B - S0 - W] + S0
                    keep = np.sort(np.concatenate([np.arange(S0), mid, np.arange(n - W, n)]))
                out[l, sl, h, :len(keep)] = acc[l, sl, h, keep]
                j = np.arange(len(keep))
                sp, dp = _dev(pages[sl, keep >> 4], torch.int64), _dev(dpages[sl, j >> 4], torch.int64)
                s["dst"][l, dp, :, _dev(j & 15, torch.int64), h] = s["kv"][l, sp, :, _dev(keep & 15, torch.int64), h]
    return dict(kv=s["dst"], lens=None, kept=None, acc=torch.as_tensor(out))
