"""The operators on a paged KV cache at the edges of what they promise (needs a B200).

Tolerances are those of the operators' other tests: a score has an fp32 error of at most ex = scale * sum |q||k| * hd *
2^-23, an output one of (2.1 ex + 2^-18) max |v| and half a unit of its type.
"""
import numpy as np
import pytest
from test_gpu_kvops import PAGE, ancestors, check_tree, gpu, make_cache, plain_tree, random_tree, rows_of, run_tree

pytestmark = pytest.mark.gpu


# ---------------------------------------------------------------- the wide form's exchange between a row's halves

@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("G,n", [(4, 30), (8, 13), (1, 64), (4, 64)])
def test_wide_trees_over_one_tile_columns(G, n, bf16):
    """Columns of one tile, where the only tile moves every maximum and the sums follow at once, several to a CTA: the
    outputs of the plain form, and the same bits in every call."""
    import torch
    from hymt2_b200.kvcache import PagedKV
    rng = np.random.default_rng(G + n)
    check_tree(rng, 2, G, 64, bf16, [int(x) for x in rng.integers(0, 128 - n, 40)], [random_tree(rng, n) for _ in range(40)])
    S, kvh, hd = 300, 4, 128
    lens = rng.integers(0, 128 - n, S).astype(np.int32)
    kv, pages = make_cache(rng, 1, kvh, hd, [128] * S)
    cache = PagedKV(gpu(kv), gpu(pages))
    q = torch.randn(S * n, kvh * G, hd, device="cuda").to(torch.bfloat16 if bf16 else torch.float32)
    args = (q, gpu(lens), gpu(np.arange(S + 1, dtype=np.int32) * n), gpu(np.concatenate([random_tree(rng, n) for _ in range(S)])), n)
    out, lse = cache.tree_attention(*args)
    assert bool(torch.isfinite(out).all()) and bool(torch.isfinite(lse).all())
    for _ in range(20):
        again, lse2 = cache.tree_attention(*args)
        assert torch.equal(out, again) and torch.equal(lse, lse2)


# ---------------------------------------------------------------- token numbers that are not there

@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("n,G", [(3, 4), (40, 4), (13, 8)])
def test_offsets_past_the_tokens(n, G, bf16):
    """Offsets that name tokens past the arrays' end, negative or falling ones: such nodes do not exist, the others are
    as ever, and nothing around the outputs is touched."""
    import torch
    from hymt2_b200.kvcache import PagedKV
    rng = np.random.default_rng(n + G)
    kvh, hd, S = 2, 64, 4
    lens = np.array([50, 200, 0, 90], np.int32)
    kv, pages = make_cache(rng, 1, kvh, hd, [int(x) + 64 for x in lens])
    nt, dt = 2 * n, torch.bfloat16 if bf16 else torch.float32
    par = np.concatenate([random_tree(rng, n), random_tree(rng, n)])
    room_q, room_o = (torch.full((nt + 200, kvh * G, hd), 3.0, device="cuda", dtype=dt) for _ in range(2))
    room_l = torch.full((nt + 200, kvh * G), 3.0, device="cuda")
    room_q[100:100 + nt] = torch.from_numpy(rng.standard_normal((nt, kvh * G, hd)).astype(np.float32)).to(dt)
    q, out, lse = room_q[100:100 + nt], room_o[100:100 + nt], room_l[100:100 + nt]
    cache = PagedKV(gpu(kv), gpu(pages))
    big = np.iinfo(np.int32)
    whole, none = [0, n, nt, nt, nt], [0, 0, 0, 0, 0]
    for off, twin in (([0, n, nt + 60, nt + 70, nt + 90], whole), ([0, n, nt, big.max, big.max], whole), ([0, n, big.max, 0, -5], whole),
                      ([-30, n, nt, nt, nt], [n, n, nt, nt, nt]), ([big.min, big.max, n, 0, big.min], none), ([0, n, n, n - 1, -1], [0, n, n, n, n])):
        got = []
        for o in (off, twin):
            room_o.fill_(3.0)
            room_l.fill_(3.0)
            cache.tree_attention(q, gpu(lens), gpu(np.array(o, np.int32)), gpu(par), 64, out=out, lse=lse)
            got.append((room_o.clone(), room_l.clone()))
        assert all(torch.equal(a, b) for a, b in zip(*got)), off
        for room in got[0]:
            rest = torch.cat([room[:100 + twin[0]], room[100 + twin[-1]:]])
            assert bool((rest == 3.0).all()) and bool((room[100 + twin[0]:100 + twin[-1]] != 3.0).any()) == (twin != none), off


def test_commit_of_offsets_past_the_tokens():
    import torch
    from hymt2_b200.kvcache import PagedKV
    rng = np.random.default_rng(1)
    kv, pages = make_cache(rng, 2, 1, 64, [80] * 3)
    par, tok = gpu(np.array([-1, 0, 1, 2], np.int32)), gpu(np.array([7, 7, 7, 7], np.int32))
    lens = gpu(np.array([5, 9, 30], np.int32))
    for off, cnt in (([0, 3, 60, 70], [3, 1, 0]), ([-4, 4, 4, 4], [0, 0, 0]), ([0, 2, 4, 2147483647], [2, 1, 0])):  # token 3 names no node below it
        d = gpu(kv)
        ln, n, path, bonus = PagedKV(d, gpu(pages)).tree_commit(lens, gpu(np.array(off, np.int32)), par, tok, tok, 8)
        assert n.tolist() == cnt and ln.tolist() == [a + b for a, b in zip((5, 9, 30), cnt)]
        assert bonus.tolist() == [7 if c else -1 for c in cnt]
        assert int(path.max()) < 4 and torch.equal(d.cpu(), kv)  # chains from node 0: no row moves


@pytest.mark.parametrize("bf16", [False, True])
def test_weights_of_tokens_that_are_not_there(bf16):
    """A selected token past the queries is left out like a negative one."""
    import torch
    from hymt2_b200.kvcache import PagedKV
    rng = np.random.default_rng(2)
    kv, pages = make_cache(rng, 2, 2, 64, [160, 90])
    q = torch.from_numpy(rng.standard_normal((2, 6, 8, 64)).astype(np.float32)).to(torch.bfloat16 if bf16 else torch.float32).cuda()
    lse = torch.full((2, 6, 8), 4.0, device="cuda")
    lens, nq = gpu(np.array([130, 40], np.int32)), gpu(np.array([4, 3], np.int32))
    cache = PagedKV(gpu(kv), gpu(pages))
    got = []
    for gone in (-1, 6, 1 << 30, 2147483647):
        acc = torch.ones(2, 2, 2, 160, device="cuda")
        cache.add_weights(acc, q, lse, lens, nq, gpu(np.array([[0, gone, 5, 2], [gone, 1, 3, gone]], np.int32)))
        got.append(acc)
    assert bool((got[0] != 1).any()) and all(torch.equal(got[0], a) for a in got[1:])


# ---------------------------------------------------------------- infinities and NaN in cached rows

def spoil(kv, pages, slot, r, what, value, dims=slice(None), layer=0):
    """K (what 0) or V (1) of a row, in some dims of every KV head."""
    kv[layer, int(pages[slot, r // PAGE]), what, r % PAGE, :, dims] = value


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("G,n,L", [(4, 5, 40), (4, 5, 3000), (8, 13, 40), (8, 13, 3000), (4, 50, 3000)])
def test_padding_nodes_over_spoiled_rows(G, n, L, hd, bf16, bad):
    """A node that sees no row gets zeros and -inf whatever the slot's cached rows hold (columns of one tile and split
    ones, both forms)."""
    import torch
    rng = np.random.default_rng(L + n + hd)
    lens, trees = [L, 33], [random_tree(rng, n, pad=2), random_tree(rng, n)]
    kv, pages = make_cache(rng, 1, 2, hd, [L + n, 33 + n])
    for r in (0, L // 2, L - 1):
        spoil(kv, pages, 0, r, 0, bad, slice(3, 5))
        spoil(kv, pages, 0, r, 1, bad)
    q = gpu(torch.from_numpy(rng.standard_normal((2 * n, 2 * G, hd)).astype(np.float32)).to(torch.bfloat16 if bf16 else torch.float32))
    out, lse = run_tree(kv, pages, 0, lens, trees, q, n)
    assert (out[n - 2:n] == 0).all() and (lse[n - 2:n] == -np.inf).all()
    assert np.isfinite(out[n:]).all() and np.isfinite(lse[n:]).all()


def exact_tree(kv, pages, lens, trees, q, G, scale):
    """plain_tree with what infinities and NaN do: rows of score -inf drop out, +inf or NaN makes the output NaN (lse +inf
    or NaN), infinite V gives infinities."""
    nt, heads, hd = q.shape
    out, lse, tol, tlse = np.zeros((nt, heads, hd)), np.full((nt, heads), -np.inf), np.zeros((nt, heads, 1)), np.zeros((nt, heads))
    t0 = 0
    with np.errstate(invalid="ignore"):
        for s, par in enumerate(trees):
            k, v = rows_of(kv, pages, 0, s, lens[s] + len(par))
            for i, see in enumerate(ancestors(par)):
                seen = np.array(list(range(lens[s])) + [lens[s] + j for j in see], dtype=int)
                if not see:
                    continue
                for h in range(heads):
                    qq, t = q[t0 + i, h].astype(np.float64), t0 + i
                    x = scale * (k[seen, h // G] * qq).sum(-1)
                    rows, x = seen[x != -np.inf], x[x != -np.inf]
                    if not len(rows):
                        continue
                    if not np.isfinite(x).all():
                        out[t, h], lse[t, h] = np.nan, np.nan if np.isnan(x).any() else np.inf
                        continue
                    kk, vv = k[rows, h // G], v[rows, h // G]
                    ex = scale * (np.abs(kk) @ np.abs(qq)).max() * hd * 2.0 ** -23
                    m, p = x.max(), np.exp(x - x.max())
                    lse[t, h] = m + np.log(p.sum())
                    out[t, h] = (p[:, None] * vv).sum(0) / p.sum()
                    tol[t, h] = (2.1 * ex + 2.0 ** -18) * np.abs(vv[np.isfinite(vv)]).max()
                    tlse[t, h] = ex + 2.0 ** -18 + 2.0 ** -22 * abs(lse[t, h])
            t0 += len(par)
    return out, lse, tol, tlse


def same(got, want, tol):
    f = np.isfinite(want)
    with np.errstate(invalid="ignore"):
        ok = np.where(f, np.abs(got - np.where(f, want, 0)) <= tol, (got == want) | (np.isnan(got) & np.isnan(want)))
    return ok.all(), np.argwhere(~ok)[:5].tolist()


@pytest.mark.parametrize("case", ["v_inf", "v_two", "v_nan", "v_far", "k_inf", "k_all", "k_nan", "drafted", "q_inf"])
@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("G,n,L", [(4, 5, 40), (4, 5, 2000), (8, 13, 40), (8, 13, 2000), (4, 40, 900)])
def test_infinities_in_rows_that_are_seen(G, n, L, hd, bf16, case):
    """The formulas' effect, dim by dim, in both forms, in columns of one tile and split ones."""
    import torch
    rng = np.random.default_rng(L + n + hd)
    kvh, inf, nan = 2, float("inf"), float("nan")
    lens, trees = [L, 33], [random_tree(rng, n, pad=1), random_tree(rng, n)]
    kv, pages = make_cache(rng, 1, kvh, hd, [L + n, 33 + n])
    q = torch.from_numpy(rng.standard_normal((2 * n, kvh * G, hd)).astype(np.float32)).to(torch.bfloat16 if bf16 else torch.float32)
    if case == "v_inf":
        spoil(kv, pages, 0, L // 3, 1, inf, slice(2, 4))
        spoil(kv, pages, 0, L - 1, 1, -inf, slice(hd - 9, hd))
    elif case == "v_two":   # both signs in one dim: NaN there
        spoil(kv, pages, 0, 0, 1, inf, slice(0, 3))
        spoil(kv, pages, 0, L - 1, 1, -inf, slice(2, 7))
    elif case == "v_nan":
        spoil(kv, pages, 0, 7, 1, nan, slice(1, 2))
    elif case == "v_far":   # a row whose probability is below fp32's range
        spoil(kv, pages, 0, 5, 1, -inf, slice(6, 7))
        q = q * 40
        q[..., 9] = 60
        spoil(kv, pages, 0, 5, 0, -8.0, slice(9, 10))
    elif case == "k_inf":   # scores of -inf and of +inf, as the query's sign has it
        spoil(kv, pages, 0, 3, 0, inf, slice(11, 12))
        spoil(kv, pages, 0, L - 2, 0, -inf, slice(20, 21))
    elif case == "k_all":   # every row of the tree's: all scores -inf or all +inf in each head
        for r in range(L + n):
            spoil(kv, pages, 0, r, 0, inf, slice(11, 12))
    elif case == "k_nan":
        spoil(kv, pages, 0, L // 2, 0, nan, slice(0, 1))
    elif case == "drafted":
        spoil(kv, pages, 0, L, 1, inf, slice(5, 6))
        spoil(kv, pages, 0, L + 1, 0, -inf, slice(8, 9))
        spoil(kv, pages, 0, L + 2, 1, nan, slice(hd - 1, hd))
    else:
        q[1, 0, 4], q[n + 2, 3, 7] = inf, -inf
    sc = hd ** -0.5
    out, lse = run_tree(kv, pages, 0, lens, trees, gpu(q), n)
    want, wlse, tol, tlse = exact_tree(kv, pages, lens, trees, q.double().numpy(), G, sc)
    if bf16:
        tol = tol + np.where(np.isfinite(want), np.abs(want), 0) * 2.0 ** -8
    assert not np.isfinite(want).all() or case == "v_far"
    ok, where = same(out, want, tol)
    assert ok, where
    ok, where = same(lse, wlse, tlse)
    assert ok, where


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("hd,maxq", [(128, 5), (64, 40)])
def test_weights_of_infinite_keys(hd, maxq, bf16):
    """A key of +-inf adds nothing where the score is -inf, and infinity where it is +inf; NaN stays in its row."""
    import torch
    from hymt2_b200.kvcache import PagedKV
    rng = np.random.default_rng(hd)
    L, kvh, G = 300, 2, 4
    kv, pages = make_cache(rng, 1, kvh, hd, [L + maxq])
    spoil(kv, pages, 0, 10, 0, float("inf"), slice(3, 4))
    spoil(kv, pages, 0, L + 1, 0, -float("inf"), slice(5, 6))
    spoil(kv, pages, 0, 200, 0, float("nan"), slice(0, 1))
    q = torch.from_numpy(rng.standard_normal((1, maxq, kvh * G, hd)).astype(np.float32)).to(torch.bfloat16 if bf16 else torch.float32)
    q[:, :, :G, 3] = -q[:, :, :G, 3].abs()  # the first head's group: scores of -inf only
    lse = torch.full((1, maxq, kvh * G), 4.0)
    acc = torch.zeros(1, 1, kvh, L + maxq, device="cuda")
    PagedKV(gpu(kv), gpu(pages)).add_weights(acc, gpu(q), gpu(lse), gpu(np.array([L], np.int32)), gpu(np.array([maxq], np.int32)),
                                             gpu(np.arange(maxq, dtype=np.int32)[None]))
    got, (k, _) = acc[0, 0].double().cpu().numpy(), rows_of(kv, pages, 0, 0, L + maxq)
    for h in range(kvh):
        qq = q[0, :, h * G:(h + 1) * G].double().numpy()
        with np.errstate(invalid="ignore"):
            x = (k[:, h][:, None, None] * qq[None]).sum(-1) * hd ** -0.5
        x = np.where(np.arange(L + maxq)[:, None, None] <= L + np.arange(maxq)[None, :, None], x, -np.inf)
        want = np.exp(x - 4.0).sum((1, 2))
        # a score's error: hd products of 2^-23 of their sum of sizes, under 200 here; sums of up to 160 terms
        ok, where = same(got[h], want, np.where(np.isfinite(want), want, 0) * (200 * hd ** -0.5 * hd * 2.0 ** -23 + 2.0 ** -16))
        assert ok, (h, where)
    assert np.isfinite(got[0, 10]) and np.isinf(got[1, 10]) and np.isnan(got[:, 200]).all()


# ---------------------------------------------------------------- eviction within one cache

@pytest.mark.parametrize("hd,kvh", [(128, 2), (64, 3)])
@pytest.mark.parametrize("budget,sinks,recent", [(1, 0, 0), (1, 0, 1), (63, 4, 8), (64, 0, 0), (65, 30, 34), (513, 3, 100), (2000, 4, 4)])
def test_evict_within_the_cache(hd, kvh, budget, sinks, recent):
    """The same rows, lists and weights as into another cache; slots within the budget, rows behind a slot's and pages of
    no slot stay."""
    import torch
    from hymt2_b200.kvcache import PagedKV
    rng = np.random.default_rng(budget + hd)
    layers, lens = 2, [0, 1, budget, budget + 1, 700, 1030, 2047]
    S, R = len(lens), 2064
    kv, pages = make_cache(rng, layers, kvh, hd, [R] * S)
    acc = gpu(np.round(np.exp(3 * rng.standard_normal((layers, S, kvh, R)))).astype(np.float32))
    acc[1, 5] = acc[1, 5].flip(-1).cumsum(-1)   # one slot whose last rows are the heaviest
    acc[0, 6] = acc[0, 6].cumsum(-1).flip(-1)   # and one whose first are
    ln = gpu(np.array(lens, np.int32))
    one, two = gpu(kv), gpu(kv)
    page_max = -(-budget // PAGE)
    dst, dpages = torch.zeros(layers, S * page_max, 2, PAGE, kvh, hd, dtype=torch.bfloat16, device="cuda"), np.arange(S * page_max).reshape(S, page_max)
    want = PagedKV(one, gpu(pages)).evict(PagedKV(dst, gpu(dpages.astype(np.int32))), ln, acc, budget, sinks, recent)
    cache = PagedKV(two, gpu(pages))
    got = cache.evict(cache, ln, acc, budget, sinks, recent)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    full, moved, dst = kv.clone(), two.cpu(), dst.cpu()
    for s in range(S):
        if lens[s] > budget:
            j = np.arange(budget)
            full[:, pages[s, j // PAGE], :, j % PAGE] = dst[:, dpages[s, j // PAGE], :, j % PAGE]
    assert torch.equal(moved, full)


# ---------------------------------------------------------------- calls without tokens or queries

def test_commit_without_tokens():
    """No slot drafts anything: every length stays, nothing is accepted or moved."""
    import torch
    from hymt2_b200.kvcache import PagedKV
    rng = np.random.default_rng(3)
    kv, pages = make_cache(rng, 2, 1, 64, [40, 40])
    d, none = gpu(kv), torch.empty(0, dtype=torch.int32, device="cuda")
    lens = gpu(np.array([7, 0], np.int32))
    for forced in (None, gpu(np.array([1, 0], np.int32))):
        ln, n, path, bonus = PagedKV(d, gpu(pages)).tree_commit(lens, gpu(np.zeros(3, np.int32)), none, none, none, 4, forced=forced)
        assert ln.tolist() == [7, 0] and n.tolist() == [0, 0] and bonus.tolist() == [-1, -1] and bool((path == -1).all())
    assert torch.equal(d.cpu(), kv)


def test_weights_without_queries_or_tokens():
    import torch
    from hymt2_b200.kvcache import PagedKV
    rng = np.random.default_rng(3)
    kv, pages = make_cache(rng, 1, 2, 64, [40, 40])
    cache, lens = PagedKV(gpu(kv), gpu(pages)), gpu(np.array([7, 20], np.int32))
    acc = torch.ones(1, 2, 2, 48, device="cuda")
    q, lse = torch.randn(1, 3, 4, 64, device="cuda"), torch.zeros(1, 3, 4, device="cuda")
    zero = gpu(np.zeros(2, np.int32))
    cache.add_weights(acc, q, lse, lens, zero, gpu(np.zeros((2, 0), np.int32)))
    cache.add_weights(acc, q, lse, lens, zero, gpu(np.zeros((2, 5), np.int32)))
    cache.add_weights(acc, q[:, :0], lse[:, :0], lens, zero, gpu(np.zeros((2, 5), np.int32)))
    assert bool((acc == 1).all())
    # queries that are not there are left out; their rows start from zero like any
    cache.add_weights(acc, q[:, :0], lse[:, :0], lens, gpu(np.array([2, 0], np.int32)), gpu(np.zeros((2, 5), np.int32)))
    assert bool((acc[0, 0, :, 7:9] == 0).all()) and float(acc.sum()) == 2 * 2 * 48 - 4


# ---------------------------------------------------------------- scratch

def _long_trees(n=12):
    from hymt2_b200.kvcache import PagedKV
    import torch
    rng = np.random.default_rng(2)
    lens, trees = [900, 2, 333], [random_tree(rng, x) for x in (n, n, 1)]
    kv, pages = make_cache(rng, 1, 4, 128, [950, 50, 400])
    args = (torch.randn(2 * n + 1, 16, 128, device="cuda"), gpu(np.array(lens, np.int32)), gpu(np.array([0, n, 2 * n, 2 * n + 1], np.int32)),
            gpu(np.concatenate(trees)))
    return PagedKV(gpu(kv), gpu(pages)), args


@pytest.mark.parametrize("n", [3, 40])
def test_a_captured_call_has_a_scratch_of_its_own(n):
    """Warmed up and captured on one side stream: replays use none of that stream's scratch, two graphs none of each
    other's, and they outlive the handle."""
    import torch
    cache, args = _long_trees(n)
    want = cache.tree_attention(*args, n)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        for _ in range(3):
            cache.tree_attention(*args, n)
    s.synchronize()
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            graphs.append((g, cache.tree_attention(*args, n)))
    held = [ws[0] for ws in cache._ws.values()]
    for buf in held:
        buf.fill_(0x55)
    torch.cuda.synchronize()
    for g, _ in graphs:
        g.replay()
    torch.cuda.synchronize()
    assert all(bool((buf == 0x55).all()) for buf in held)
    streams = [torch.cuda.Stream() for _ in graphs]
    for _ in range(20):  # side by side
        for st, (g, _) in zip(streams, graphs):
            with torch.cuda.stream(st):
                g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(o, w) for _, out in graphs for o, w in zip(out, want))
    kv, pages = cache.kv, cache.pages  # the graphs' inputs stay, their handle goes
    del cache, held, buf
    torch.cuda.empty_cache()
    for g, out in graphs:
        out[0].zero_()
        g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(o, w) for _, out in graphs for o, w in zip(out, want)) and kv.is_cuda and pages.is_cuda


def test_one_scratch_for_all_widths():
    import torch
    cache, args = _long_trees(12)
    want = cache.tree_attention(*args, 12)
    for n in list(range(12, 65)) + [12, 64, 12]:
        out = cache.tree_attention(*args, n)[0]
        assert float((out - want[0]).abs().max()) < 1e-4   # other splits and forms of the same sums
    assert len(cache._ws) == 1
    need = [cache._lib.hyc_tree_attention_ws(cache._ref, 16, n) for n in range(12, 65)]
    assert next(iter(cache._ws.values()))[0].numel() == max(need)
    assert all(ws is next(iter(cache._ws.values())) for ws in cache._fit.values())
    torch.cuda.synchronize()


def test_queries_of_one_head():
    """One head has no stride of its own: any that torch carries for it will do."""
    import torch
    from hymt2_b200.kvcache import PagedKV
    rng = np.random.default_rng(4)
    kv, pages = make_cache(rng, 2, 1, 64, [60])
    cache, n = PagedKV(gpu(kv), gpu(pages)), 5
    lens, off, par = gpu(np.array([50], np.int32)), gpu(np.array([0, n], np.int32)), gpu(random_tree(rng, n))
    q = torch.randn(2, n, 1, 64, device="cuda")
    want, lse = cache.tree_attention(q[0], lens, off, par, n)
    odd = torch.empty(1, n, 64, device="cuda").copy_(q[0].transpose(0, 1)).transpose(0, 1)   # [n][1][64] of strides (64, 64 n, 1)
    assert odd.stride(1) == 64 * n
    out = torch.zeros(1, n, 64, device="cuda").transpose(0, 1)
    got, lse2 = cache.tree_attention(odd, lens, off, par, n, out=out)
    assert torch.equal(got, want) and torch.equal(lse, lse2)
    acc = [torch.zeros(2, 1, 1, 64, device="cuda") for _ in range(2)]
    sel, e = gpu(np.arange(n, dtype=np.int32)[None]), torch.full((2, n, 1), 3.0, device="cuda")
    for a, x in zip(acc, (q, torch.empty(2, 1, n, 64, device="cuda").copy_(q.transpose(1, 2)).transpose(1, 2))):
        cache.add_weights(a, x, e, lens, gpu(np.array([n], np.int32)), sel)
    assert torch.equal(*acc) and bool((acc[0] != 0).any())


@pytest.mark.parametrize("scale", [float("nan"), float("inf"), -float("inf")])
def test_a_scale_that_is_not_finite_is_refused(scale):
    """(It was taken for one next to 0: every row the same weight.)"""
    import torch
    from hymt2_b200.device import BackendError
    from hymt2_b200.kvcache import PagedKV
    rng = np.random.default_rng(4)
    kv, pages = make_cache(rng, 1, 1, 64, [60])
    cache, q = PagedKV(gpu(kv), gpu(pages)), torch.randn(1, 1, 64, device="cuda")
    one, off = gpu(np.array([50], np.int32)), gpu(np.array([0, 1], np.int32))
    with pytest.raises(BackendError, match="scale"):
        cache.tree_attention(q, one, off, gpu(np.array([-1], np.int32)), 1, scale=scale)
    with pytest.raises(BackendError, match="scale"):
        cache.add_weights(torch.zeros(1, 1, 1, 64, device="cuda"), q[None], torch.zeros(1, 1, 1, device="cuda"), one, off[1:],
                          gpu(np.zeros((1, 1), np.int32)), scale=scale)


# ---------------------------------------------------------------- pages that are not there, lengths out of range

NO_PAGE = (-1, -2 ** 31, 2 ** 31 - 1)


def holes(rng, kv, pages, slots):
    """Page tables with numbers outside the pool in some places, and for the plain form a pool with a page of zeros there."""
    import torch
    plain_kv = torch.cat([kv, torch.zeros_like(kv[:, :1])], 1)
    plain, table = pages.copy(), pages.copy()
    for s in slots:
        for i, j in enumerate(rng.choice(pages.shape[1], max(1, pages.shape[1] // 3), replace=False)):
            plain[s, j] = kv.shape[1]
            table[s, j] = (*NO_PAGE, kv.shape[1])[i % 4]
    return plain_kv, plain, table


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("G,n,L", [(4, 5, 60), (4, 5, 700), (8, 13, 60), (8, 13, 700)])
def test_attention_over_pages_that_are_not_there(G, n, L, bf16):
    """They read as rows of zeros."""
    import torch
    rng = np.random.default_rng(n + L)
    lens, trees = [L, 30], [random_tree(rng, n), random_tree(rng, n)]
    kv, pages = make_cache(rng, 1, 2, 64, [L + n, 30 + n])
    plain_kv, plain, table = holes(rng, kv, pages, (0, 1))
    q = torch.from_numpy(rng.standard_normal((2 * n, 2 * G, 64)).astype(np.float32)).to(torch.bfloat16 if bf16 else torch.float32)
    out, lse = run_tree(kv, table, 0, lens, trees, gpu(q), n)
    want, wlse, tol, tlse = plain_tree(plain_kv, plain, 0, lens, trees, q.double().numpy(), G, 64 ** -0.5)
    if bf16:
        tol = tol + np.abs(want) * 2.0 ** -8
    assert (np.abs(out - want) <= tol).all() and (np.abs(lse - wlse) <= tlse).all()


@pytest.mark.parametrize("G,n", [(4, 5), (8, 13)])
def test_lengths_out_of_range(G, n):
    """Below 0 they count as 0, past the page table as all of its rows; nodes' rows past it do not exist."""
    import torch
    from hymt2_b200.kvcache import PagedKV
    rng = np.random.default_rng(n)
    kv, pages = make_cache(rng, 2, 2, 64, [160] * 4)
    cap = pages.shape[1] * PAGE
    cache, big = PagedKV(gpu(kv), gpu(pages)), np.iinfo(np.int32)
    off, par = gpu(np.arange(5, dtype=np.int32) * n), gpu(np.concatenate([random_tree(rng, n) for _ in range(4)]))
    q = torch.randn(2, 4 * n, 2 * G, 64, device="cuda")
    wild, tame = (gpu(np.array(x, np.int32)) for x in ([-1, big.min, cap + 1, big.max], [0, 0, cap, cap]))
    got, want = (cache.tree_attention(q[0], x, off, par, n) for x in (wild, tame))
    assert all(torch.equal(a, b) for a, b in zip(got, want)) and bool(torch.isfinite(got[0]).all())
    ref = plain_tree(kv, pages, 0, [0, 0, cap, cap], np.split(par.cpu().numpy(), 4), q[0].cpu().double().numpy(), G, 64 ** -0.5)
    assert (np.abs(got[0].cpu().numpy() - ref[0]) <= ref[2]).all() and (np.abs(got[1].cpu().numpy() - ref[1]) <= ref[3]).all()
    acc, e = [torch.ones(2, 4, 2, cap, device="cuda") for _ in range(2)], torch.full((2, 4 * n, 2 * G), 4.0, device="cuda")
    sel, nq = gpu(np.arange(4 * n, dtype=np.int32).reshape(4, n)), gpu(np.array([n, big.max, n, -3], np.int32))
    for a, x in zip(acc, (wild, tame)):
        cache.add_weights(a, q, e, x, nq, sel)
    assert torch.equal(*acc) and bool((acc[0][:, 3] == 1).all()) and bool((acc[0][:, 2] > 1).all())
    assert bool((acc[0][:, :2, :, n:] == 1).all())
    kept = [cache.evict(PagedKV(torch.zeros_like(cache.kv), cache.pages), x, acc[0], 20, 2, 5) for x in (wild, tame)]
    assert all(torch.equal(a, b) for a, b in zip(*kept)) and kept[0][0].tolist() == [0, 0, 20, 20]


def test_moves_over_pages_that_are_not_there():
    """Commit and eviction: such rows move as zeros, and nothing is written in their place."""
    import torch
    from hymt2_b200.kvcache import PagedKV
    rng = np.random.default_rng(6)
    kv, pages = make_cache(rng, 2, 2, 64, [96])
    par, n = np.array([-1, 0, 0, 2, 2, 4], np.int32), 6
    tok, nxt = np.array([9, 1, 2, 3, 4, 5], np.int32), np.array([2, 0, 4, 0, 5, 0], np.int32)   # the path 0, 2, 4, 5
    zero = torch.zeros(2, 2, 2, 64, dtype=torch.bfloat16)
    row = lambda t, r: t[:, int(pages[0, r // PAGE]), :, r % PAGE]
    for no in NO_PAGE + (kv.shape[1],):
        for L, hole in ((29, 2), (29, 1), (13, 0), (91, 5)):
            table, d = pages.copy(), gpu(kv)
            table[0, hole] = no
            PagedKV(d, gpu(table)).tree_commit(gpu(np.array([L], np.int32)), gpu(np.array([0, n], np.int32)), gpu(par), gpu(tok), gpu(nxt), n)
            want = kv.clone()
            for j, i in enumerate((0, 2, 4, 5)):
                if i != j and (L + j) // PAGE != hole and L + j < 96:
                    src = zero if L + i >= 96 or (L + i) // PAGE == hole else row(want, L + i).clone()
                    row(want, L + j)[:] = src
            assert torch.equal(d.cpu(), want), (no, L, hole)
    acc = gpu(rng.random((2, 1, 2, 96)).astype(np.float32))
    for no in NO_PAGE + (kv.shape[1],):
        table = pages.copy()
        table[0, 1] = no
        dst, dtable = torch.full_like(kv, 7.0).cuda(), np.array([[3, no, 5]], np.int32)
        _, kept, _ = PagedKV(gpu(kv), gpu(table)).evict(PagedKV(dst, gpu(dtable)), gpu(np.array([90], np.int32)), acc, 40, 3, 9)
        kept, want = kept.cpu().numpy(), torch.full_like(kv, 7.0)
        for l in range(2):
            for h in range(2):
                for j, r in enumerate(kept[l, 0, h]):
                    if j // PAGE != 1:
                        want[l, int(dtable[0, j // PAGE]), :, j % PAGE, h] = 0 if r // PAGE == 1 else kv[l, int(pages[0, r // PAGE]), :, r % PAGE, h]
        assert torch.equal(dst.cpu(), want), no
