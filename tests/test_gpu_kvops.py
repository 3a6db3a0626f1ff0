"""The operators on a paged KV cache against plain 64-bit implementations (needs a B200).

Tolerances.  A score x = scale * q . k has an fp32 error of at most ex = scale * sum |q||k| * hd * 2^-23 (hd products
and sums, each rounded or truncated to 24 bits).  A probability is then off by a factor of at most e^(2 ex) (its own
score and the sum's) and by the exponential's and the sums' roundings, under 2^-18 for these lengths; outputs are
averages of V by those probabilities, so they are off by at most (2.1 ex + 2^-18) max |v|, plus half a unit of the
output's type.  Weights add such probabilities to a stored fp32 sum (one rounding of 2^-23 at most).
"""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

PAGE = 16


def make_cache(rng, layers, kvh, hd, caps, garbage=None):
    """A pool whose slots own shuffled pages for caps[s] rows; rows hold N(0, 1), spare pages `garbage`."""
    import torch
    page_max = max(1, max(-(-c // PAGE) for c in caps))
    npages = len(caps) * page_max + 2
    kv = torch.from_numpy(rng.standard_normal((layers, npages, 2, PAGE, kvh, hd)).astype(np.float32)).to(torch.bfloat16)
    pages = rng.permutation(npages)[:len(caps) * page_max].reshape(len(caps), page_max).astype(np.int32)
    if garbage is not None:
        spare = np.setdiff1d(np.arange(npages), pages.reshape(-1))
        kv[:, torch.from_numpy(spare)] = garbage
    return kv, pages


def rows_of(kv, pages, layer, slot, n):
    """(K, V) of rows 0 .. n - 1 in 64 bits, [n][kvh][hd]."""
    p = pages[slot][np.arange(n) // PAGE]
    x = kv[layer, p, :, np.arange(n) % PAGE].double().numpy()
    return x[:, 0], x[:, 1]


def random_tree(rng, n, pad=0):
    par = np.array([-1] + [int(rng.integers(max(0, i - 7), i)) for i in range(1, n)], dtype=np.int32)[:n]
    if pad:
        par[n - pad:] = -2
    return par


def ancestors(par):
    """see[i]: the nodes node i sees (itself and its ancestors)."""
    out = []
    for i in range(len(par)):
        see, j = [], i
        if par[i] != -2:
            while True:
                see.append(j)
                p = par[j]
                if p < 0 or p >= j or par[p] == -2:
                    break
                j = int(p)
        out.append(sorted(see))
    return out


def plain_tree(kv, pages, layer, lens, trees, q, G, scale):
    """out [nt][heads][hd], lse [nt][heads] in 64 bits, and the error bound of each."""
    nt, heads, hd = q.shape
    out, lse = np.zeros((nt, heads, hd)), np.full((nt, heads), -np.inf)
    tol, tlse = np.zeros((nt, heads, 1)), np.zeros((nt, heads))
    t0 = 0
    cap = pages.shape[1] * PAGE
    for s, par in enumerate(trees):
        L, n = lens[s], len(par)
        k, v = rows_of(kv, pages, layer, s, min(cap, L + n))
        for i, see in enumerate(ancestors(par)):
            rows = np.array([r for r in list(range(L)) + [L + j for j in see] if r < cap], dtype=int)
            if not see or not len(rows):
                continue
            for h in range(heads):
                qq = q[t0 + i, h].astype(np.float64)
                x = scale * (k[rows, h // G] @ qq)
                ex = abs(scale) * (np.abs(k[rows, h // G]) @ np.abs(qq)).max() * hd * 2.0 ** -23
                m = x.max()
                p = np.exp(x - m)
                out[t0 + i, h] = p @ v[rows, h // G] / p.sum()
                lse[t0 + i, h] = m + np.log(p.sum())
                tol[t0 + i, h] = (2.1 * ex + 2.0 ** -18) * np.abs(v[rows, h // G]).max()
                tlse[t0 + i, h] = ex + 2.0 ** -18 + 2.0 ** -22 * abs(lse[t0 + i, h])
        t0 += n
    return out, lse, tol, tlse


def gpu(x, dtype=None):
    import torch
    t = x if isinstance(x, torch.Tensor) else torch.from_numpy(np.ascontiguousarray(x))
    return t.to("cuda", dtype=dtype) if dtype else t.cuda()


def run_tree(kv, pages, layer, lens, trees, q, max_nodes, **kw):
    from hymt2_b200.kvcache import PagedKV
    off = np.concatenate([[0], np.cumsum([len(t) for t in trees])]).astype(np.int32)
    par = np.concatenate([np.zeros(0, np.int32)] + [np.asarray(t, np.int32) for t in trees])
    cache = PagedKV(gpu(kv), gpu(pages))
    out, lse = cache.tree_attention(q, gpu(np.asarray(lens, np.int32)), gpu(off), gpu(par), max_nodes, layer=layer, **kw)
    return out.float().cpu().numpy().astype(np.float64), lse.cpu().numpy().astype(np.float64)


def check_tree(rng, kvh, G, hd, bf16, lens, trees, layers=1, layer=0, qscale=1.0, spread=0, max_nodes=None, kv_pages=None, scale=None):
    import torch
    nt = sum(len(t) for t in trees)
    caps = [L + len(t) for L, t in zip(lens, trees)]
    kv, pages = kv_pages or make_cache(rng, layers, kvh, hd, caps, garbage=float("nan"))
    q = torch.from_numpy(rng.standard_normal((nt, kvh * G * hd + spread)).astype(np.float32) * qscale)
    q = q.to(torch.bfloat16 if bf16 else torch.float32)
    dq = gpu(q)[:, :kvh * G * hd].view(nt, kvh * G, hd)
    hq = q[:, :kvh * G * hd].reshape(nt, kvh * G, hd).double().numpy()
    sc = hd ** -0.5 if scale is None else scale
    out, lse = run_tree(kv, pages, layer, lens, trees, dq, max_nodes or max(1, max(len(t) for t in trees)), scale=scale)
    want, wlse, tol, tlse = plain_tree(kv, pages, layer, lens, trees, hq, G, sc)
    if bf16:
        tol = tol + np.abs(want) * 2.0 ** -8
    assert np.isfinite(out).all()
    err = np.abs(out - want)
    assert (err <= tol).all(), (float(err.max()), float(tol.max()))
    assert (np.isinf(lse) == np.isinf(wlse)).all()
    f = np.isfinite(wlse)
    assert (np.abs(lse - wlse)[f] <= tlse[f]).all()


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("G", [1, 2, 4, 8])
def test_tree_attention_geometries(hd, G, bf16):
    rng = np.random.default_rng(100 + hd + G + bf16)
    lens = [0, 1, 17, 300, 95]
    trees = [random_tree(rng, n) for n in (5, 1, 16, 33, 64)]
    check_tree(rng, 3, G, hd, bf16, lens, trees, layers=2, layer=1, spread=64)


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("L", [0, 1, 15, 16, 31, 32, 63, 64, 65, 127, 128, 129, 1000, 4097])
def test_tree_attention_lengths(L, bf16):
    """A single token and a few nodes at lengths around every tile's edge."""
    rng = np.random.default_rng(L + 7 * bf16)
    for n in (1, 3):
        check_tree(rng, 2, 4, 128, bf16, [L], [random_tree(rng, n)])


@pytest.mark.parametrize("n", [1, 2, 4, 5, 7, 8, 9, 16, 17, 31, 32, 33, 63, 64])
def test_tree_attention_widths(n):
    rng = np.random.default_rng(n)
    check_tree(rng, 1, 4, 128, False, [200, 61], [random_tree(rng, n), random_tree(rng, n)])


@pytest.mark.parametrize("bf16", [False, True])
def test_tree_attention_shapes_of_trees(bf16):
    """Chains, stars, several roots, padding nodes, a parent that is not below its node, empty trees."""
    rng = np.random.default_rng(5)
    chain = np.arange(-1, 63)
    star = np.array([-1] + [0] * 40)
    roots = np.full(20, -1)
    odd = np.array([-1, 0, 5, 3, -7, 2, 1, 4])       # nodes 2, 3, 4: no parent below them
    pads = np.array([-1, 0, -2, 2, 1, -2, 4])         # node 3 hangs from a padding node
    trees = [chain, star, np.zeros(0, int), roots, odd, pads, np.full(9, -2)]
    check_tree(rng, 2, 4, 128, bf16, [70, 33, 50, 0, 9, 64, 12], trees)


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("G,n", [(1, 32), (4, 8), (4, 5), (8, 4), (4, 40), (1, 60)])
def test_tree_attention_padding_over_long_caches(G, n, hd, bf16):
    """Padding nodes see no row of a cache of several tiles either, and one-node trees stand beside them."""
    rng = np.random.default_rng(G + n + hd)
    trees = [random_tree(rng, n, pad=n // 2), random_tree(rng, 1), np.full(n, -2), random_tree(rng, n - 1, pad=1)]
    check_tree(rng, 2, G, hd, bf16, [700, 300, 511, 64], trees, max_nodes=n)


def test_tree_attention_many_ragged_slots():
    rng = np.random.default_rng(8)
    lens = [int(x) for x in rng.integers(0, 400, 90)]
    trees = [random_tree(rng, int(n)) for n in rng.integers(0, 20, 90)]
    check_tree(rng, 2, 4, 64, False, lens, trees, max_nodes=25)
    check_tree(rng, 2, 8, 128, True, lens, trees, max_nodes=20)


@pytest.mark.parametrize("qscale", [0.0, 30.0, 2000.0])
def test_tree_attention_sharp_and_flat_softmax(qscale):
    """All scores equal; scores whose exponentials span the whole range; a maximum that keeps growing along the rows."""
    rng = np.random.default_rng(3)
    for bf16 in (False, True):
        check_tree(rng, 2, 4, 128, bf16, [700, 129], [random_tree(rng, 24), random_tree(rng, 2)], qscale=qscale)
    kv, pages = make_cache(rng, 1, 1, 64, [600])
    for r in range(600):
        kv[0, int(pages[0, r // PAGE]), 0, r % PAGE] *= r / 100.0
    check_tree(rng, 1, 8, 64, False, [590], [random_tree(rng, 10)], qscale=4.0, kv_pages=(kv, pages))
    check_tree(rng, 1, 8, 64, False, [590], [random_tree(rng, 10)], scale=-0.3, kv_pages=(kv, pages))


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("n,bf16", [(4, False), (30, False), (30, True)])
def test_tree_attention_hidden_rows_never_reach(bad, n, bf16):
    """NaN and infinities in rows behind the tree, and in drafted rows that a node does not see, stay out of it."""
    import torch
    rng = np.random.default_rng(17)
    L, G, hd = 85, 4, 128
    par = random_tree(rng, n)
    kv, pages = make_cache(rng, 1, 2, hd, [L + n + 40])
    see = ancestors(par)
    for r in range(L + n, pages.shape[1] * PAGE):
        kv[0, int(pages[0, r // PAGE]), :, r % PAGE] = bad
    q = torch.from_numpy(rng.standard_normal((n, 2 * G, hd)).astype(np.float32)).to(torch.bfloat16 if bf16 else torch.float32)
    clean, clse = run_tree(kv, pages, 0, [L], [par], gpu(q), n)
    assert np.isfinite(clean).all()
    j = n - 2  # a drafted row whose K and V go bad
    r = L + j
    kv[0, int(pages[0, r // PAGE]), :, r % PAGE] = bad
    out, lse = run_tree(kv, pages, 0, [L], [par], gpu(q), n)
    blind = [i for i in range(n) if j not in see[i]]
    assert len(blind) >= n // 2
    assert np.array_equal(out[blind], clean[blind]) and np.array_equal(lse[blind], clse[blind])
    # V alone: the probabilities stay, the nodes that see the row have it in their output
    kv[0, int(pages[0, r // PAGE]), 0, r % PAGE] = 0.5
    out, lse = run_tree(kv, pages, 0, [L], [par], gpu(q), n)
    assert np.isfinite(out[blind]).all() and np.isfinite(lse).all()
    seers = [i for i in range(n) if j in see[i]]
    assert not np.isfinite(out[seers]).any()


def test_tree_attention_same_bits_twice_other_stream_graph_and_out():
    import torch
    from hymt2_b200.kvcache import PagedKV
    rng = np.random.default_rng(2)
    lens, trees = [900, 2, 333], [random_tree(rng, n) for n in (12, 40, 1)]
    kv, pages = make_cache(rng, 1, 4, 128, [950, 50, 400])
    off = gpu(np.array([0, 12, 52, 53], np.int32))
    par, ln = gpu(np.concatenate(trees)), gpu(np.array(lens, np.int32))
    q = torch.randn(53, 16, 128, device="cuda")
    cache = PagedKV(gpu(kv), gpu(pages))
    first, lse1 = cache.tree_attention(q, ln, off, par, 40)
    for _ in range(5):
        again, lse2 = cache.tree_attention(q, ln, off, par, 40)
        assert torch.equal(first, again) and torch.equal(lse1, lse2)
    wide = torch.full((53, 16 * 128 + 32), 7.0, device="cuda")
    view = wide[:, :2048].view(53, 16, 128)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        cache.tree_attention(q, ln, off, par, 40, out=view)
    s.synchronize()
    assert torch.equal(view, first) and bool((wide[:, 2048:] == 7.0).all())
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out, lse = cache.tree_attention(q, ln, off, par, 40)
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, first) and torch.equal(lse, lse1)


@pytest.mark.parametrize("n", [1, 6, 40])
def test_tree_attention_long_sums_do_not_drift(n):
    """fp32 outputs over 20000 rows: no error that grows with the rows.  Queries, keys and probabilities keep 24 bits and
    a tile's sum is cut eight times at most at its full size, by 2^-24 of it on average half: 2^-22; scores' errors (as
    2^-24 of a sum of 128 products of size one, times the score's scale) stay below that.  Bound: 2^-20, where cutting
    every sum would leave over 2^-16."""
    import torch
    from hymt2_b200.kvcache import PagedKV
    torch.manual_seed(3)
    S, L, kvh, G, hd = 6, 20000, 2, 4, 128
    page_max = (L + n + 15) // 16
    kv = torch.randn(1, S * page_max, 2, 16, kvh, hd, device="cuda").to(torch.bfloat16)
    pages = torch.randperm(S * page_max, device="cuda").to(torch.int32).view(S, page_max)
    q = torch.randn(S * n, kvh * G, hd, device="cuda")
    off = gpu(np.arange(S + 1, dtype=np.int32) * n)
    par = np.tile(np.arange(-1, n - 1), S).astype(np.int32)
    out, lse = PagedKV(kv, pages).tree_attention(q, gpu(np.full(S, L, np.int32)), off, gpu(par), n)
    for s in (0, S - 1):
        x = kv[0, pages[s].long()].double()  # [pages][2][16][kvh][hd]
        k, v = (x[:, i].flatten(0, 1)[:L + n] for i in range(2))
        hide = torch.arange(L + n, device="cuda")[None] > L + torch.arange(n, device="cuda")[:, None]
        for h in range(kvh * G):
            y = (q[s * n:(s + 1) * n, h].double() @ k[:, h // G].T * hd ** -0.5).masked_fill(hide, -torch.inf)
            want = torch.softmax(y, -1) @ v[:, h // G]
            got = out[s * n:(s + 1) * n, h].double()
            assert float((got - want).norm() / want.norm()) < 2.0 ** -20
            assert float((lse[s * n:(s + 1) * n, h].double() - torch.logsumexp(y, -1)).abs().max()) < 2.0 ** -18


def test_no_wait_has_given_up():
    from hymt2_b200.device import load_library
    assert load_library().hyc_kvops_timeouts() == 0


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("n,L", [(3, 900), (40, 200), (40, 3000)])
def test_tree_attention_rows_of_16_byte_alignment(n, L, bf16):
    """Queries and outputs whose rows start at odd multiples of 16 bytes (split and unsplit columns, both forms)."""
    import torch
    rng = np.random.default_rng(n + L)
    kvh, G, hd = 2, 4, 128
    kv, pages = make_cache(rng, 1, kvh, hd, [L + n])
    par, w = random_tree(rng, n), kvh * G * hd
    dt = torch.bfloat16 if bf16 else torch.float32
    step = 8 if bf16 else 4  # 16 bytes
    q = torch.from_numpy(rng.standard_normal((n, w)).astype(np.float32)).to(dt)
    want, wlse = run_tree(kv, pages, 0, [L], [par], gpu(q).view(n, kvh * G, hd), n)
    room_q, room_o = (torch.zeros(n * (w + step) + step, dtype=dt, device="cuda")[step:].view(n, w + step)[:, :w] for _ in range(2))
    room_q.copy_(q)
    assert room_q.data_ptr() % 32 == 16 and room_o.data_ptr() % 32 == 16
    got, lse = run_tree(kv, pages, 0, [L], [par], room_q.view(n, kvh * G, hd), n, out=room_o.view(n, kvh * G, hd))
    assert np.array_equal(got, want) and np.array_equal(lse, wlse)


def test_operators_past_32_bit_offsets():
    """A cache of over 2^32 elements, used at its far end."""
    import torch
    from hymt2_b200.kvcache import PagedKV
    rng = np.random.default_rng(12)
    kvh, hd, n, L = 4, 128, 6, 150
    npages = (1 << 32) // (2 * PAGE * kvh * hd) + 64
    kv = torch.empty((1, npages, 2, PAGE, kvh, hd), dtype=torch.bfloat16, device="cuda")
    small, _ = make_cache(rng, 1, kvh, hd, [L + n])
    used = small.shape[1]
    pages = (npages - 1 - np.arange(10)[::-1]).astype(np.int32)[None]
    kv[:, npages - used:] = small.cuda()
    local = pages - (npages - used)
    par = random_tree(rng, n)
    q = torch.randn(n, 16, hd, device="cuda")
    cache = PagedKV(kv, gpu(pages))
    ln, off = gpu(np.array([L], np.int32)), gpu(np.array([0, n], np.int32))
    out, lse = cache.tree_attention(q, ln, off, gpu(par), n)
    want, wlse, tol, tlse = plain_tree(small, local, 0, [L], [par], q.cpu().numpy().astype(np.float64), 4, hd ** -0.5)
    assert (np.abs(out.cpu().numpy() - want) <= tol).all() and (np.abs(lse.cpu().numpy() - wlse) <= tlse).all()
    acc = torch.zeros(1, 1, kvh, 160, device="cuda")
    sel = gpu(np.arange(n, dtype=np.int32)[None])
    cache.add_weights(acc, q[None], lse[None], ln, gpu(np.array([n], np.int32)), sel)
    tok = gpu(np.arange(n, dtype=np.int32))
    nxt = torch.full((n,), -5, dtype=torch.int32, device="cuda")
    nxt[0] = n - 1  # the last node, made a child of node 0, is accepted
    par2 = par.copy()
    par2[n - 1] = 0
    lens2, acc_n, path, bonus = cache.tree_commit(ln, off, gpu(par2), tok, nxt, n)
    assert acc_n.tolist() == [2] and path[0, :2].tolist() == [0, n - 1]
    kv2 = kv[:, npages - used:].cpu()
    a, b = L + n - 1, L + 1
    assert torch.equal(kv2[0, local[0, b // PAGE], :, b % PAGE], small[0, local[0, a // PAGE], :, a % PAGE])
    dst = PagedKV(kv, gpu((npages - used - 1 - np.arange(4)).astype(np.int32)[None]))  # far pages of the same pool
    got_len, kept, w = cache.evict(dst, lens2, acc, 50, 2, 10)
    rows = kept[0, 0, 1].cpu().numpy()
    assert got_len.tolist() == [50] and (np.diff(rows) > 0).all()
    p = dst.pages[0].cpu().numpy()[np.arange(50) // PAGE]
    got = kv[0, gpu(p.astype(np.int64)), :, gpu(np.arange(50) % PAGE), 1].cpu()
    assert torch.equal(got, kv2[0, local[0, rows // PAGE], :, rows % PAGE, 1])


# ---------------------------------------------------------------- commit

def plain_commit(kv, pages, lens, trees, tok, nxt, forced):
    kv = kv.clone()
    t0, outs = 0, []
    for s, par in enumerate(trees):
        n, L = len(par), lens[s]
        path = []
        if n and forced is not None and forced[s]:
            path = list(range(n))
        elif n:
            path, cur = [0], 0
            while True:
                hit = [i for i in range(cur + 1, n) if par[i] == cur and tok[t0 + i] == nxt[t0 + cur]]
                if not hit:
                    break
                cur = hit[0]
                path.append(cur)
        for j, i in enumerate(path):
            kv[:, int(pages[s, (L + j) // PAGE]), :, (L + j) % PAGE] = kv[:, int(pages[s, (L + i) // PAGE]), :, (L + i) % PAGE]
        outs.append((L + len(path), len(path), [t0 + i for i in path], int(nxt[t0 + path[-1]]) if path else -1))
        t0 += n
    return kv, outs


@pytest.mark.parametrize("hd,kvh,layers", [(128, 4, 3), (64, 1, 1), (64, 3, 2)])
def test_tree_commit(hd, kvh, layers):
    import torch
    from hymt2_b200.kvcache import PagedKV
    rng = np.random.default_rng(hd + kvh)
    counts = [1, 0, 64, 33, 20, 12, 64, 7]
    lens = [0, 5, 13, 31, 16, 250, 1, 47]
    trees = [random_tree(rng, n) for n in counts]
    trees[6] = np.arange(-1, 63)  # a chain, wholly accepted below
    nt = sum(counts)
    off = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
    tok = rng.integers(0, 4, nt).astype(np.int32)   # few tokens: many matches, several equal children
    nxt = rng.integers(0, 4, nt).astype(np.int32)
    nxt[off[6]:off[7] - 1] = tok[off[6] + 1:off[7]]
    for forced in (None, np.array([0, 1, 0, 1, 0, 0, 0, 1], np.int32)):
        kv, pages = make_cache(rng, layers, kvh, hd, [L + n for L, n in zip(lens, counts)])
        want, outs = plain_commit(kv, pages, lens, trees, tok, nxt, forced)
        d = gpu(kv)
        cache = PagedKV(d, gpu(pages))
        ln, n, path, bonus = cache.tree_commit(gpu(np.array(lens, np.int32)), gpu(off), gpu(np.concatenate(trees).astype(np.int32)),
                                               gpu(tok), gpu(nxt), 64, forced=None if forced is None else gpu(forced))
        assert torch.equal(d.cpu(), want)
        for s, (l, c, p, b) in enumerate(outs):
            assert (ln[s], n[s], bonus[s]) == (l, c, b)
            assert path[s].tolist() == p + [-1] * (64 - c)
        assert max(c for _, c, _, _ in outs) == 64 and outs[6][1] == 64


# ---------------------------------------------------------------- weights

@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("hd,kvh,G,layers,maxq", [(128, 2, 4, 2, 9), (64, 3, 8, 1, 64), (128, 1, 1, 3, 33), (64, 2, 2, 1, 1), (128, 2, 8, 1, 64)])
def test_cache_weights(hd, kvh, G, layers, maxq, bf16):
    import torch
    from hymt2_b200.kvcache import PagedKV
    rng = np.random.default_rng(hd + G + maxq + bf16)
    lens = [0, 1, 127, 128, 300, 640, 50]
    nq = [maxq, 1, max(1, maxq // 2), maxq, 1, maxq, 0]
    S, R = len(lens), 720
    kv, pages = make_cache(rng, layers, kvh, hd, [R] * S, garbage=float("nan"))
    for s in range(S):  # rows behind the queries' own are stale
        for r in range(lens[s] + nq[s], R):
            kv[:, int(pages[s, r // PAGE]), :, r % PAGE] = float("nan")
    nt, heads = 80, kvh * G
    q = torch.from_numpy(rng.standard_normal((layers, nt, heads * hd + 16)).astype(np.float32)).to(torch.bfloat16 if bf16 else torch.float32)
    lse = torch.from_numpy((3.0 + rng.standard_normal((layers, nt, heads))).astype(np.float32))
    lse[:, 3] = float("inf")  # a query of no weight
    sel = rng.integers(0, nt, (S, maxq)).astype(np.int32)
    if maxq > 4:
        sel[3, 2] = -1
    sel[5, 0] = 3
    acc = torch.from_numpy(rng.random((layers, S, kvh, R)).astype(np.float32))
    acc[:, 5, :, 7] = float("inf")
    d = gpu(acc)
    cache = PagedKV(gpu(kv), gpu(pages))
    args = (gpu(q)[:, :, :heads * hd].view(layers, nt, heads, hd), gpu(lse), gpu(np.array(lens, np.int32)),
            gpu(np.array(nq, np.int32)), gpu(sel))
    cache.add_weights(d, *args)
    d2 = gpu(acc)
    cache.add_weights(d2, *args)
    assert torch.equal(d, d2)
    got, sc = d.cpu().numpy().astype(np.float64), hd ** -0.5
    qn = q[:, :, :heads * hd].reshape(layers, nt, heads, hd).double().numpy()
    for l in range(layers):
        for s in range(S):
            L, n = lens[s], nq[s]
            k, _ = rows_of(kv, pages, l, s, L + n)
            for h in range(kvh):
                want = acc[l, s, h].double().numpy().copy()
                want[L:L + n] = 0
                tol = np.full(R, 0.0)
                for j in range(n):
                    if sel[s, j] < 0:
                        continue
                    qq = qn[l, sel[s, j], h * G:(h + 1) * G]
                    x = sc * (k[:L + j + 1, h] @ qq.T)
                    ex = sc * (np.abs(k[:L + j + 1, h]) @ np.abs(qq.T)) * hd * 2.0 ** -23
                    e = lse[l, sel[s, j], h * G:(h + 1) * G].double().numpy()[None]
                    p = np.exp(x - e)
                    want[:L + j + 1] += p.sum(1)
                    tol[:L + j + 1] += (p * (1.1 * ex + 2.0 ** -20 + 2.0 ** -22 * (np.abs(x) + np.where(np.isinf(e), 0, np.abs(e))))).sum(1)
                tol += 2.0 ** -21 * np.where(np.isinf(want), 0, np.abs(want))
                g = got[l, s, h]
                assert np.array_equal(g[L + n:], acc[l, s, h, L + n:].numpy())
                f = np.isfinite(want)
                assert np.array_equal(g[~f], want[~f])
                assert (np.abs(g - want)[f] <= tol[f]).all(), (l, s, h, float((np.abs(g - want)[f] - tol[f]).max()))


def test_weights_of_attention_sum_to_the_queries():
    """The probabilities of n queries of G heads sum to n G over the rows (lse from tree_attention, a chain)."""
    import torch
    from hymt2_b200.kvcache import PagedKV
    rng = np.random.default_rng(4)
    L, n = 500, 11
    kv, pages = make_cache(rng, 1, 2, 128, [L + n])
    cache = PagedKV(gpu(kv), gpu(pages))
    q = torch.randn(n, 8, 128, device="cuda")
    ln, off = gpu(np.array([L], np.int32)), gpu(np.array([0, n], np.int32))
    _, lse = cache.tree_attention(q, ln, off, gpu(np.arange(-1, n - 1, dtype=np.int32)), n)
    acc = torch.zeros(1, 1, 2, 528, device="cuda")
    cache.add_weights(acc, q[None], lse[None], ln, gpu(np.array([n], np.int32)), gpu(np.arange(n, dtype=np.int32)[None]))
    got = acc.double().sum(-1).reshape(-1).tolist()
    # each of the 44 probability rows sums to 1 within the bound of lse and of its own terms (under 1e-4 each)
    assert all(abs(x - 4 * n) < 4 * n * 1e-4 for x in got), got


# ---------------------------------------------------------------- eviction

def plain_kept(a, n, budget, sinks, recent):
    if n <= budget:
        return np.arange(n)
    mid = np.where(np.isnan(a[sinks:n - recent]), -np.inf, a[sinks:n - recent]).astype(np.float64)
    top = np.argsort(-mid, kind="stable")[:budget - sinks - recent] + sinks
    return np.sort(np.concatenate([np.arange(sinks), top, np.arange(n - recent, n)]))


@pytest.mark.parametrize("hd,kvh", [(128, 2), (64, 3)])
@pytest.mark.parametrize("budget,sinks,recent", [(1, 0, 0), (1, 0, 1), (40, 4, 8), (64, 0, 0), (64, 30, 34), (513, 3, 100), (2000, 4, 4)])
def test_evict(hd, kvh, budget, sinks, recent):
    import torch
    from hymt2_b200.kvcache import PagedKV
    rng = np.random.default_rng(budget + hd)
    layers, lens = 2, [0, 1, budget, budget + 1, 700, 1030, 2047]
    S, R = len(lens), 2064
    kv, pages = make_cache(rng, layers, kvh, hd, [R] * S)
    acc = np.exp(3 * rng.standard_normal((layers, S, kvh, R))).astype(np.float32)
    acc[0] = np.round(acc[0])                              # many ties, zeros
    acc[1, 3, 0, :50] = np.nan
    acc[1, 4, 0, 10:30] = np.inf
    acc[1, 4, 1, 10:300] = -np.inf
    acc[1, 5] = 0.0                                        # all tied
    acc[1, 5, 0, ::2] = -0.0
    acc[1, 6, 0] = np.nan
    dkv, dpages = make_cache(rng, layers, kvh, hd, [budget] * S)
    src, dst = gpu(kv), gpu(dkv)
    a = PagedKV(src, gpu(pages))
    b = PagedKV(dst, gpu(dpages))
    ln, kept, w = a.evict(b, gpu(np.array(lens, np.int32)), gpu(acc), budget, sinks, recent)
    assert ln.tolist() == [min(n, budget) for n in lens]
    want = dkv.clone()
    kept, w = kept.cpu().numpy(), w.cpu().numpy()
    for l in range(layers):
        for s in range(S):
            for h in range(kvh):
                rows = plain_kept(acc[l, s, h], lens[s], budget, sinks, recent)
                m = len(rows)
                assert np.array_equal(kept[l, s, h, :m], rows), (l, s, h)
                assert (kept[l, s, h, m:] == -1).all() and (w[l, s, h, m:] == 0).all()
                assert np.array_equal(w[l, s, h, :m], acc[l, s, h, rows], equal_nan=True)
                j = np.arange(m)
                want[l, dpages[s, j // PAGE], :, j % PAGE, h] = kv[l, pages[s, rows // PAGE], :, rows % PAGE, h]
    assert torch.equal(dst.cpu(), want) and torch.equal(src.cpu(), kv)


# ---------------------------------------------------------------- refusals

def test_refusals():
    import ctypes as C

    import torch
    from hymt2_b200 import abi
    from hymt2_b200.device import BackendError, load_library
    from hymt2_b200.kvcache import PagedKV
    rng = np.random.default_rng(1)
    kv, pages = make_cache(rng, 2, 2, 64, [40, 40])
    kv, pages = gpu(kv), gpu(pages)
    cache = PagedKV(kv, pages)
    ln, off = gpu(np.array([20, 20], np.int32)), gpu(np.array([0, 2, 4], np.int32))
    par = gpu(np.array([-1, 0, -1, 0], np.int32))
    q = torch.randn(4, 8, 64, device="cuda")
    lse = torch.zeros(2, 4, 8, device="cuda")
    for bad in (kv.float(), kv[0], kv.transpose(4, 5), kv.cpu()):
        with pytest.raises(ValueError):
            PagedKV(bad, pages)
    for bad in (pages.long(), pages[0], pages.cpu(), pages.t()):
        with pytest.raises(ValueError):
            PagedKV(kv, bad)
    for kw in (dict(q=q.half()), dict(q=q[:, :, :32]), dict(q=q[:, :7]), dict(q=q.transpose(0, 1)), dict(q=q.cpu()),
               dict(lens=ln.long()), dict(lens=ln[:1]), dict(offsets=ln), dict(parent=par[:3]), dict(out=q[:2]),
               dict(lse=lse[0, :, :4])):
        with pytest.raises(ValueError):
            cache.tree_attention(**dict(dict(q=q, lens=ln, offsets=off, parent=par, max_nodes=2), **kw))
    for kw in (dict(max_nodes=0), dict(max_nodes=65), dict(layer=2), dict(layer=-1), dict(q=torch.randn(4, 6, 64, device="cuda")),
               dict(q=torch.randn(4 * 513 + 1, device="cuda")[1:].view(4, 513)[:, :512].view(4, 8, 64))):
        with pytest.raises(BackendError):
            cache.tree_attention(**dict(dict(q=q, lens=ln, offsets=off, parent=par, max_nodes=2), **kw))
    tok = gpu(np.zeros(4, np.int32))
    with pytest.raises(BackendError):
        cache.tree_commit(ln, off, par, tok, tok, 65)
    with pytest.raises(ValueError):
        cache.tree_commit(ln, off, par, tok, tok[:3], 4)
    acc = torch.zeros(2, 2, 2, 48, device="cuda")
    sel = gpu(np.zeros((2, 3), np.int32))
    q2 = torch.randn(2, 4, 8, 64, device="cuda")
    with pytest.raises(ValueError):
        cache.add_weights(acc[:1], q2, lse, ln, ln, sel)
    with pytest.raises(ValueError):
        cache.add_weights(acc, q2[:1], lse, ln, ln, sel)
    with pytest.raises(BackendError):
        cache.add_weights(acc, q2, lse, ln, ln, gpu(np.zeros((2, 65), np.int32)))
    dst = PagedKV(torch.zeros_like(kv), pages)
    one = PagedKV(torch.zeros_like(kv[:1]), pages)
    with pytest.raises(BackendError):
        cache.evict(one, ln, acc, 10, 0, 0)              # another number of layers
    with pytest.raises(BackendError):
        cache.evict(dst, ln, acc, 10, 6, 5)              # sinks + recent over the budget
    with pytest.raises(BackendError):
        cache.evict(dst, ln, acc, 49, 0, 0)              # no room in the destination
    with pytest.raises(ValueError):
        cache.evict(dst, ln, acc.double(), 10, 0, 0)
    with pytest.raises(ValueError):
        cache.evict(dst, ln, acc, 0, 0, 0)
    # the C entries themselves: null and misaligned arguments, aliased lengths, a view that is none
    lib, err = load_library(), C.create_string_buffer(256)
    assert lib.hyc_tree_attention(None, None, 0, 8, 2, 1, 1, 1, 16, 512, 0, 1.0, 16, 512, None, 16, 64, err, 256) == -1
    v = abi.KVView(kv.data_ptr() + 2, pages.data_ptr(), 2, 8, 2, 64, 2, 3)
    assert lib.hyc_tree_commit(None, C.byref(v), 4, ln.data_ptr(), off.data_ptr(), par.data_ptr(), tok.data_ptr(),
                               tok.data_ptr(), None, ln.data_ptr(), ln.data_ptr(), ln.data_ptr(), ln.data_ptr(), err, 256) == -1
    assert b"aligned" in err.value
    assert lib.hyc_tree_commit(None, cache._ref, 4, ln.data_ptr(), off.data_ptr(), par.data_ptr(), tok.data_ptr(),
                               tok.data_ptr(), None, ln.data_ptr(), tok.data_ptr(), tok.data_ptr(), tok.data_ptr(), err, 256) == -1
    assert b"d_len_out" in err.value
    assert lib.hyc_tree_commit(None, cache._ref, 4, ln.data_ptr(), off.data_ptr(), None, tok.data_ptr(), tok.data_ptr(), None,
                               off.data_ptr(), tok.data_ptr(), tok.data_ptr(), tok.data_ptr(), None, 0) == -1
    need = lib.hyc_tree_attention_ws(cache._ref, 8, 2)
    assert need > 0
    assert lib.hyc_tree_attention(None, cache._ref, 0, 8, 2, ln.data_ptr(), off.data_ptr(), par.data_ptr(), q.data_ptr(),
                                  512, 0, 1.0, q.data_ptr(), 512, None, q.data_ptr(), need - 1, err, 256) == -1
    assert b"scratch" in err.value


def test_no_tokens():
    """A batch whose every tree is empty, and one of no tokens at all."""
    import torch
    from hymt2_b200.kvcache import PagedKV
    rng = np.random.default_rng(1)
    kv, pages = make_cache(rng, 1, 2, 64, [40])
    cache = PagedKV(gpu(kv), gpu(pages))
    zero = gpu(np.zeros(1, np.int32))
    none = gpu(np.zeros(0, np.int32))
    out, lse = cache.tree_attention(torch.empty(0, 4, 64, device="cuda"), zero, gpu(np.zeros(2, np.int32)), none, 4)
    assert out.shape == (0, 4, 64) and lse.shape == (0, 4)
    q = torch.randn(3, 4, 64, device="cuda")
    keep = torch.full((3, 4, 64), 5.0, device="cuda")
    cache.tree_attention(q, zero, gpu(np.zeros(2, np.int32)), gpu(np.zeros(3, np.int32)), 4, out=keep)
    assert bool((keep == 5.0).all())  # tokens of no tree are not touched
