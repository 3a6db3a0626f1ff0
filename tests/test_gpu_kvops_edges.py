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
