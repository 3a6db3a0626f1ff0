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
