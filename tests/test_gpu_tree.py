"""Drafted token trees and the bounded cache on whole models (needs a B200).

The ids of a pass over drafted trees are those of the plain greedy loop
(reference src/model.c:943-954), whatever was drafted; the prompts are those of
the greedy tests whose top two logits lie apart at every step.
"""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

PROMPTS = {"t_q4km": 25, "t_q2c": 1}


def _open(backend, synth, model_dir, cfg, slots, weights, nodes=64, max_tokens=128, ctx=256):
    from hymt2_b200.device import DeviceModel
    dm = DeviceModel(synth.ensure(cfg, model_dir), backend, ctx=ctx)
    dm.batch_prepare(slots=slots, slot_ctx=192, max_tokens=max_tokens, max_out=max_tokens)
    dm.tree_prepare(nodes, weights=weights)
    return dm


def _want(oracle, synth, model_dir, cfg, ids, n):
    import oracle as O
    om = O.OracleModel(oracle, synth.ensure(cfg, model_dir), ctx=256)
    try:
        return om.greedy(ids, n, chunk=16)[0]
    finally:
        om.close()


def _prompt(cfg):
    return np.random.default_rng(PROMPTS[cfg]).integers(0, 1000, 12).tolist()


@pytest.mark.parametrize("budget", [0, 150])
@pytest.mark.parametrize("cfg", ["t_q4km", "t_q2c"])
def test_drafted_ids_are_the_greedy_ids(backend, oracle, synth, model_dir, cfg, budget):
    """No guesses, guesses by repetition, a perfect chain, and trees in which the right path hides among wrong tokens:
    always the ids of the plain loop, in fewer passes where the guesses are right."""
    from hymt2_b200.draft import PromptLookup, generate
    ids = _prompt(cfg)
    want = _want(oracle, synth, model_dir, cfg, ids, 6)
    seq = ids + want
    rng = np.random.default_rng(3)

    def perfect(got):
        rest = seq[len(got):]
        return [got[-1]] + rest, list(range(-1, len(rest)))

    def hidden(got):
        tokens, parents, node = [got[-1]], [-1], 0
        for t in seq[len(got):]:
            for _ in range(3):  # wrong siblings, some with children of their own
                tokens.append(int(1000 + rng.integers(0, 5)) % 999 if rng.random() < 0.5 else int(rng.integers(0, 999)))
                parents.append(int(rng.integers(max(0, node - 2), node + 1)))
            tokens.append(t)
            parents.append(node)
            node = len(tokens) - 1
        return tokens, parents

    dm = _open(backend, synth, model_dir, cfg, slots=2, weights=budget > 0)
    try:
        for draft, most in ((lambda got: ([got[-1]], [-1]), 6), (PromptLookup(nodes=24), 6), (perfect, 1), (hidden, 6)):
            out, st = generate(dm, [ids, ids[:]], 6, draft, budget=budget)
            assert out == [want, want], (cfg, out, want)
            assert st.passes <= most and st.evictions == 0
            assert st.rows[0] >= len(ids) + 5 - 1
    finally:
        dm.close()


def test_stop_ids_end_a_slot(backend, oracle, synth, model_dir):
    from hymt2_b200.draft import generate
    ids = _prompt("t_q4km")
    want = _want(oracle, synth, model_dir, "t_q4km", ids, 6)
    dm = _open(backend, synth, model_dir, "t_q4km", slots=1, weights=False)
    try:
        out, _ = generate(dm, [ids], 6, stop=[want[3]])
        assert out == [want[:want.index(want[3])]]
    finally:
        dm.close()


def test_accepted_rows_follow_the_cache(backend, synth, model_dir):
    """After a pass that keeps a path from inside a tree, the slot's rows are those of the same tokens fed one after the
    other (projections of other batch sizes sum in another order: bf16 rows within two units of the last place)."""
    cfg, n0 = "t_q4km", 30
    rng = np.random.default_rng(8)
    ids = rng.integers(0, 900, n0).tolist()
    dm = _open(backend, synth, model_dir, cfg, slots=2, weights=False)
    try:
        dm.batch_forward(ids[:-1], [0] * (n0 - 1), list(range(n0 - 1)), [])
        dm.tree_open(0, n0 - 1)
        first = dm.tree_forward({0: ([ids[-1]], [-1])}, 2)[0]
        assert first[0] == [ids[-1]]
        nxt = first[1]
        # second pass: nxt, two wrong nodes, then the model's own continuation found by a probe on slot 1
        dm.batch_forward(ids + [nxt], [1] * (n0 + 1), list(range(n0 + 1)), [])
        dm.tree_open(1, n0)
        after = dm.tree_forward({1: ([nxt], [-1])}, 2)[1][1]
        wrong = (after + 1) % 900
        path, _ = dm.tree_forward({0: ([nxt, wrong, wrong, after, wrong], [-1, 0, 1, 0, 3])}, 2)[0]
        assert path == [nxt, after]
        rows, pos, _ = dm.tree_state(0)
        assert (rows, pos) == (n0 + 2, n0 + 2)
        dm.tree_open(1, 0)
        seq = ids + path
        dm.batch_forward(seq, [1] * len(seq), list(range(len(seq))), [])
        for layer in range(dm.hp.n_layer):
            for a, b in zip(dm.batch_kv(0, layer, rows), dm.batch_kv(1, layer, rows)):
                x, y = ((v.astype(np.uint32) << 16).view(np.float32) for v in (a, b))
                # layer 0 depends on the token alone; later layers also on the attention's sums
                assert np.abs(x - y).max() <= 2 * 2.0 ** -8 * np.abs(y).max(), layer
    finally:
        dm.close()


def test_weights_count_every_kept_query(backend, synth, model_dir):
    """Each counted query's probabilities sum to one per head: a slot's weights sum to (heads of a group) x queries."""
    from hymt2_b200.draft import generate
    rng = np.random.default_rng(5)
    dm = _open(backend, synth, model_dir, "t_q4km", slots=2, weights=True)
    try:
        prompts = [rng.integers(0, 900, 50).tolist(), rng.integers(0, 900, 90).tolist()]
        generate(dm, prompts, 9, budget=190, window=16)
        for s, p in enumerate(prompts):
            rows, pos, w = dm.tree_state(s, weights=True)
            counted = rows - (len(p) - 1 - 16)
            assert rows == pos and counted >= 16 + 9 - 1
            G = dm.hp.heads // dm.hp.kv_heads
            assert np.allclose(w.sum(-1), G * counted, rtol=1e-4) and (w >= 0).all()
    finally:
        dm.close()


def test_eviction_keeps_the_heaviest_rows_and_decoding_goes_on(backend, synth, model_dir):
    from hymt2_b200.draft import generate
    rng = np.random.default_rng(6)
    dm = _open(backend, synth, model_dir, "t_q4km", slots=3, weights=True)
    try:
        prompts = [rng.integers(0, 900, n).tolist() for n in (120, 40, 100)]
        generate(dm, prompts, 1, budget=190, window=32)
        before = [(dm.tree_state(s, weights=True), [dm.batch_kv(s, l, dm.tree_state(s)[0]) for l in range(dm.hp.n_layer)]) for s in range(3)]
        budget, sinks, recent, hd = 64, 3, 10, dm.hp.hdim
        dm.tree_evict(budget, sinks, recent)
        for s in range(3):
            (n, pos, w), kv = before[s]
            rows, pos2, w2 = dm.tree_state(s, weights=True)
            assert pos2 == pos and rows == min(n, budget)
            for l in range(dm.hp.n_layer):
                k, v = dm.batch_kv(s, l, rows)
                for h in range(dm.hp.kv_heads):
                    if n <= budget:
                        keep = np.arange(n)
                    else:
                        mid = np.argsort(-w[l, h, sinks:n - recent].astype(np.float64), kind="stable")[:budget - sinks - recent] + sinks
                        keep = np.sort(np.concatenate([np.arange(sinks), mid, np.arange(n - recent, n)]))
                    c = slice(h * hd, (h + 1) * hd)
                    assert np.array_equal(k[:, c], kv[l][0][keep][:, c]) and np.array_equal(v[:, c], kv[l][1][keep][:, c])
                    assert np.array_equal(w2[l, h], w[l, h, keep])
        out, st = generate(dm, prompts, 12, budget=70, recent=20)
        assert [len(o) for o in out] == [12, 12, 12] and st.evictions >= 1
        assert all(dm.tree_state(s)[1] >= len(prompts[s]) + 11 for s in range(3))
    finally:
        dm.close()


def test_refusals(backend, synth, model_dir):
    from hymt2_b200.device import BackendError, DeviceModel
    dm = DeviceModel(synth.ensure("t_q4km", model_dir), backend, ctx=256)
    try:
        dm.batch_prepare(slots=2, slot_ctx=64, max_tokens=32, max_out=2)
        with pytest.raises(BackendError):
            dm.tree_prepare(64)                 # fewer head rows than nodes
        dm.batch_prepare(slots=2, slot_ctx=64, max_tokens=32, max_out=32)
        for n in (0, 65):
            with pytest.raises(BackendError):
                dm.tree_prepare(n)
        dm.tree_prepare(8)
        with pytest.raises(BackendError):
            dm.tree_open(2, 0)
        with pytest.raises(BackendError):
            dm.tree_open(0, 65)
        dm.tree_open(0, 60)
        for tree in (([1] * 9, list(range(-1, 8))), ([1] * 5, list(range(-1, 4))), ([1, 2], [-1, 1]), ([1, 2], [-1, -1]), ([1], [0])):
            with pytest.raises(BackendError):
                dm.tree_forward({0: tree}, 2)   # too many nodes, no room, a parent that is not below, two roots
        with pytest.raises(BackendError):
            dm.tree_evict(8, 0, 0)              # no weights kept
        with pytest.raises(BackendError):
            dm.tree_state(0, weights=True)
        assert dm.tree_state(0)[:2] == (60, 60)
        assert dm.tree_forward({1: ([5], [-1])}, 2)[1][0] == [5]   # the handle stays usable
    finally:
        dm.close()
