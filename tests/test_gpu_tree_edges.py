"""Drafted token trees and the bounded cache on whole models, at the edges of what they promise (needs a B200)."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def _open(backend, synth, model_dir, slots, weights=False, nodes=64, max_tokens=128, slot_ctx=192):
    from hymt2_b200.device import DeviceModel
    dm = DeviceModel(synth.ensure("t_q4km", model_dir), backend, ctx=256)
    dm.batch_prepare(slots=slots, slot_ctx=slot_ctx, max_tokens=max_tokens, max_out=max_tokens)
    dm.tree_prepare(nodes, weights=weights)
    return dm


def _forward(dm, slots, tokens, parent, off):
    """hyc_tree_forward itself; every output array with room behind it."""
    a = [np.asarray(x, dtype=np.int32) for x in (tokens, parent, off)]
    acc, nxt = np.zeros(slots + 8, np.int32), np.zeros(slots + 8, np.int32)
    path = np.zeros((slots + 8, 64), np.int32)
    rc = dm.be.lib.hyc_tree_forward(dm.be.impl, a[0].ctypes.data, a[1].ctypes.data, a[2].ctypes.data, None, 0, acc.ctypes.data,
                                    path.ctypes.data, nxt.ctypes.data)
    return rc, acc[:slots]


def test_offsets_that_rise_past_the_tokens_and_fall(backend, synth, model_dir):
    """Only the last offset says how many nodes there are; one before it may not lie past it."""
    slots = 3
    dm = _open(backend, synth, model_dir, slots)
    try:
        tok, par = np.ones(1024), np.tile(np.arange(-1, 63), 16)
        for off in ([0, 64, 128, 5], [0, 64, 120, 119], [0, -3, 5, 8], [0, 65, 65, 65], [0, 2 ** 31 - 1, 0, 5], [0, 5, -2 ** 31, 8]):
            rc, _ = _forward(dm, slots, tok, par, np.array(off))
            assert rc == -1 and "offsets" in dm.be.error(), off
        assert [dm.tree_state(s)[:2] for s in range(slots)] == [(0, 0)] * 3
        rc, acc = _forward(dm, slots, tok, [-1, 0, -1, 0, 1], [0, 2, 2, 5])
        assert rc == 0 and acc[0] >= 1 and acc[1] == 0 and acc[2] >= 1   # the handle stays usable
    finally:
        dm.close()


def test_eviction_leaves_a_slot_that_is_being_fed(backend, synth, model_dir):
    """Slot 1's second prompt goes in in two parts with a cut of slot 0 between them, while its last sequence was long
    enough to be cut itself: its rows and ids are those of an undisturbed run.  A third slot, never opened, keeps its rows."""
    rng = np.random.default_rng(9)
    first, second, other = (rng.integers(0, 900, n).tolist() for n in (100, 60, 40))

    def run(evict):
        dm = _open(backend, synth, model_dir, slots=3, weights=True)
        feed = lambda s, ids, at=0: dm.batch_forward(ids, [s] * len(ids), list(range(at, at + len(ids))), [])
        try:
            for s in (0, 1):  # both hold 100 rows with weights of their last 20
                feed(s, first[:80])
                dm.tree_open(s, 80)
                dm.tree_forward({s: (first[80:], list(range(-1, 19)))}, 3, forced=[s])
            feed(2, other)
            feed(1, second[:31])
            if evict:
                dm.tree_evict(40, 2, 8)
                assert dm.tree_state(0)[:2] == (40, 100)
                assert dm.tree_state(1)[:2] == (100, 100)
            feed(1, second[31:-1], 31)
            dm.tree_open(1, len(second) - 1)
            if evict:
                dm.tree_evict(100, 2, 8)
            path, nxt = dm.tree_forward({1: ([second[-1]], [-1])}, 3)[1]
            return path, nxt, [dm.batch_kv(s, l, n) for s, n in ((1, 60), (2, 40)) for l in range(dm.hp.n_layer)]
        finally:
            dm.close()

    a, b = run(True), run(False)
    assert a[:2] == b[:2]
    for (ka, va), (kb, vb) in zip(a[2], b[2]):
        assert np.array_equal(ka, kb) and np.array_equal(va, vb)
        assert (ka != 0).any()


def test_a_slot_goes_on_after_a_cut(backend, synth, model_dir):
    """Cuts one after the other, the budget growing in between; a tree pass on a fed slot takes it as it is."""
    rng = np.random.default_rng(10)
    ids = rng.integers(0, 900, 120).tolist()
    dm = _open(backend, synth, model_dir, slots=2, weights=True)
    try:
        dm.batch_forward(ids[:90], [0] * 90, list(range(90)), [])
        dm.tree_open(0, 90)
        dm.tree_forward({0: (ids[90:], list(range(-1, 29)))}, 2, forced=[0])
        for budget in (100, 31, 60, 30):
            rows, pos, w = dm.tree_state(0, weights=True)
            kv = [dm.batch_kv(0, l, rows) for l in range(dm.hp.n_layer)]
            dm.tree_evict(budget, 1, 5)
            n, pos2, w2 = dm.tree_state(0, weights=True)
            assert n == min(rows, budget) and pos2 == pos
            hd = dm.hp.hdim
            for l in range(dm.hp.n_layer):
                k, v = dm.batch_kv(0, l, n)
                for h in range(dm.hp.kv_heads):
                    keep = np.arange(rows)
                    if rows > budget:
                        mid = np.argsort(-w[l, h, 1:rows - 5].astype(np.float64), kind="stable")[:budget - 6] + 1
                        keep = np.sort(np.concatenate([[0], mid, np.arange(rows - 5, rows)]))
                    c = slice(h * hd, (h + 1) * hd)
                    assert np.array_equal(k[:, c], kv[l][0][keep][:, c]) and np.array_equal(v[:, c], kv[l][1][keep][:, c])
                    assert np.array_equal(w2[l, h], w[l, h, keep])
            dm.tree_forward({0: ([5, 6, 7], [-1, 0, 1])}, 2, forced=[0])
        dm.batch_forward([1], [0], [3], [])
        rows = dm.tree_state(0)[0]
        dm.tree_evict(20, 1, 5)
        assert dm.tree_state(0)[0] == rows       # fed: left alone
        dm.tree_forward({0: ([5], [-1])}, 2)
        dm.tree_evict(20, 1, 5)
        assert dm.tree_state(0)[0] == 20
    finally:
        dm.close()


def test_the_server_empties_the_slots(backend, synth, model_dir):
    """hyc_serve puts its requests' rows where the drafted sequences' were, so nothing of those is left to go on from."""
    rng = np.random.default_rng(11)
    ids = rng.integers(0, 900, 40).tolist()
    dm = _open(backend, synth, model_dir, slots=2, weights=True)
    try:
        fresh = dm.tree_forward({0: ([ids[0]], [-1])}, 2)[0]
        dm.tree_open(0, 0)
        dm.batch_forward(ids[:-1], [0] * 39, list(range(39)), [])
        dm.tree_open(0, 39)
        dm.tree_forward({0: ([ids[-1]], [-1])}, 2)
        assert dm.tree_state(0)[:2] == (40, 40)
        dm.serve([rng.integers(0, 900, 20).tolist()], 4, 32)
        assert [dm.tree_state(s)[:2] for s in (0, 1)] == [(0, 0)] * 2
        assert dm.tree_forward({0: ([ids[0]], [-1])}, 2)[0] == fresh
        assert np.allclose(dm.tree_state(0, weights=True)[2].sum(-1), dm.hp.heads // dm.hp.kv_heads, rtol=1e-4)
    finally:
        dm.close()


def test_forced_nodes_are_a_chain(backend, synth, model_dir):
    """All of a forced slot's nodes become rows one after the other; two of one position would not be a sequence."""
    from hymt2_b200.device import BackendError
    dm = _open(backend, synth, model_dir, slots=2)
    try:
        for parents in ([-1, 0, 0], [-1, 0, 1, 1]):
            with pytest.raises(BackendError, match="chain"):
                dm.tree_forward({0: ([1] * len(parents), parents)}, 2, forced=[0])
        assert dm.tree_state(0)[:2] == (0, 0)
        assert dm.tree_forward({0: ([1, 2, 3], [-1, 0, 1]), 1: ([1, 2, 3], [-1, 0, 0])}, 2, forced=[0])[0][0] == [1, 2, 3]
    finally:
        dm.close()
