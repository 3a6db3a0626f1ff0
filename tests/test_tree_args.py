"""Arguments of DeviceModel's tree calls (CPU: the library is a stand-in)."""
import ctypes as C

import numpy as np
import pytest

from hymt2_b200.device import DeviceModel


class Lib:
    """hyc_tree_forward of an engine of `slots` slots: keeps node 0 of every tree; writes as many entries as the engine."""

    def __init__(self, slots, nodes):
        self.slots, self.nodes, self.calls = slots, nodes, 0

    def hyc_tree_forward(self, impl, tk, pa, off, forced, vocab_out, acc, path, nxt):
        self.calls += 1
        view = lambda p, n: np.ctypeslib.as_array((C.c_int * n).from_address(p))
        o = view(off, self.slots + 1)
        for s in range(self.slots):
            view(acc, self.slots)[s] = o[s + 1] > o[s]
            view(nxt, self.slots)[s] = 100 + s
            view(path, self.slots * self.nodes)[s * self.nodes] = o[s]
        return 0


def model(slots=3, nodes=8):
    dm = DeviceModel.__new__(DeviceModel)
    dm.be = type("Be", (), dict(lib=Lib(slots, nodes), impl=None))()
    dm.batch_slots, dm.tree_nodes, dm.vocab_out = slots, nodes, 1000
    return dm


def test_trees_of_some_slots():
    dm = model()
    got = dm.tree_forward({2: ([7, 8], [-1, 0]), 0: ([5], [-1])}, 3, forced=[2])
    assert got == {0: ([5], 100), 2: ([7], 102)}


@pytest.mark.parametrize("slots", [0, 1, 2, 4, 100])
def test_another_number_of_slots_than_the_engine_has(slots):
    """The engine writes an entry for each of its own slots, whatever the caller says."""
    dm = model()
    with pytest.raises(ValueError):
        dm.tree_forward({0: ([5], [-1])}, slots)
    assert dm.be.lib.calls == 0


@pytest.mark.parametrize("trees,forced", [({}, None), ({3: ([1], [-1])}, None), ({-1: ([1], [-1])}, None), ({0: ([1], [-1])}, [3]),
                                          ({0: ([1], [-1])}, [-1]), ({0: ([1, 2], [-1]), 1: ([1], [-1, 0])}, None)])
def test_slots_and_trees_that_do_not_fit(trees, forced):
    dm = model()
    with pytest.raises(ValueError):
        dm.tree_forward(trees, 3, forced=forced)
    assert dm.be.lib.calls == 0
