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
