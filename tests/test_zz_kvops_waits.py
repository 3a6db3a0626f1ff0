"""What the KV-cache operators' bounded waits report (needs a B200)."""
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu

CHILD = """
import os, sys, tempfile
import numpy as np, torch
from hymt2_b200 import synth
from hymt2_b200.device import Backend, BackendError, DeviceModel
from hymt2_b200.kvcache import PagedKV
be = Backend(0)
dm = DeviceModel(synth.ensure("t_q4km", sys.argv[1]), be, ctx=128)
dm.batch_prepare(slots=1, slot_ctx=64, max_tokens=32, max_out=32)
dm.tree_prepare(8)
cache = PagedKV(torch.zeros(1, 4, 2, 16, 2, 64, dtype=torch.bfloat16, device="cuda"), torch.zeros(1, 4, dtype=torch.int32, device="cuda"))
assert dm.tree_forward({0: ([5], [-1])}, 1)[0][0] == [5]
cache.check_waits()
assert be.lib.hyc_kvops_wait_probe(0) == -1 and be.lib.hyc_kvops_wait_probe(2_000_000_000) == -1
assert be.lib.hyc_kvops_wait_probe(2_000_000) == 0 and be.lib.hyc_kvops_timeouts() == 1
for call in (cache.check_waits, lambda: dm.tree_forward({0: ([5], [-1])}, 1)):
    try:
        call()
    except BackendError as e:
        assert "timed out" in str(e), e
    else:
        raise AssertionError("not reported")
try:
    dm.tree_open(0, 1)
except BackendError:
    print("reported")
"""


def test_a_wait_that_gave_up_is_reported(model_dir):
    """In a process of its own: the probe's wait runs out after 2 ms, the context stays usable, and the next pass over
    drafted trees and PagedKV.check_waits say so; the handle then refuses work like after any failed launch."""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", CHILD, model_dir], cwd=root, capture_output=True, text=True, timeout=300,
                       env=dict(os.environ, PYTHONPATH=root))
    assert r.returncode == 0 and "reported" in r.stdout, r.stdout + r.stderr


def test_no_wait_has_given_up_in_this_session():
    from hymt2_b200.device import load_library
    assert load_library().hyc_kvops_timeouts() == 0
