"""The build with index checks over the 4-bit cache's kernels: a page-table entry outside the declared bound is reported and never followed.  As in
test_debug_checks_gpu.py nothing here can fault even if a check were wrong: the page lies in memory that the test owns."""
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

SCRIPT = r'''
import sys
import torch
sys.path.insert(0, %(root)r)
from mivi_v4_b200.ops import kernels as K
from mivi_v4_b200.engine.step import Workspace
assert K.DEBUG_CHECKS
dev = "cuda:0"
ints = lambda v: torch.tensor(v, dtype=torch.int32, device=dev)

def flagged(what):
    try:
        K.check_device_errors()
    except K.KernelError as e:
        assert "outside its bounds" in str(e), str(e)
        return
    raise AssertionError(what + ": an index outside the declared bound went unreported")

nh, nkv, page = 4, 2, 16
bad, good = ints([[1, 6, 0, 0]]), ints([[1, 3, 0, 0]])
for hd in (64, 40):
    big = torch.zeros(8, nkv, page * (hd + 8), dtype=torch.uint8, device=dev)
    pool = big[:4]
    for dtype in (torch.float32, torch.bfloat16):
        big.zero_()
        qkv = torch.randn(1, (nh + 2 * nkv) * hd, device=dev)
        q = torch.empty(1, nh * hd, dtype=dtype, device=dev)
        K.kv4_prepare(qkv, None, None, 1e-5, None, False, ints([17]), ints([0]), bad, pool, q, nh, nkv, hd)
        flagged("kv4_prepare")
        assert float(q.float().abs().max()) > 0 and int(big.max()) == 0
        K.kv4_prepare(qkv, None, None, 1e-5, None, False, ints([17]), ints([0]), good, pool, q, nh, nkv, hd)
        K.check_device_errors()
        assert int(big[3].max()) > 0 and int(big[4:].max()) == 0
        k, v = torch.empty(2, 1, nkv, hd, dtype=dtype, device=dev).unbind(0)
        K.kv4_read(pool, bad, ints([17]), ints([0]), k, v, nkv, hd)
        flagged("kv4_read")
        for m in (1, 21):                                        # few tokens and many
            qs = torch.randn(m, nh * hd, device=dev).to(dtype)
            for table in (bad, good):
                K.attention_kv4(qs, pool, table, ints(list(range(21 - m, 21))), ints([0] * m), ints([0, m]), ints([21 - m]), torch.empty_like(qs),
                                nh, nkv, hd, 0.2, 0, Workspace(dev), [21 - m], [m])
                if table is bad:
                    flagged("attention_kv4 of %%d tokens, heads of %%d" %% (m, hd))
                else:
                    K.check_device_errors()
print("all reported")
'''


def test_pages_outside_the_pool_are_skipped_and_reported():
    env = dict(os.environ, MIVI_DEBUG_CHECKS="1")
    r = subprocess.run([sys.executable, "-c", SCRIPT % {"root": ROOT}], capture_output=True, text=True, env=env, timeout=600)
    assert r.returncode == 0 and "all reported" in r.stdout, r.stdout + r.stderr
