"""What a 4-bit cache says that it holds."""
import pytest
import torch

import plain_kv4 as Q
from mivi_v4_b200.cache import KVNeed, SequenceCache, plan_cache
from mivi_v4_b200.cache.cache import rows_of_4_bits

NEEDS = [KVNeed(2, 64, bits=4), KVNeed(2, 64, bits=4), KVNeed(2, 64, 9, bits=4), KVNeed(2, 64), KVNeed(1, 40, bits=4)]


def test_rows_whose_span_is_beyond_the_largest_float():
    """15 steps may pass the largest float32 where the row's ends do not."""
    k = torch.linspace(-3e38, 3e38, 64, dtype=torch.float64).float().view(1, 1, 1, 64)
    assert torch.isfinite(k).all()
    pool = Q.pool_bytes(k, -k)
    wk, wv = Q.rows_of(pool, 1, 64)
    got = rows_of_4_bits(pool, 1, 64)
    assert torch.equal(got[:, 0], wk.float()) and torch.equal(got[:, 1], wv.float()) and torch.isfinite(got).all()
