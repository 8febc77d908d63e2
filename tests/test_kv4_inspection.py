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


def filled(device):
    """A cache of several groups (in 4 bits, behind a window that has left pages behind, with kept first rows, in float32) with two sequences."""
    needs = NEEDS + [KVNeed(2, 64, 9, keep_first=3, bits=4)]
    c = SequenceCache(plan_cache(needs, [None] * len(needs)), n_slots=3, n_pages=40, page_size=4, dtype=torch.float32, device=device)
    g = torch.Generator().manual_seed(3)
    for st in c.storage.values():
        st.copy_(torch.randint(0, 256, st.shape, generator=g) if st.dtype == torch.uint8 else torch.randn(st.shape, generator=g))
    for gi, group in enumerate(c.plan.groups):
        if group.need.bits:                                      # numbers of sizes that rows have
            st, hd = c.storage[gi], group.need.head_dim
            numbers = torch.randn(st.shape[:-1] + (4 * 4,), generator=g).bfloat16().abs().contiguous().view(torch.uint8)
            st[..., 4 * hd:] = numbers.to(st.device)
    slots = [c.assign() for _ in range(3)]
    for n in (5, 1, 17, 9):
        c.reserve(slots[0], n)
        c.advance(slots[0], n)
    c.reserve(slots[2], 3)
    c.advance(slots[2], 3)
    return c, slots


def test_windows_and_empty_sequences():
    c, slots = filled("cpu")
    for s, n in zip(slots, (32, 0, 3)):
        for gi, rows in c.dump_slot(s).items():
            group = c.plan.groups[gi]
            assert rows.shape == (group.n_layers, 2, n, group.need.n_kv_heads, group.need.head_dim) and rows.dtype == torch.float32
            for blk, page in enumerate(c._seq[s].pages[gi]):
                here = rows[:, :, 4 * blk:4 * blk + 4]
                assert (page is None) == bool((here == 0).all()) or here.numel() == 0
    assert any(p is None for p in c._seq[slots[0]].pages[1]) and c._seq[slots[0]].pages[len(c.plan.groups) - 1][0] is not None


@pytest.mark.gpu
def test_a_cache_on_a_gpu_reads_its_rows_with_the_kernel():
    from mivi_v4_b200.ops import kernels as K
    here, slots = filled("cpu")
    there, _ = filled("cuda:0")
    for s in slots:
        before = K.launch_count()
        got, want = there.dump_slot(s), here.dump_slot(s)
        layers = sum(g.n_layers for g in there.plan.groups if g.need.bits)
        assert K.launch_count() - before == (layers if here._len[s] else 0)
        for gi in want:
            assert got[gi].is_cuda and torch.equal(got[gi].cpu(), want[gi]), gi
    K.check_device_errors()
