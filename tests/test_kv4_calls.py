"""Calls of the 4-bit cache's operators that have to be refused, or taken, before a GPU sees them."""
import numpy as np
import pytest
import torch

from mivi_v4_b200.ops import kernels as K
from mivi_v4_b200.ops.kernels import KernelError


def ints(v):
    return torch.tensor(v, dtype=torch.int32)


def attend(**over):
    a = dict(q=torch.zeros(3, 64), pool=torch.zeros(5, 2, 4 * 24, dtype=torch.uint8), page_table=ints([[1, 2]]), positions=ints([0, 1, 2]),
             seq_of=ints([0, 0, 0]), cu=ints([0, 3]), starts=ints([0]), out=torch.zeros(3, 64), nh=4, nkv=2, hd=16, scale=0.25, window=0, ws=None,
             host_starts=[0], host_lens=[3])
    return K.attention_kv4(**{**a, **over})


def test_sequences_begin_at_0_or_later():
    """A negative position would be looked up in front of the page table."""
    with pytest.raises(KernelError, match="position 0 or later"):
        attend(host_starts=[-1])
    with pytest.raises(KernelError, match="position 0 or later"):
        attend(host_starts=[5, -64], host_lens=[1, 2])


@pytest.mark.gpu
def test_starts_and_lengths_may_be_arrays():
    """One sequence near the page table's end and another that brings many tokens: together more than the table's width, each within it."""
    from mivi_v4_b200.engine import Workspace
    dev, hd, page = "cuda:0", 64, 64
    g = torch.Generator().manual_seed(1)
    pool = torch.randint(0, 16, (4, 1, page * (hd + 8)), generator=g, dtype=torch.uint8).to(dev)
    pool[:, :, page * hd:] = torch.ones(4, 1, page * 4, dtype=torch.bfloat16).view(torch.uint8).to(dev)
    starts, lens = [0, 120], [10, 2]
    q = torch.randn(12, 2 * hd, generator=g).to(dev, torch.bfloat16)
    a = dict(q=q, pool=pool, page_table=ints([[0, 1], [2, 3]]).to(dev), positions=ints([*range(10), 120, 121]).to(dev), seq_of=ints([0] * 10 + [1] * 2).to(dev),
             cu=ints([0, 10, 12]).to(dev), starts=ints(starts).to(dev), nh=2, nkv=1, hd=hd, scale=0.125, window=0, ws=Workspace(dev))
    want, got = torch.empty_like(q), torch.empty_like(q)
    K.attention_kv4(**a, out=want, host_starts=starts, host_lens=lens)
    K.attention_kv4(**a, out=got, host_starts=np.array(starts), host_lens=np.array(lens))
    assert torch.equal(want, got) and torch.isfinite(got).all()
    with pytest.raises(KernelError, match="reaches 128"):
        K.attention_kv4(**a, out=got, host_starts=np.array([0, 127]), host_lens=np.array(lens))
