"""Calls of the 4-bit cache's operators that have to be refused, or taken, before a GPU sees them."""
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
