"""A swapped sequence goes back only to a pool of its own geometry."""

from __future__ import annotations

import pytest

from llm_serving_layer_amd import BlockAllocator, FourBitBackend, KVSwapSpace, SequenceBlocks

from .test_gpu_fourbit import DEV

pytestmark = pytest.mark.gpu


def test_blocks_of_as_many_bytes_but_other_heads_are_refused():
    """8 heads of 64 and 4 of 128 take as many bytes and lie differently."""
    one = FourBitBackend(2, 8, 16, 8, 8, 64, device=DEV)
    two = FourBitBackend(2, 8, 16, 4, 4, 128, device=DEV)
    assert one.block_bytes() == two.block_bytes()
    alloc = BlockAllocator(8, 16)
    s, t = (SequenceBlocks(alloc, seq_id=i) for i in range(2))
    s.append(40)
    t.append(40)
    space = KVSwapSpace(one)
    h = space.swap_out("r", s)
    with pytest.raises(RuntimeError, match="KV heads"):
        KVSwapSpace(two).swap_in(h, t)
    space.swap_in(h, t)
    space.release(h)
