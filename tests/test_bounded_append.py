"""
append_kv with page bounds, without a GPU: the rows go out behind the upload of
their slots, by the slots that a captured graph keeps.
"""

from __future__ import annotations

import dataclasses

import pytest
import torch

from llm_serving_layer_amd import BlockAllocator, SequenceBlocks, backend

from ._host import host_backend
from ._util import grow_and_assemble


def step(bk, n=17):
    s = SequenceBlocks(BlockAllocator(bk.num_blocks, 16), seq_id=0)
    return grow_and_assemble([s], [n], 16)


def test_the_rows_wait_for_their_slots(monkeypatch):
    bk = host_backend(monkeypatch, page_bounds=True)
    meta, k = step(bk), torch.zeros((17, 8, 64), dtype=torch.float16)
    bk.append_kv(0, k, k, meta)
    order = bk._lib.calls = []
    monkeypatch.setattr(bk, "_enter", lambda p: order.append(("enter", p)) or 11)
    bk.append_kv(0, k, k, meta)
    assert [c[0] for c in order] == ["enter", "pkv_append_kv", "pkv_page_bounds"]
    assert order[0][1] is bk._rows
    assert order[1][1][-1] == order[2][1][-1] == 11, "on the stream that waited"


@pytest.mark.parametrize("tokens", [17, 5])       # with and without a page completed
def test_a_graph_keeps_the_slots_that_its_append_reads(tokens, monkeypatch):
    """Slots of another type than the kernel's: converted once, by the plan."""
    bk = host_backend(monkeypatch, page_bounds=True)
    meta, k = step(bk, tokens), torch.zeros((tokens, 8, 64), dtype=torch.float16)
    meta = dataclasses.replace(meta, slot_mapping=meta.slot_mapping.long(), host=None)
    bk.append_kv(0, k, k, meta)
    bk._slot_cache = None                          # (another meta's append came between)
    monkeypatch.setattr(backend, "_capturing", lambda: True)
    bk.append_kv(0, k, k, meta)
    slots = next(c for c in reversed(bk._lib.calls) if c[0] == "pkv_append_kv")[1][5]
    assert slots == bk._rows.slots.data_ptr() and any(p is bk._rows for p in bk._captured)
