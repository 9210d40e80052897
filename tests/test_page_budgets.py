"""
attend_selected with several budgets in a step, without a GPU: each is planned
once a meta, and all of them can be captured.
"""

from __future__ import annotations

import pytest
import torch

from llm_serving_layer_amd import BlockAllocator, SequenceBlocks, backend

from ._host import host_backend
from ._util import grow_and_assemble


def test_layers_with_budgets_of_their_own(monkeypatch):
    bk = host_backend(monkeypatch, page_bounds=True, layers=4)
    alloc = BlockAllocator(bk.num_blocks, 16)
    seqs = [SequenceBlocks(alloc, seq_id=i) for i in range(3)]
    for s in seqs:
        s.append(600)
    q = torch.zeros((3, 32, 64), dtype=torch.float16)

    def step(meta):
        for l in range(4):
            bk.attend_selected(q, l, 0.125, meta, [8, 20][l % 2])
        return [bytes(c[2]) for c in bk._lib.calls[-4:]]

    meta = grow_and_assemble(seqs, [1] * 3, 16)
    first = step(meta)
    assert bk.n_plans == 2 and first[0] == first[2] != first[1] == first[3]
    monkeypatch.setattr(backend, "_capturing", lambda: True)
    assert step(meta) == first and bk.n_plans == 2
    assert {p.asked for p in bk._captured} == {8, 20}
    with pytest.raises(RuntimeError, match="before a graph is captured"):
        bk.attend_selected(q, 0, 0.125, meta, 9)
    monkeypatch.setattr(backend, "_capturing", lambda: False)
    step(grow_and_assemble(seqs, [1] * 3, 16))
    assert bk.n_plans == 4 and len(bk._budgets) == 2, "the step before's are let go"
    bk.invalidate_plan()
    assert not bk._budgets
