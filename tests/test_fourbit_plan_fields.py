"""A meta whose index fields disagree in length is refused before the planner reads
them."""

from __future__ import annotations

import dataclasses

import pytest
import torch

from llm_serving_layer_amd import BlockAllocator, SequenceBlocks, backend

from ._util import grow_and_assemble
from .test_fourbit import host_backend


@pytest.mark.parametrize("field,keep", [
    ("cu_query_lens", slice(None, -1)), ("cu_query_lens", slice(1, 1)), ("kv_lens", slice(None, 2)),
    ("kv_lens", slice(0, 1)), ("kv_indptr", slice(None, 3)), ("kv_last_page_len", slice(0, 1)),
    ("query_lens", slice(0, 2))])
def test_fields_of_other_lengths(field, keep, monkeypatch):
    monkeypatch.setattr(backend, "_capturing", lambda: False)
    alloc = BlockAllocator(8, 16)
    meta = grow_and_assemble([SequenceBlocks(alloc, seq_id=i) for i in range(3)], [4, 1, 3], 16)
    meta = dataclasses.replace(meta, **{field: getattr(meta, field)[keep]})
    with pytest.raises(ValueError, match="entries for"):
        host_backend()._plan(meta)
