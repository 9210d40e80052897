"""``verify_drafts`` without a GPU: a meta whose fields the kernels would read past
their ends is refused."""

from __future__ import annotations

import dataclasses

import pytest
import torch

from llm_serving_layer_amd import BlockAllocator, SequenceBlocks, sampling
from llm_serving_layer_amd.sampling import _step_lengths

from ._util import grow_and_assemble


@pytest.fixture(autouse=True)
def nothing_is_captured(monkeypatch):
    monkeypatch.setattr(sampling, "_capturing", lambda: False)


def step():
    alloc = BlockAllocator(8, 16)
    return grow_and_assemble([SequenceBlocks(alloc, seq_id=i) for i in range(3)], [4, 1, 3], 16)


@pytest.mark.parametrize("mirror", [True, False])
def test_lengths_of_a_step(mirror):
    meta = step() if mirror else dataclasses.replace(step(), host=None)
    assert _step_lengths(meta, 8) == [4, 1, 3]


@pytest.mark.parametrize("change,match", [
    ({"batch_indices": torch.zeros(7, dtype=torch.int32)}, "batch_indices"),
    ({"batch_indices": torch.zeros(0, dtype=torch.int32)}, "batch_indices"),
    ({"batch_indices": torch.zeros((8, 1), dtype=torch.int32)}, "batch_indices"),
    ({"cu_query_lens": torch.tensor([0, 4, 5], dtype=torch.int32)}, "cu_query_lens"),
    ({"cu_query_lens": torch.tensor([0, 4, 5, 7], dtype=torch.int32)}, "sums"),
    ({"query_lens": torch.tensor([5, 0, 3], dtype=torch.int32)}, "sums|make up"),
    ({"query_lens": torch.tensor([4, 4], dtype=torch.int32)}, "cu_query_lens")])
def test_lengths_that_do_not_fit_are_refused(change, match):
    with pytest.raises(ValueError, match=match):
        _step_lengths(dataclasses.replace(step(), **change), 8)
