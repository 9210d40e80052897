"""
Which positions a rotated append is checked against on the host: those that it
rotates by, as far as the meta's mirror holds them.
"""

from __future__ import annotations

import dataclasses

import numpy as np
import pytest
import torch

from llm_serving_layer_amd import BlockAllocator, RotaryTable, SequenceBlocks
from llm_serving_layer_amd.stepping import DecodeStepper

from ._host import STREAM, host_backend
from ._util import grow_and_assemble, make_meta, meta_to_device


def sequences(lens):
    alloc = BlockAllocator(512, 16)
    seqs = [SequenceBlocks(alloc, seq_id=i) for i in range(len(lens))]
    for s, n in zip(seqs, lens):
        s.append(n)
    return seqs


def append(bk, meta, table):
    T = meta.n_tokens
    q, k = (torch.zeros((T, h, 64), dtype=torch.float16) for h in (32, 8))
    table.stream = STREAM
    return bk.append_kv_rotated(0, q, k, k, meta, table)


def test_positions_set_anew_are_not_taken_for_the_lengths(monkeypatch):
    """A sequence of 41 tokens whose new one is rotated as position 3: the table
    of 8 positions has it."""
    bk = host_backend(monkeypatch)
    meta = grow_and_assemble(sequences([40]), [1], 16)
    table = RotaryTable(8, 64, device="cpu")
    with pytest.raises(ValueError, match="position 40"):
        append(bk, meta, table)
    near = dataclasses.replace(meta, positions=torch.tensor([3]))
    assert near.host_arrays() is not None and near.host_positions() is None
    append(bk, near, table)
    assert [c[0] for c in bk._lib.calls] == ["pkv_append_rotated_batch"]


def test_a_sequence_without_new_tokens_is_not_asked_for_its_length(monkeypatch):
    """Only the tokens of this step are rotated."""
    bk = host_backend(monkeypatch)
    meta = grow_and_assemble(sequences([40, 2]), [1, 1], 16)
    skipped = dataclasses.replace(
        meta, query_lens=torch.tensor([0, 1], dtype=torch.int32),
        cu_query_lens=torch.tensor([0, 0, 1], dtype=torch.int32), positions=meta.positions[1:],
        batch_indices=meta.batch_indices[1:], slot_mapping=meta.slot_mapping[1:])
    skipped = meta_to_device(skipped, "cpu")
    skipped = dataclasses.replace(skipped, host=dataclasses.replace(
        skipped.host, positions=(skipped.positions, skipped.positions.numpy())))
    append(bk, skipped, RotaryTable(8, 64, device="cpu"))


@pytest.mark.parametrize("bad", [-1, 8])
def test_a_position_outside_is_refused(bad, monkeypatch):
    bk = host_backend(monkeypatch)
    meta = grow_and_assemble(sequences([3]), [2], 16)
    pos = torch.tensor([2, bad])
    meta = dataclasses.replace(meta, positions=pos,
                               host=dataclasses.replace(meta.host, positions=(pos, pos.numpy())))
    with pytest.raises(ValueError, match=f"position {bad} is outside"):
        append(bk, meta, RotaryTable(8, 64, device="cpu"))


def test_assembled_metas_hold_their_positions():
    meta = grow_and_assemble(sequences([40, 3]), [1, 5], 16)
    assert np.array_equal(meta.host_positions(), meta.positions.numpy())
    stepper = DecodeStepper(sequences([15, 3]), "cpu", 16)
    for _ in range(3):
        meta = stepper.step()
        assert np.array_equal(meta.host_positions(), meta.positions.numpy())
    assert make_meta(sequences([4]), [4], 16).host_positions() is None
