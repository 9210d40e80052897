"""
The rotation table's memory on streams other than its own, without a GPU: each
that a launch reads it on is recorded, so that a dropped table's memory is not
used again before.
"""

from __future__ import annotations

import torch

from llm_serving_layer_amd import BlockAllocator, RotaryTable, SequenceBlocks, backend

from . import _host
from ._host import host_backend
from ._util import grow_and_assemble


class Rows:
    """A table's tensor that notes the streams recorded."""

    def __init__(self, t):
        self.t, self.streams = t, []

    def data_ptr(self):
        return self.t.data_ptr()

    def record_stream(self, stream):
        self.streams.append(stream)


def test_a_table_of_another_stream_is_recorded(monkeypatch):
    monkeypatch.setattr(torch.cuda, "current_stream", lambda device: "current")
    bk = host_backend(monkeypatch)
    s = SequenceBlocks(BlockAllocator(64, 16), seq_id=0)
    meta = grow_and_assemble([s], [5], 16)
    q, k = (torch.zeros((5, h, 64), dtype=torch.float16) for h in (32, 8))
    own, other = RotaryTable(8, 64, device="cpu"), RotaryTable(8, 64, device="cpu")
    own.stream, other.stream = _host.STREAM, 99
    for table in (own, other):
        table.table = Rows(table.table)
        bk.append_kv_rotated(0, q, k, k, meta, table)
        assert any(t is table.table for t in bk._rows.buffers), "another stream records it"
    assert own.table.streams == [] and other.table.streams == ["current"]
    kept = RotaryTable(8, 64, device="cpu")
    kept.stream, kept.table = 99, Rows(kept.table)
    monkeypatch.setattr(backend, "_capturing", lambda: True)
    bk.append_kv_rotated(0, q, k, k, meta, kept)   # (a graph keeps the table itself)
    assert bk._captured[-1].table is kept and kept.table.streams == []
