"""
What the host does while a graph is captured, without a GPU: no plan is made
(what it uploads would be on the device only once the graph has run), what the
launches read is kept, and it is nobody else's to write.
"""

from __future__ import annotations

import pytest
import torch

from llm_serving_layer_amd import BlockAllocator, SequenceBlocks, backend

from ._host import host_backend
from ._util import grow_and_assemble


def batch(bk, lens, counts=None, alloc=None):
    alloc = alloc or BlockAllocator(bk.num_blocks, bk.block_size)
    seqs = [SequenceBlocks(alloc, seq_id=i) for i in range(len(lens))]
    for s, n in zip(seqs, lens):
        s.append(n)
    return grow_and_assemble(seqs, counts or [1] * len(lens), bk.block_size)


def rows(bk, meta, heads):
    return torch.zeros((meta.n_tokens, heads, bk.head_dim), dtype=bk.dtype)


@pytest.mark.parametrize("counts", [None, [1, 9, 1]])
@pytest.mark.parametrize("scale", [0.125, -0.125])
def test_a_batch_that_does_not_share_keeps_its_plan(counts, scale, monkeypatch):
    """attend_shared of a meta that it has seen, after another meta was planned:
    the first call's plan, kept, and a workspace that the other's does not touch."""
    bk = host_backend(monkeypatch)
    alloc = BlockAllocator(bk.num_blocks, 16)
    a, b = batch(bk, [700, 20, 400], counts, alloc), batch(bk, [3000], None, alloc)
    qa, qb = rows(bk, a, 32), rows(bk, b, 32)
    bk.attend_shared(qa, 0, scale, a)
    name, _, eager = bk._lib.calls[-1]
    assert name == "pkv_attend_batch" and eager.n_slots > 0, "a cut sequence"
    bk.attend(qb, 0, scale, b)
    plans = bk.n_plans
    monkeypatch.setattr(backend, "_capturing", lambda: True)
    monkeypatch.setattr(bk, "_upload", None)     # nothing is uploaded
    bk.attend_shared(qa, 0, scale, a)
    name, _, held = bk._lib.calls[-1]
    assert bk.n_plans == plans and held.workspace != bk._ws_ptr, "a workspace of the graph's"
    assert held.workspace and held.workspace_bytes < bk._ws_bytes
    for name, _ in held._fields_:
        if name not in ("workspace", "workspace_bytes"):
            assert getattr(held, name) == getattr(eager, name), name
    (p,) = bk._captured
    w, d = p.whole, p.whole.dec or p.whole
    kept = {t.data_ptr() for t in (w.plan, d.plan, w.indptr, w.indices, w.kv_lens, w.cu_q, w.bidx,
                                   w.slots)}
    assert {held.prefill_plan, held.decode_plan, held.kv_indptr, held.kv_indices, held.kv_lens,
            held.cu_query_lens, held.batch_indices, held.slot_mapping} == kept
    monkeypatch.setattr(backend, "_capturing", lambda: False)
    assert bk._planned.meta is b, "eager calls find what they planned"


def test_a_meta_not_seen_before_is_refused(monkeypatch):
    bk = host_backend(monkeypatch)
    a = batch(bk, [700, 20, 400])
    monkeypatch.setattr(backend, "_capturing", lambda: True)
    with pytest.raises(RuntimeError, match="before a graph is captured"):
        bk.attend_shared(rows(bk, a, 32), 0, 0.125, a)
    monkeypatch.setattr(backend, "_capturing", lambda: False)
    bk.attend(rows(bk, a, 32), 0, 0.125, a)      # attend's plan is not attend_shared's
    monkeypatch.setattr(backend, "_capturing", lambda: True)
    with pytest.raises(RuntimeError, match="before a graph is captured"):
        bk.attend_shared(rows(bk, a, 32), 0, 0.125, a)


def test_a_shared_batch_with_a_scale_not_seen_before_is_refused(monkeypatch):
    monkeypatch.setattr(backend, "SHARED_PART_BYTES", 0)
    monkeypatch.setattr(backend, "SHARED_LEAST_BYTES", 0)
    bk = host_backend(monkeypatch)
    alloc = BlockAllocator(bk.num_blocks, 16)
    head = alloc.allocate(20)
    seqs = []
    for i in range(3):
        s = SequenceBlocks(alloc, seq_id=i)
        alloc.incref(head)
        s.block_ids, s.num_tokens = list(head), 320
        seqs.append(s)
    alloc.free(head)
    a = grow_and_assemble(seqs, [1, 1, 1], 16)
    q = rows(bk, a, 32)
    bk.attend_shared(q, 0, 0.125, a)
    assert bk._lib.calls[-1][0] == "pkv_attend_shared_batch"
    monkeypatch.setattr(backend, "_capturing", lambda: True)
    bk.attend_shared(q, 0, 0.125, a)
    assert bk._lib.calls[-1][0] == "pkv_attend_shared_batch"
    with pytest.raises(RuntimeError, match="before a graph is captured"):
        bk.attend_shared(q, 0, -0.125, a)


def test_a_captured_append_plans_nothing_and_keeps_its_slots(monkeypatch):
    """append_kv then attend_shared in a graph, the meta's plan replaced by
    another's since: the rows are appended on their own, by slots that stay."""
    bk = host_backend(monkeypatch)
    alloc = BlockAllocator(bk.num_blocks, 16)
    a, b = batch(bk, [700, 20, 400], None, alloc), batch(bk, [3000], None, alloc)
    q, k = rows(bk, a, 32), rows(bk, a, 8)
    bk.append_kv(0, k, k, a)
    bk.attend_shared(q, 0, 0.125, a)
    assert bk._lib.calls[-1][1][6], "fused"
    bk.attend(rows(bk, b, 32), 0, 0.125, b)
    plans = bk.n_plans
    monkeypatch.setattr(backend, "_capturing", lambda: True)
    bk.append_kv(0, k, k, a)
    bk.attend_shared(q, 0, 0.125, a)
    names = [c[0] for c in bk._lib.calls[-2:]]
    assert names == ["pkv_append_kv", "pkv_attend_batch"] and bk.n_plans == plans
    slots = bk._lib.calls[-2][1][5]
    assert any(torch.is_tensor(t) and t.data_ptr() == slots for t in bk._captured)
    assert bk._slot_cache is None
    monkeypatch.setattr(backend, "_capturing", lambda: False)
    bk.append_kv(0, k, k, a)                       # eager again: planned, fused
    assert bk._planned.meta is a and bk._pending is not None


def test_an_append_that_a_captured_call_lands_keeps_its_slots(monkeypatch):
    """A deferred append of another layer, in slots that were converted for it."""
    import dataclasses

    bk = host_backend(monkeypatch, layers=2)
    a = batch(bk, [700, 20, 400])
    a = dataclasses.replace(a, slot_mapping=a.slot_mapping.long(), host=None)
    q, k = rows(bk, a, 32), rows(bk, a, 8)
    bk.append_kv(1, k, k, a)
    bk.attend_shared(q, 0, 0.125, a)
    monkeypatch.setattr(backend, "_capturing", lambda: True)
    bk.append_kv(1, k, k, a)
    bk.attend_shared(q, 0, 0.125, a)
    name, args, _ = bk._lib.calls[-2]
    assert name == "pkv_append_kv"
    assert any(torch.is_tensor(t) and t.data_ptr() == args[5] for t in bk._captured)
