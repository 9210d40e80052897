"""
Graphs of calls that run as ``attend`` does (``attend_shared`` of batches that
share too little), replayed after other metas were planned and run: each
replay gives the eager result.
"""

from __future__ import annotations

import pytest
import torch

from llm_serving_layer_amd import BlockAllocator, SequenceBlocks
from llm_serving_layer_amd.backend import MI355XBackend

from ._util import grow_and_assemble

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("counts", [[1] * 40, [1] * 20 + [30] + [1] * 19])
@pytest.mark.parametrize("scale", [0.125, -0.125])
@pytest.mark.parametrize("between", [False, True])
def test_a_batch_that_does_not_share_replays_among_other_plans(counts, scale, between):
    """Decodes and a mixed batch, some of whose sequences are cut; ``between``:
    another meta was planned between the eager call and the capture. The other
    meta's partials would lie where this one's arrival counters are in a workspace
    they shared."""
    print(f"captured {len(counts)} {scale} {between}", flush=True)
    bk = MI355XBackend(2, 3000, 16, 8, 32, 64, device=DEV)
    g = torch.Generator(device=DEV).manual_seed(3)
    bk._pool.copy_(torch.randn(bk._pool.shape, generator=g, device=DEV))
    alloc = BlockAllocator(3000, 16)
    seqs = [SequenceBlocks(alloc, seq_id=i) for i in range(40)]
    for i, s in enumerate(seqs):
        s.append(1 + 23 * i)
    meta = grow_and_assemble(seqs, counts, 16, device=DEV)
    long = SequenceBlocks(alloc, seq_id=99)
    long.append(9000)
    T = sum(counts)
    q, k, v = (torch.randn((2, T, h, 64), generator=g, device=DEV).half() for h in (32, 8, 8))
    q1 = torch.randn((1, 32, 64), generator=g, device=DEV).half()

    def step():
        out = []
        for l in range(2):
            bk.append_kv(l, k[l], v[l], meta)
            out.append(bk.attend_shared(q[l], l, scale, meta))
        return out

    def other():
        bk.attend(q1, 0, 0.125, grow_and_assemble([long], [1], 16, device=DEV))

    want = step()
    plain = [bk.attend(q[l], l, scale, meta) for l in range(2)]
    assert all(torch.equal(a, b) for a, b in zip(want, plain)), "as attend runs it"
    assert not bk._shared.n_tiles and (bk._planned.dec or bk._planned).n_slots > 0
    rows = bk._pool.clone()
    if between:
        other()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for i in range(3):
        other()
        bk.invalidate_plan()
        junk = [torch.full((1 << 18,), -1, dtype=torch.int32, device=DEV) for _ in range(64)]
        for l in range(2):
            got[l].zero_()
            for p in (bk.k_pool, bk.v_pool):   # the rows are appended again
                p[l].view(-1, 8, 64)[meta.slot_mapping.long()] = 0
        torch.cuda.synchronize()
        del junk
        graph.replay()
        torch.cuda.synchronize()
        for l in range(2):
            assert torch.equal(got[l], want[l]), f"replay {i} layer {l}"
        assert torch.equal(bk._pool, rows)
    now = step()
    assert all(torch.equal(a, b) for a, b in zip(now, want))
    bk.check_device_errors()
