"""
The rotated append, the choice of pages and shared prefixes together, as a
serving loop uses them: prompts in chunks, then decode steps over several
layers, blocks copied and swapped between; every step against 64 bits. And
what none of them does while a graph is captured: plan.
"""

from __future__ import annotations

import pytest
import torch

from llm_serving_layer_amd import BlockAllocator, KVSwapSpace, SequenceBlocks, backend
from llm_serving_layer_amd.backend import MI355XBackend

from ._ops64 import assert_within, attend64, chosen64
from ._util import grow_and_assemble
from .test_gpu_rotary import assert_turned, table_of

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


class Server:
    def __init__(self, n_heads, n_kv, d, dtype, layers=2, blocks=300):
        self.bk = MI355XBackend(layers, blocks, 16, n_kv, n_heads, d, device=DEV, dtype=dtype,
                                page_bounds=True)
        self.table = table_of(1000, d)
        self.g = torch.Generator(device=DEV).manual_seed(7)
        self.alloc = BlockAllocator(blocks, 16)
        self.alloc.allocate(blocks)
        self.alloc.free(torch.randperm(blocks, generator=self.g, device=DEV).tolist())
        self.seqs = []

    def rand(self, *shape):
        return torch.randn(shape, generator=self.g, device=DEV).to(self.bk.dtype)

    def new(self):
        s = SequenceBlocks(self.alloc, seq_id=len(self.seqs))
        self.seqs.append(s)
        return s

    def fork(self, s):
        """A sequence that begins with s's whole pages, and a copy of its last
        one where that is not full."""
        t, whole = self.new(), s.num_tokens // 16
        t.block_ids = list(s.block_ids[:whole])
        self.alloc.incref(t.block_ids)
        t.num_tokens = s.num_tokens
        if s.num_tokens % 16:
            t.block_ids += self.alloc.allocate(1)
            self.bk.copy_block(s.block_ids[whole], t.block_ids[whole])
        return t

    def rows(self, s, layer):
        ids = torch.tensor(s.block_ids, device=DEV)
        return [p[layer][ids] for p in (self.bk.k_pool, self.bk.v_pool)]

    def append(self, counts, layer, meta):
        bk, n = self.bk, sum(counts)
        qkv = self.rand(n, bk.n_heads + 2 * bk.n_kv_heads, bk.head_dim)
        q, k, v = qkv.split([bk.n_heads, bk.n_kv_heads, bk.n_kv_heads], dim=1)
        turned = bk.append_kv_rotated(layer, q, k, v, meta, self.table)
        slots = meta.slot_mapping.long()
        kp, vp = (p[layer].view(-1, bk.n_kv_heads, bk.head_dim) for p in (bk.k_pool, bk.v_pool))
        assert_turned(turned, q, meta.positions, self.table)
        assert_turned(kp[slots], k, meta.positions, self.table)
        assert torch.equal(vp[slots], v)
        return turned

    def step(self, counts):
        meta = grow_and_assemble(self.seqs, counts, 16, device=DEV)
        assert meta.host_arrays() is not None
        return meta

    def check(self, q, out, layer, pages=None, chosen=None):
        bk, i0 = self.bk, 0
        for i, s in enumerate(self.seqs):
            k, v = self.rows(s, layer)
            lists = [list(range(len(k)))] * bk.n_kv_heads
            if pages:
                lists = chosen64(q[i], k.amin(1), k.amax(1), len(k), pages)
                for h, w in enumerate(lists):
                    assert chosen[i, h].tolist()[:len(w)] == w, f"seq {i} head {h}"
            live = s.num_tokens - (len(k) - 1) * 16
            keys, values = ([x[w, :, h].flatten(0, 1)[:(len(w) - 1) * 16 + live]
                             for h, w in enumerate(lists)] for x in (k, v))
            assert_within(out[i], *attend64(q[i], keys, values, 0.125, bk.dtype),
                          label=f"layer {layer} seq {i}")


@pytest.mark.parametrize("n_heads, n_kv, d, dtype", [
    (32, 8, 64, torch.float16), (8, 2, 128, torch.bfloat16), (4, 2, 48, torch.float32)])
def test_prompts_forks_swaps_and_steps(n_heads, n_kv, d, dtype, monkeypatch):
    print(f"serving steps {n_heads}/{n_kv}/{d} {dtype}", flush=True)
    monkeypatch.setattr(backend, "SHARED_PART_BYTES", 0)
    monkeypatch.setattr(backend, "SHARED_LEAST_BYTES", 0)
    sv = Server(n_heads, n_kv, d, dtype)
    bk = sv.bk
    for _ in range(2):
        sv.new()
    for counts in ([100, 37], [77, 201], [1, 15]):       # chunks, one beside a single token
        meta = sv.step(counts)
        for layer in range(2):
            q = sv.append(counts, layer, meta)
            bk.attend(q, layer, 0.125, meta)
    for s in list(sv.seqs):
        for _ in range(3):
            sv.fork(s)
    n = len(sv.seqs)
    space = KVSwapSpace(bk)
    for i in range(20):                                  # past a page's end in every sequence
        if i == 7:
            handle, tokens = space.swap_out("a", sv.seqs[3]), sv.seqs[3].num_tokens
            sv.seqs[3].free()
            back = SequenceBlocks(sv.alloc, seq_id=3)    # all its pages its own now
            back.append(tokens)
            space.swap_in(handle, back)
            sv.seqs[3] = back
        meta = sv.step([1] * n)
        for layer in range(2):
            q = sv.append([1] * n, layer, meta)
            if i % 4 == 3:
                out, chosen = bk.attend_selected(q, layer, 0.125, meta, 6, return_pages=True)
                sv.check(q, out, layer, 6, chosen)
            out = bk.attend_shared(q, layer, 0.125, meta)
            if i % 4 == 1:
                sv.check(q, out, layer)
        if bk._fast_decode:
            assert bk._shared.n_tiles, "the shared kernel ran"
    bk.check_device_errors()


def test_nothing_plans_while_a_graph_is_captured():
    sv = Server(8, 2, 64, torch.float16, layers=1)
    for _ in range(3):
        sv.new()
    meta = sv.step([1] * 3)
    q, k, v = sv.rand(3, 8, 64), sv.rand(3, 2, 64), sv.rand(3, 2, 64)
    calls = (lambda: sv.bk.append_kv_rotated(0, q, k, v, meta, sv.table),
             lambda: sv.bk.append_kv(0, k, v, meta),
             lambda: sv.bk.attend_selected(q, 0, 0.125, meta, 4),
             lambda: sv.bk.attend_shared(q, 0, 0.125, meta))
    side = torch.zeros(8, device=DEV)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        side += 1
        for call in calls:
            with pytest.raises(RuntimeError, match="before a graph is captured"):
                call()
    graph.replay()
    want = [call() for call in calls]
    with torch.cuda.graph(graph := torch.cuda.CUDAGraph()):
        got = [call() for call in calls]
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert (a is None and b is None) or torch.equal(a, b)
