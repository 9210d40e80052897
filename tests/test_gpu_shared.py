"""
Shared-prefix attention against attention in 64 bits and against ``attend``:
head layouts and types, one prefix and trees of them, two sequences to more
than a tile holds, prefixes of an odd number of pages and of thousands, own
parts of one token to many pieces; with the step's append fused and not; rows
that must not matter; graphs, streams, what runs ``attend`` instead.
"""

from __future__ import annotations

import dataclasses

import pytest
import torch

from llm_serving_layer_amd import BlockAllocator, RotaryTable, SequenceBlocks, backend
from llm_serving_layer_amd.backend import MI355XBackend

from ._ops64 import assert_within, attend64
from ._util import grow_and_assemble, make_meta, meta_to_device

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.fixture(autouse=True)
def share_all(request, monkeypatch):
    """Small batches too, which by the rule run ``attend``."""
    if request.function is not test_batches_that_save_too_little_run_attend:
        monkeypatch.setattr(backend, "SHARED_PART_BYTES", 0)
        monkeypatch.setattr(backend, "SHARED_LEAST_BYTES", 0)


class Batch:
    """A backend over a shuffled pool, sequences with page lists that begin
    alike: ``groups`` of (shared pages behind the common ones, own lengths)."""

    def __init__(self, root, groups, n_heads=32, n_kv=8, d=64, dtype=torch.float16, seed=0,
                 layers=1, ps=16, **kw):
        need = root + sum(b + sum(-(-n // ps) + 1 for n in own) for b, own in groups) + 8
        self.bk = MI355XBackend(layers, need, ps, n_kv, n_heads, d, device=DEV, dtype=dtype, **kw)
        self.g = torch.Generator(device=DEV).manual_seed(seed)
        for l in range(layers):
            self.bk.k_pool[l].copy_(self.rand(self.bk.k_pool[l].shape))
            self.bk.v_pool[l].copy_(self.rand(self.bk.k_pool[l].shape))
        self.alloc = BlockAllocator(need, ps)
        self.alloc.allocate(need)
        self.alloc.free(torch.randperm(need, generator=self.g, device=DEV).tolist())
        head = self.alloc.allocate(root) if root else []
        self.seqs = []
        for b, own in groups:
            pre = head + (self.alloc.allocate(b) if b else [])
            for n in own:
                s = SequenceBlocks(self.alloc, seq_id=len(self.seqs))
                if pre:
                    self.alloc.incref(pre)
                    s.block_ids, s.num_tokens = list(pre), len(pre) * ps
                if n > 1:
                    s.append(n - 1)
                self.seqs.append(s)
        self.meta = self.step()

    def step(self, mirror=True):
        meta = grow_and_assemble(self.seqs, [1] * len(self.seqs), self.bk.block_size)
        return meta_to_device(meta, DEV, mirror)

    def rand(self, shape):
        return torch.randn(shape, generator=self.g, device=DEV).to(self.bk.dtype)

    def q(self, heads=None):
        return self.rand((len(self.seqs), heads or self.bk.n_heads, self.bk.head_dim))

    def check(self, q, out, layer=0, scale=0.125, label=""):
        kp, vp = self.bk.k_pool[layer], self.bk.v_pool[layer]
        for i, s in enumerate(self.seqs):
            ids = torch.tensor(s.block_ids, device=DEV)
            k, v = (p[ids].flatten(0, 1)[:s.num_tokens] for p in (kp, vp))
            assert_within(out[i], *attend64(q[i], k, v, scale, self.bk.dtype),
                          label=f"{label} seq {i}")


GROUPS = {
    "one prefix": (33, [(0, [1, 2, 16, 17, 300, 900])]),
    "two sequences": (8, [(0, [5, 700])]),
    "a tree": (5, [(12, [3, 40, 1]), (9, [100, 1, 2, 3]), (0, [60]), (31, [7, 7])]),
    "more than a tile": (21, [(0, [1 + 3 * i for i in range(67)]), (6, [4] * 70)]),
    "no common head": (0, [(40, [9, 10, 11]), (7, [2, 200]), (0, [50]), (0, [5])]),
}


@pytest.mark.parametrize("groups", list(GROUPS))
@pytest.mark.parametrize("n_heads, n_kv, d", [
    (32, 8, 64), (8, 2, 128), (8, 8, 64), (16, 1, 64), (16, 2, 128), (6, 3, 128)])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_against_64_bits(groups, n_heads, n_kv, d, dtype):
    print(f"shared {groups} {n_heads}/{n_kv}/{d} {dtype}", flush=True)
    b = Batch(*GROUPS[groups], n_heads, n_kv, d, dtype)
    q = b.q()
    out = b.bk.attend_shared(q, 0, 0.125, b.meta)
    b.bk.check_device_errors()
    assert b.bk._shared.n_tiles > 0, "the shared kernel ran"
    b.check(q, out)
    assert torch.equal(b.bk.attend_shared(q, 0, 0.125, b.meta), out), "counters are left at zero"


@pytest.mark.parametrize("root, part_pages", [(1000, 17), (4097, 64), (64, 1), (127, 3)])
def test_long_prefixes_and_any_pieces(root, part_pages):
    print(f"shared root={root} part_pages={part_pages}", flush=True)
    b = Batch(root, [(0, [1, 30, 500, 1500])], 8, 2, 64, torch.bfloat16, part_pages=part_pages)
    q = b.q()
    out = b.bk.attend_shared(q, 0, 0.125, b.meta)
    assert b.bk._shared.n_tiles > 0
    b.check(q, out)


@pytest.mark.parametrize("root", [4, 5, 6, 7, 9, 10, 13, 16, 19, 131, 258, 531])
@pytest.mark.parametrize("n_heads, n_kv, d", [(32, 8, 64), (8, 2, 128), (4, 4, 128)])
def test_runs_in_one_tile(root, n_heads, n_kv, d, monkeypatch):
    """Every number of a tile's steps around its pipeline's length, whole and
    partial last steps, and runs past the page ids it holds at a time."""
    print(f"one tile root={root} {n_heads}/{n_kv}/{d}", flush=True)
    monkeypatch.setattr(backend, "SHARED_TILES", 1)
    b = Batch(root, [(0, [1, 30, 200])], n_heads, n_kv, d)
    q = b.q()
    q[1] *= 30                      # (a peaked row, whose reference moves)
    out = b.bk.attend_shared(q, 0, 0.125, b.meta)
    b.bk.check_device_errors()
    assert b.bk._shared.n_tiles == 1
    b.check(q, out)
    assert torch.equal(b.bk.attend_shared(q, 0, 0.125, b.meta), out)


def test_large_scores_move_the_reference():
    """Scores that grow along the prefix: the running maximum moves in the
    middle of a split, and the parts' maxima lie far apart."""
    b = Batch(64, [(0, [20, 400, 3])], 8, 2, 64, torch.float16)
    ids = b.seqs[0].block_ids[:64]
    ramp = torch.linspace(0.1, 8, 64, device=DEV)[:, None, None, None]
    b.bk.k_pool[0][ids] = (b.bk.k_pool[0][ids].float() * ramp).half()
    q = b.q()
    b.check(q, b.bk.attend_shared(q, 0, 0.125, b.meta))


@pytest.mark.parametrize("decode_workgroups", [1, 8, None])
@pytest.mark.parametrize("rotated", [False, True])
def test_steps_with_their_appends(decode_workgroups, rotated):
    """A running batch over a tree: append then attend_shared, layer by layer,
    the append fused where it may be; the pool and the outputs as by append
    then attend on a second backend."""
    kw = {"layers": 2, "decode_workgroups": decode_workgroups}
    a, b = (Batch(20, [(8, [1, 15, 33]), (4, [16, 200])], **kw) for _ in range(2))
    b.bk._pool.copy_(a.bk._pool)
    table = RotaryTable(4096, 64, device=DEV)
    for _ in range(18):
        ma, mb = a.step(), b.step()
        for l in range(2):
            q, k, v = a.q(), a.q(8), a.q(8)
            if rotated:
                qa = a.bk.append_kv_rotated(l, q, k, v, ma, table)
                qb = b.bk.append_kv_rotated(l, q, k, v, mb, table)
                assert torch.equal(qa, qb)
            else:
                qa = qb = q
                a.bk.append_kv(l, k, v, ma)
                b.bk.append_kv(l, k, v, mb)
            out = a.bk.attend_shared(qa, l, 0.125, ma)
            want = b.bk.attend(qb, l, 0.125, mb)
            a.check(qa, out, l)
            assert float((out.float() - want.float()).abs().max()) < 4e-3
            assert torch.equal(a.bk.k_pool[l], b.bk.k_pool[l])
            assert torch.equal(a.bk.v_pool[l], b.bk.v_pool[l])
    a.bk.check_device_errors()


def test_a_deferred_append_of_another_layer_or_meta_lands_first():
    b = Batch(20, [(0, [1, 15, 33])], layers=2)
    meta = b.step()
    q, k, v = b.q(), b.q(8), b.q(8)
    b.bk.append_kv(1, k, v, meta)
    b.check(q, b.bk.attend_shared(q, 0, 0.125, meta))
    rows = b.bk.k_pool[1].view(-1, 8, 64)[meta.slot_mapping.long()]
    assert torch.equal(rows, k)


def test_new_rows_at_an_odd_address():
    b = Batch(20, [(0, [1, 30, 200])], 8, 2, 64)
    q, n = b.q(), 3 * 2 * 64
    k, v = (b.rand((n + 1,))[1:].view(3, 2, 64) for _ in range(2))
    assert k.data_ptr() % 16
    b.bk.append_kv(0, k, v, b.meta)
    out = b.bk.attend_shared(q, 0, 0.125, b.meta)
    slots = b.meta.slot_mapping.long()
    assert torch.equal(b.bk.k_pool[0].view(-1, 2, 64)[slots], k)
    b.check(q, out)


def test_rows_behind_the_ends_and_other_pages_do_not_matter():
    b = Batch(9, [(0, [1, 5, 40])])
    q = b.q()
    out = b.bk.attend_shared(q, 0, 0.125, b.meta)
    used = set(x for s in b.seqs for x in s.block_ids)
    for p in (b.bk.k_pool[0], b.bk.v_pool[0]):
        for s in b.seqs:
            p[s.block_ids[-1], (s.num_tokens - 1) % 16 + 1:] = float("nan")
        for x in set(range(b.bk.num_blocks)) - used:
            p[x] = float("nan")
    assert torch.equal(b.bk.attend_shared(q, 0, 0.125, b.meta), out)


def test_pages_far_into_a_large_pool():
    nb = 140000                                  # 4.6 GB a tensor
    bk = MI355XBackend(1, nb, 16, 8, 32, 128, device=DEV, dtype=torch.bfloat16)
    b = object.__new__(Batch)
    b.bk, b.g, b.alloc = bk, torch.Generator(device=DEV).manual_seed(5), BlockAllocator(nb, 16)
    b.alloc.allocate(nb)
    b.seqs = []
    for i in range(5):
        s = SequenceBlocks(b.alloc, seq_id=i)
        s.block_ids = list(range(nb - 1, nb - 41, -1)) + [nb - 50 - i]
        s.num_tokens = 40 * 16 + 3 * i + 1
        b.seqs.append(s)
    for p in (bk.k_pool[0], bk.v_pool[0]):
        p[nb - 64:] = b.rand((64, 16, 8, 128))
    meta = meta_to_device(make_meta(b.seqs, [1] * 5, 16), DEV)
    q = b.q()
    out = bk.attend_shared(q, 0, 0.125, meta)
    bk.check_device_errors()
    assert bk._shared.n_tiles > 0
    b.check(q, out)


def test_what_runs_attend_itself():
    """Chunks in the batch, nothing shared, no matrix-core kernel, a scale of
    zero or below: the same bits as attend, planned without a mirror too."""
    b = Batch(20, [(0, [1, 15, 33])])
    q = b.q()
    for scale in (0.0, -0.2):
        assert torch.equal(b.bk.attend_shared(q, 0, scale, b.meta),
                           b.bk.attend(q, 0, scale, b.meta))
    alone = Batch(0, [(0, [100]), (0, [40])])
    q = alone.q()
    assert torch.equal(alone.bk.attend_shared(q, 0, 0.125, alone.meta),
                       alone.bk.attend(q, 0, 0.125, alone.meta))
    chunk = meta_to_device(grow_and_assemble(b.seqs, [1, 7, 1], 16), DEV)
    q = b.rand((9, 32, 64))
    assert torch.equal(b.bk.attend_shared(q, 0, 0.125, chunk), b.bk.attend(q, 0, 0.125, chunk))
    for kw in ({"dtype": torch.float32}, {"d": 80}, {"n_heads": 24}, {"ps": 8}):
        c = Batch(12, [(0, [1, 15, 33])], **kw)
        q = c.q()
        assert torch.equal(c.bk.attend_shared(q, 0, 0.125, c.meta),
                           c.bk.attend(q, 0, 0.125, c.meta)), kw
    d = Batch(20, [(0, [1, 15, 33])])
    q = d.q()
    want = d.bk.attend_shared(q, 0, 0.125, d.meta)
    bare = dataclasses.replace(d.meta, host=None)
    assert torch.equal(d.bk.attend_shared(q, 0, 0.125, bare), want)
    odd = torch.empty(q.numel() + 1, dtype=q.dtype, device=DEV)[1:].view_as(q).copy_(q)
    assert torch.equal(d.bk.attend_shared(odd, 0, 0.125, d.meta), want)


def test_batches_that_save_too_little_run_attend():
    few = Batch(96, [(0, [3, 20, 40])])
    q = few.q()
    assert torch.equal(few.bk.attend_shared(q, 0, 0.125, few.meta),
                       few.bk.attend(q, 0, 0.125, few.meta))
    assert not few.bk._shared.n_tiles
    many = Batch(256, [(0, [5] * 40), (3, [9, 9])])
    q = many.q()
    out = many.bk.attend_shared(q, 0, 0.125, many.meta)
    assert many.bk._shared.n_tiles and many.bk._shared.n_merges == 42
    many.check(q, out)


def test_two_graphs_and_another_stream():
    b = Batch(40, [(6, [1, 150, 33]), (0, [500])])
    some = b.seqs[:3]
    other = meta_to_device(make_meta(some, [1] * 3, 16), DEV)
    q = b.q()
    q1 = q[:3].clone()
    want = b.bk.attend_shared(q, 0, 0.125, b.meta)
    want1 = b.bk.attend_shared(q1, 0, 0.125, other)
    graphs = []
    for qq, meta in ((q, b.meta), (q1, other)):
        b.bk.attend_shared(qq, 0, 0.125, meta)          # planned before the capture
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = b.bk.attend_shared(qq, 0, 0.125, meta)
        graphs.append((graph, out))
    b.bk.invalidate_plan()
    junk = [torch.full((1 << 20,), -1, dtype=torch.int32, device=DEV) for _ in range(8)]
    for _ in range(3):
        for (graph, out), w in zip(graphs, (want, want1)):
            out.zero_()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, w)
        assert not torch.equal(b.bk.attend_shared(q * 2, 0, 0.125, b.meta), want)
        torch.cuda.synchronize()
    del junk
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = [b.bk.attend_shared(q, 0, 0.125, b.meta) for _ in range(3)]
    got.append(b.bk.attend_shared(q, 0, 0.125, b.meta))
    torch.cuda.synchronize()
    assert all(torch.equal(x, want) for x in got)


def test_bad_pages_are_flagged():
    """A bad id among the shared pages, in every list and in one of them."""
    for rows in ([0, 1, 2], [1]):
        b = Batch(20, [(0, [1, 15, 33])])
        idx = b.meta.kv_indices.clone()
        ptr = b.meta.kv_indptr.tolist()
        for i in rows:
            idx[ptr[i] + 7] = b.bk.num_blocks + 3
        meta = dataclasses.replace(b.meta, kv_indices=idx, host=None)
        b.bk.attend_shared(b.q(), 0, 0.125, meta)
        with pytest.raises(IndexError, match="kv_indices"):
            b.bk.check_device_errors()


@pytest.mark.parametrize("at, bad", [(0, -1), (299, 10 ** 6), (150, -2 ** 31)])
def test_a_bad_page_anywhere_in_a_long_tile(at, bad, monkeypatch):
    monkeypatch.setattr(backend, "SHARED_TILES", 1)
    b = Batch(300, [(0, [5, 40])], 8, 2, 128)
    q = b.q()
    idx, ptr = b.meta.kv_indices.clone(), b.meta.kv_indptr.tolist()
    idx[ptr[0] + at] = idx[ptr[1] + at] = bad
    meta = dataclasses.replace(b.meta, kv_indices=idx, host=None)
    b.bk.attend_shared(q, 0, 0.125, meta)
    assert b.bk._shared.n_tiles == 1
    with pytest.raises(IndexError, match="kv_indices"):
        b.bk.check_device_errors()
    b.check(q, b.bk.attend_shared(q, 0, 0.125, b.meta))
    b.bk.check_device_errors()


def test_refusals():
    b = Batch(20, [(0, [1, 15])])
    q = b.q()
    wrong = dataclasses.replace(b.meta, kv_last_page_len=b.meta.kv_last_page_len + 1, host=None)
    for args, match in (((q, 1, 0.1, b.meta), "layer_idx"), ((q[:, :4], 0, 0.1, b.meta), "q has"),
                        ((q[:1], 0, 0.1, b.meta), "tokens"),
                        ((q, 0, 0.1, wrong), "kv_last_page_len")):
        with pytest.raises(ValueError, match=match):
            b.bk.attend_shared(*args)
