"""
Page bounds, the choice of pages by them, and the attention over the chosen
pages, against their definitions in 64 bits: head layouts and types with and
without matrix-core kernels, budgets around the lists' lengths, ties, NaN and
infinite keys, rows behind a sequence's end; the bounds under every way rows
reach the pool; graphs and streams; refusals.
"""

from __future__ import annotations

import dataclasses

import pytest
import torch

from llm_serving_layer_amd import (BlockAllocator, KVSwapSpace, RotaryTable, SequenceBlocks,
                                   backend)
from llm_serving_layer_amd.backend import MI355XBackend

from ._ops64 import assert_within, attend64, chosen64
from ._util import grow_and_assemble, make_meta, meta_to_device

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


class Cache:
    """A backend with page bounds over a shuffled pool of random rows."""

    def __init__(self, lens, n_heads, n_kv, d, dtype, ps=16, seed=0, layers=1, spare=4, **kw):
        need = sum(-(-n // ps) + 1 for n in lens) + spare
        self.bk = MI355XBackend(layers, need, ps, n_kv, n_heads, d, device=DEV, dtype=dtype,
                                page_bounds=True, **kw)
        self.alloc = BlockAllocator(need, ps)
        self.alloc.allocate(need)
        self.g = torch.Generator(device=DEV).manual_seed(seed)
        self.alloc.free(torch.randperm(need, generator=self.g, device=DEV).tolist())
        for l in range(layers):
            k = self.rand(self.bk.k_pool[l].shape)
            k += self.rand((need, 1, n_kv, d))
            self.bk.k_pool[l].copy_(k)
            self.bk.v_pool[l].copy_(self.rand(k.shape))
        self.bk.refresh_page_bounds()
        self.seqs = [SequenceBlocks(self.alloc, seq_id=i) for i in range(len(lens))]
        for s, n in zip(self.seqs, lens):
            s.append(n - 1) if n > 1 else None
        self.meta = meta_to_device(grow_and_assemble(self.seqs, [1] * len(lens), ps), DEV)

    def rand(self, shape):
        return torch.randn(shape, generator=self.g, device=DEV).to(self.bk.dtype)

    def q(self):
        return self.rand((len(self.seqs), self.bk.n_heads, self.bk.head_dim))

    def check(self, q, pages, out, chosen, layer=0, scale=0.125, label=""):
        bk = self.bk
        kp, vp = bk.k_pool[layer], bk.v_pool[layer]
        lo, hi = kp.amin(1), kp.amax(1)
        width = min(pages, max(s.num_blocks for s in self.seqs))
        assert chosen.shape == (len(self.seqs), bk.n_kv_heads, width)
        for i, s in enumerate(self.seqs):
            ids = torch.tensor(s.block_ids, device=DEV)
            want = chosen64(q[i], lo[ids], hi[ids], len(ids), pages)
            keys, values = [], []
            for h, w in enumerate(want):
                assert chosen[i, h].tolist() == w + [-1] * (width - len(w)), f"{label} {i} {h}"
                live = (len(w) - 1) * bk.block_size + s.num_tokens - (len(ids) - 1) * bk.block_size
                keys.append(kp[ids[w], :, h].flatten(0, 1)[:live])
                values.append(vp[ids[w], :, h].flatten(0, 1)[:live])
            assert_within(out[i], *attend64(q[i], keys, values, scale, bk.dtype),
                          label=f"{label} seq {i}")


LENS = [1, 15, 16, 17, 33, 500, 1600, 700]


@pytest.mark.parametrize("n_heads, n_kv, d", [
    (32, 8, 64), (8, 2, 128), (8, 8, 64), (16, 1, 64), (12, 3, 128), (16, 2, 128)])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("pages", [1, 2, 7, 30, 100, 1000])
def test_choice_and_attention(n_heads, n_kv, d, dtype, pages):
    print(f"selected {n_heads}/{n_kv}/{d} {dtype} pages={pages}", flush=True)
    c = Cache(LENS, n_heads, n_kv, d, dtype)
    q = c.q()
    out, chosen = c.bk.attend_selected(q, 0, 0.125, c.meta, pages, return_pages=True)
    c.bk.check_device_errors()
    c.check(q, pages, out, chosen)
    assert torch.equal(c.bk.attend_selected(q, 0, 0.125, c.meta, pages), out)


@pytest.mark.parametrize("n_heads, n_kv, d, dtype, ps", [
    (32, 8, 64, torch.float32, 16), (9, 3, 80, torch.float16, 16), (4, 2, 7, torch.bfloat16, 16),
    (8, 2, 64, torch.float16, 8), (4, 4, 256, torch.float32, 32), (12, 4, 64, torch.bfloat16, 16)])
@pytest.mark.parametrize("pages", [1, 5, 40])
def test_geometries_without_a_matrix_core_kernel(n_heads, n_kv, d, dtype, ps, pages):
    print(f"selected generic {n_heads}/{n_kv}/{d} {dtype} ps={ps} pages={pages}", flush=True)
    c = Cache([1, ps, ps + 1, 23 * ps + 5], n_heads, n_kv, d, dtype, ps=ps)
    q = c.q()
    out, chosen = c.bk.attend_selected(q, 0, 0.125, c.meta, pages, return_pages=True)
    c.bk.check_device_errors()
    c.check(q, pages, out, chosen)


@pytest.mark.parametrize("part_pages", [1, 3, 17, 64])
def test_pieces_of_any_size(part_pages):
    c = Cache([2000, 90, 400], 8, 2, 64, torch.float16, part_pages=part_pages)
    q = c.q()
    out, chosen = c.bk.attend_selected(q, 0, 0.125, c.meta, 90, return_pages=True)
    c.check(q, 90, out, chosen)


@pytest.mark.parametrize("n_heads, n_kv, d", [
    (32, 8, 64), (8, 2, 128), (8, 8, 64), (16, 1, 64), (12, 3, 128), (16, 2, 128)])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("pages, part_pages", [(1, 17), (7, 3), (30, 17), (100, 1), (1000, 64)])
def test_the_streaming_kernel(n_heads, n_kv, d, dtype, pages, part_pages, monkeypatch):
    """The kernel for many pieces, whatever their number: page words placed by
    the plan, pieces with a folded remainder, whole lists and cut ones."""
    print(f"selected stream {n_heads}/{n_kv}/{d} {dtype} {pages} {part_pages}", flush=True)
    monkeypatch.setattr(backend, "SELECTED_PIECES", 0)
    c = Cache(LENS, n_heads, n_kv, d, dtype, part_pages=part_pages)
    q = c.q()
    out, chosen = c.bk.attend_selected(q, 0, 0.125, c.meta, pages, return_pages=True)
    c.bk.check_device_errors()
    assert c.bk._selected.plan is not None
    c.check(q, pages, out, chosen)
    assert torch.equal(c.bk.attend_selected(q, 0, 0.125, c.meta, pages), out)


def test_bad_pages_in_a_streamed_choice(monkeypatch):
    monkeypatch.setattr(backend, "SELECTED_PIECES", 0)
    test_bad_pages_are_flagged_and_read_nothing()


def test_a_long_history_and_many_sequences():
    for lens, pages in (([70001], 64), ([300 + 7 * i for i in range(150)], 9)):
        print("lengths", lens[:3], flush=True)
        c = Cache(lens, 32, 8, 64, torch.bfloat16)
        q = c.q()
        out, chosen = c.bk.attend_selected(q, 0, 0.125, c.meta, pages, return_pages=True)
        c.check(q, pages, out, chosen)


def test_equal_scores_take_the_earlier_pages():
    """Small whole numbers: every score is exact, many are equal; all pages of
    one sequence hold the same keys."""
    c = Cache([640, 640, 333], 8, 2, 64, torch.float16)
    kp = c.bk.k_pool[0]
    kp.copy_(torch.randint(-1, 2, kp.shape, generator=c.g, device=DEV))
    kp[torch.tensor(c.seqs[1].block_ids, device=DEV)] = kp[c.seqs[1].block_ids[0]].clone()
    c.bk.refresh_page_bounds()
    q = torch.randint(-2, 3, (3, 8, 64), generator=c.g, device=DEV).half()
    out, chosen = c.bk.attend_selected(q, 0, 0.125, c.meta, 12, return_pages=True)
    c.check(q, 12, out, chosen)
    assert chosen[1].tolist() == [list(range(11)) + [39]] * 2


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("n_heads, n_kv, d", [(32, 8, 64), (8, 1, 128), (16, 1, 64)])
def test_scores_that_only_64_bits_tell_apart(n_heads, n_kv, d, dtype):
    """Every page the same but for the last place of one small element: scores
    that differ by far less than 32-bit sums do."""
    c = Cache([1500, 900, 40], n_heads, n_kv, d, dtype)
    for s in c.seqs[:2]:
        ids = torch.tensor(s.block_ids, device=DEV)
        page = c.rand((16, n_kv, d)).abs() + 1
        page[..., 5] = 2.0 ** -9
        kp = page.repeat(len(ids), 1, 1, 1)
        step = torch.randperm(len(ids), generator=c.g, device=DEV) % 7
        kp[..., 5] *= (1 + step * torch.finfo(dtype).eps)[:, None, None].to(dtype)
        c.bk.k_pool[0][ids] = kp
    c.bk.refresh_page_bounds()
    q = c.q().abs()
    for pages in (2, 9, 30):
        out, chosen = c.bk.attend_selected(q, 0, 0.125, c.meta, pages, return_pages=True)
        c.check(q, pages, out, chosen)


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_lists_longer_than_a_workgroup_holds(dtype):
    """16 500 candidates: the choice that re-reads its scores."""
    c = Cache([16500 * 16 + 5, 4], 8, 1, 64, dtype)
    q = c.q()
    out, chosen = c.bk.attend_selected(q, 0, 0.125, c.meta, 40, return_pages=True)
    c.bk.check_device_errors()
    c.check(q, 40, out, chosen)


@pytest.mark.parametrize("n_heads, n_kv, d", [
    (32, 8, 64), (8, 8, 128), (16, 8, 64), (64, 8, 128), (64, 4, 64)])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("kind", ["random", "close", "whole numbers", "tiny", "nan"])
def test_many_candidates(n_heads, n_kv, d, dtype, kind):
    """Enough of them that their scores run in 32 bits first: random pages,
    pages that only 64 bits tell apart, ties, subnormal keys, and a NaN key."""
    pages = (17 << 20) // (n_kv * d)
    lens = [pages * 16 // 4 + 16, pages * 16 // 4 + 3, 40 * 16, 5]
    print(f"many candidates {n_heads}/{n_kv}/{d} {dtype} {kind} {lens}", flush=True)
    c = Cache(lens, n_heads, n_kv, d, dtype)
    q, kp = c.q(), c.bk.k_pool[0]
    if kind == "close":
        page = c.rand((16, n_kv, d)).abs() + 1
        page[..., 5] = 2.0 ** -9
        step = torch.randperm(kp.shape[0], generator=c.g, device=DEV) % 50
        kp.copy_(page)
        kp[..., 5] *= (1 + step * torch.finfo(dtype).eps)[:, None, None].to(dtype)
        q = q.abs()
    elif kind == "whole numbers":
        kp.copy_(torch.randint(-1, 2, kp.shape, generator=c.g, device=DEV))
        q = torch.randint(-2, 3, q.shape, generator=c.g, device=DEV).to(dtype)
    elif kind == "tiny":
        kp *= 2.0 ** -20 if dtype == torch.float16 else 2.0 ** -128
        q *= 2.0 ** 9 if dtype == torch.float16 else 2.0 ** 120
    c.bk.refresh_page_bounds()
    if kind == "nan":                                  # in one KV head of one sequence
        ids = c.seqs[0].block_ids
        c.bk.key_bounds[0][:, ids[77], n_kv - 1, 3] = float("nan")
        out, chosen = c.bk.attend_selected(q, 0, 0.125, c.meta, 30, return_pages=True)
        assert (chosen[0, n_kv - 1] == 77).any()
        lo, hi = (b[ids] for b in c.bk.key_bounds[0])
        want = chosen64(q[0], lo, hi, len(ids), 30)
        assert chosen[0].tolist() == want
        return
    for pages in (2, 30):
        out, chosen = c.bk.attend_selected(q, 0, 0.125, c.meta, pages, return_pages=True)
        c.bk.check_device_errors()
        c.check(q, pages, out, chosen)


def test_lists_of_every_kernel_size():
    """Around 1024, 4096 and 16384 pages, where the choice's kernels change."""
    for n in (1023, 1024, 1025, 4096, 4097, 16384, 16385):
        print("pages", n, flush=True)
        c = Cache([n * 16 - 3], 4, 2, 64, torch.bfloat16)
        q = c.q()
        out, chosen = c.bk.attend_selected(q, 0, 0.125, c.meta, 21, return_pages=True)
        c.check(q, 21, out, chosen)


def test_signs_and_sizes_of_scores():
    """All scores negative, all zero, of one exponent, and far apart."""
    c = Cache([900] * 4, 4, 4, 64, torch.bfloat16)
    kp = c.bk.k_pool[0]
    for i, f in enumerate((lambda k: -k.abs(), lambda k: k * 0, lambda k: 1 + k / 512,
                           lambda k: k * torch.logspace(-30, 30, k.shape[0], device=DEV)
                           [:, None, None, None])):
        ids = torch.tensor(c.seqs[i].block_ids, device=DEV)
        kp[ids] = f(kp[ids].float()).bfloat16()
    c.bk.refresh_page_bounds()
    q = c.q().abs()
    q[3] *= 1e-30                  # (scores within the softmax's range)
    out, chosen = c.bk.attend_selected(q, 0, 0.125, c.meta, 20, return_pages=True)
    c.check(q, 20, out, chosen)


def test_nan_and_infinite_keys():
    """A page with a NaN key, or an infinite bound, is chosen first; the heads
    without them are unharmed."""
    c = Cache([640], 8, 2, 64, torch.float16)
    q, ids = c.q(), c.seqs[0].block_ids
    c.bk.k_pool[0][ids[5], 3, 0, 9] = float("nan")
    c.bk.k_pool[0][ids[20], 3, 0, 9] = float("inf")
    c.bk.refresh_page_bounds([ids[5], ids[20]])
    assert torch.isnan(c.bk.key_bounds[0][:, ids[5], 0, 9]).all()
    out, chosen = c.bk.attend_selected(q, 0, 0.125, c.meta, 2, return_pages=True)
    assert chosen[0, 0].tolist() == [5, 39]
    _, more = c.bk.attend_selected(q, 0, 0.125, c.meta, 3, return_pages=True)
    if bool((q[0, :4, 9] > 0).any()):
        assert more[0, 0].tolist() == [5, 20, 39]
    lo, hi = c.bk.k_pool[0].amin(1)[ids], c.bk.k_pool[0].amax(1)[ids]
    want = chosen64(q[0], lo, hi, 40, 2)[1]
    assert chosen[0, 1].tolist() == want and torch.isfinite(out[0, 4:]).all()


def test_rows_behind_the_last_sequence_token_do_not_matter():
    """NaN in the rows of the last pages past the sequences' ends, and in pages
    of no sequence: neither the choice nor the output changes."""
    c = Cache([250, 1601, 16, 3], 32, 8, 64, torch.float16)
    q = c.q()
    out, chosen = c.bk.attend_selected(q, 0, 0.125, c.meta, 8, return_pages=True)
    used = set(b for s in c.seqs for b in s.block_ids)
    for p in (c.bk.k_pool[0], c.bk.v_pool[0]):
        for s in c.seqs:
            p[s.block_ids[-1], (s.num_tokens - 1) % 16 + 1:] = float("nan")
        for b in set(range(c.bk.num_blocks)) - used:
            p[b] = float("nan")
    c.bk.refresh_page_bounds()
    again, same = c.bk.attend_selected(q, 0, 0.125, c.meta, 8, return_pages=True)
    assert torch.equal(chosen, same) and torch.equal(out, again)


def test_pages_far_into_a_large_pool():
    """Rows past 2^32 bytes of each tensor, bounds past 2^28."""
    nb = 140000
    bk = MI355XBackend(1, nb, 16, 8, 32, 128, device=DEV, dtype=torch.float16, page_bounds=True)
    alloc = BlockAllocator(nb, 16)
    alloc.allocate(nb)
    s = SequenceBlocks(alloc, seq_id=0)
    s.block_ids, s.num_tokens = list(range(nb - 1, nb - 81, -1)), 1279
    c = object.__new__(Cache)
    c.bk, c.alloc, c.g, c.seqs = bk, alloc, torch.Generator(device=DEV).manual_seed(3), [s]
    for p in (bk.k_pool[0], bk.v_pool[0]):
        p[nb - 80:] = c.rand((80, 16, 8, 128))
    bk.refresh_page_bounds(s.block_ids)
    meta = meta_to_device(make_meta([s], [1], 16), DEV)
    q = c.q()
    out, chosen = bk.attend_selected(q, 0, 0.125, meta, 10, return_pages=True)
    bk.check_device_errors()
    kp = bk.k_pool[0][nb - 80:].flip(0)
    want = chosen64(q[0], kp.amin(1), kp.amax(1), 80, 10)
    assert chosen[0].tolist() == want
    vp = bk.v_pool[0][nb - 80:].flip(0)
    keys = [kp[w, :, h].flatten(0, 1)[:159] for h, w in enumerate(want)]
    values = [vp[w, :, h].flatten(0, 1)[:159] for h, w in enumerate(want)]
    assert_within(out[0], *attend64(q[0], keys, values, 0.125, torch.float16))


# ------------------------------------------------------------------ bounds ---

def complete_pages(seqs, ps):
    return sorted({b for s in seqs for b in s.block_ids[:s.num_tokens // ps]})


def assert_bounds(bk, blocks, layers=None):
    for l in layers if layers is not None else range(bk.num_layers):
        kp = bk.k_pool[l][blocks]
        assert torch.equal(bk.key_bounds[l][0][blocks], kp.amin(1))
        assert torch.equal(bk.key_bounds[l][1][blocks], kp.amax(1))


@pytest.mark.parametrize("n_kv, d, dtype, ps", [
    (8, 64, torch.float16, 16), (2, 128, torch.bfloat16, 16), (3, 5, torch.float16, 8),
    (4, 64, torch.float32, 16), (1, 80, torch.bfloat16, 32), (64, 128, torch.float16, 16)])
@pytest.mark.parametrize("rotated", [False, True])
def test_appends_bound_the_pages_they_complete(n_kv, d, dtype, ps, rotated):
    print(f"bounds {n_kv}/{d} {dtype} ps={ps} rotated={rotated}", flush=True)
    bk = MI355XBackend(2, 64, ps, n_kv, 2 * n_kv, d, device=DEV, dtype=dtype, page_bounds=True)
    assert bk.bounds_bytes() * ps == bk.pool_bytes()
    g = torch.Generator(device=DEV).manual_seed(1)
    table = RotaryTable(64 * ps, d // 2 * 2, device=DEV)
    alloc = BlockAllocator(64, ps)
    seqs = [SequenceBlocks(alloc, seq_id=i) for i in range(3)]
    steps = [[3 * ps + 1, ps - 1, 1], [1, 1, ps], [2 * ps, 1, 0]] + [[1, 1, 1]] * ps
    for step in steps:
        meta = meta_to_device(grow_and_assemble(seqs, step, ps), DEV)
        T = sum(step)
        for l in range(2):
            k, v = (torch.randn(T, n_kv, d, generator=g, device=DEV).to(dtype) for _ in "kv")
            if rotated:
                q = torch.randn(T, 2 * n_kv, d, generator=g, device=DEV).to(dtype)
                bk.append_kv_rotated(l, q, k, v, meta, table)
            else:
                bk.append_kv(l, k, v, meta)
        blocks = complete_pages(seqs, ps)
        if blocks:
            assert_bounds(bk, blocks)
    bk.check_device_errors()


def test_rows_sent_elsewhere_renew_the_pages_they_touch():
    """slot_mapping that disagrees with the page table: the touched pages are
    renewed; slots outside the pool renew nothing."""
    c = Cache([64, 40], 8, 2, 64, torch.float16)
    slots = torch.tensor([5 * 16 + 3, 10 ** 6], dtype=torch.int32, device=DEV)
    for mirror in (True, False):
        meta = dataclasses.replace(meta_to_device(make_meta(c.seqs, [1, 1], 16), DEV, mirror),
                                   slot_mapping=slots, host=None)
        k = 9 + c.rand((2, 2, 64))
        c.bk.append_kv(0, k, k, meta)
        assert_bounds(c.bk, [5])
        assert float(c.bk.key_bounds[0][1][5].amin()) > 3
    with pytest.raises(IndexError, match="slot_mapping"):
        c.bk.check_device_errors()


def test_block_copies_and_swaps_carry_the_bounds():
    c = Cache([160, 90], 8, 2, 64, torch.bfloat16, layers=3, spare=20)
    free = [b for b in range(c.bk.num_blocks) if not any(b in s.block_ids for s in c.seqs)]
    src, dst = c.seqs[0].block_ids[:3], free[:3]
    c.bk.copy_blocks(src, dst)
    c.bk.copy_block(c.seqs[1].block_ids[0], free[3])
    assert_bounds(c.bk, dst + [free[3]])
    space = KVSwapSpace(c.bk)
    s = c.seqs[0]
    handle = space.swap_out("a", s)
    s.free()
    for p in (*c.bk.k_pool, *c.bk.v_pool):
        p.mul_(-2)
    c.bk.refresh_page_bounds()
    back = SequenceBlocks(c.alloc, seq_id=9)
    back.append(160)
    space.swap_in(handle, back)
    assert_bounds(c.bk, back.block_ids)
    c.bk.reset()
    assert not c.bk.key_bounds[0].any()


def test_refresh_of_some_blocks_and_of_all():
    c = Cache([64], 8, 2, 64, torch.float16, layers=2)
    c.bk.k_pool[1].mul_(3)
    old = c.bk.key_bounds[1].clone()
    c.bk.refresh_page_bounds([1, 3, 3])
    assert_bounds(c.bk, [1, 3])
    keep = [b for b in range(c.bk.num_blocks) if b not in (1, 3)]
    assert torch.equal(c.bk.key_bounds[1][:, keep], old[:, keep])
    c.bk.refresh_page_bounds([])
    c.bk.refresh_page_bounds()
    assert_bounds(c.bk, list(range(c.bk.num_blocks)))


# ---------------------------------------------------- graphs, streams, errors ---

def test_two_graphs_and_another_stream():
    """Two captured metas replayed in turn with eager work between, and the
    same meta on a second stream: all equal the eager result."""
    c = Cache([1700, 400, 60], 32, 8, 64, torch.float16)
    small = [c.seqs[0]]
    other = meta_to_device(make_meta(small, [1], 16), DEV)
    q, q1 = c.q(), c.q()[:1].clone()
    want, want1 = (c.bk.attend_selected(q, 0, 0.125, c.meta, 30),
                   c.bk.attend_selected(q1, 0, 0.125, other, 60))
    graphs = []
    for qq, meta, pages in ((q, c.meta, 30), (q1, other, 60)):
        c.bk.attend_selected(qq, 0, 0.125, meta, pages)      # planned before the capture
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out, chosen = c.bk.attend_selected(qq, 0, 0.125, meta, pages, return_pages=True)
        graphs.append((graph, out, chosen))
    c.bk.invalidate_plan()
    junk = [torch.full((1 << 20,), -1, dtype=torch.int32, device=DEV) for _ in range(8)]
    for _ in range(3):
        for (graph, out, _), w in zip(graphs, (want, want1)):
            out.zero_()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, w)
        eager = c.bk.attend_selected(q * 2, 0, 0.125, c.meta, 30)
        assert not torch.equal(eager, want)
        torch.cuda.synchronize()
    del junk
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = [c.bk.attend_selected(q, 0, 0.125, c.meta, 30) for _ in range(3)]
    got.append(c.bk.attend_selected(q, 0, 0.125, c.meta, 30))
    torch.cuda.synchronize()
    for x in got:
        assert torch.equal(x, want)


def test_bad_pages_are_flagged_and_read_nothing():
    c = Cache([300, 300], 8, 2, 64, torch.float16)
    idx = c.meta.kv_indices.clone()
    idx[2], idx[5] = -3, c.bk.num_blocks
    meta = dataclasses.replace(c.meta, kv_indices=idx, host=None)
    q = c.q()
    good, _ = c.bk.attend_selected(q, 0, 0.125, c.meta, 6, return_pages=True)
    c.bk.check_device_errors()
    out = c.bk.attend_selected(q, 0, 0.125, meta, 6)
    with pytest.raises(IndexError, match="kv_indices"):
        c.bk.check_device_errors()
    assert torch.equal(out[1], good[1])


def test_refusals():
    c = Cache([300, 20], 8, 2, 64, torch.float16)
    q = c.q()
    for args, match in (((q, 1, 0.1, c.meta, 4), "layer_idx"),
                        ((q[:, :4], 0, 0.1, c.meta, 4), "q has shape"),
                        ((q[:1], 0, 0.1, c.meta, 4), "tokens"),
                        ((q, 0, 0.1, c.meta, 0), "pages"),
                        ((q, 0, 0.1, c.meta, -1), "pages"),
                        ((q, 0, 0.0, c.meta, 4), "scale"),
                        ((q, 0, -1.0, c.meta, 4), "scale"),
                        ((q, 0, float("nan"), c.meta, 4), "scale")):
        with pytest.raises(ValueError, match=match):
            c.bk.attend_selected(*args)
    with pytest.raises(TypeError):
        c.bk.attend_selected(q, 0, 0.1, c.meta, 2.5)
    every = c.bk.attend_selected(q, 0, 0.1, c.meta, 10 ** 12)
    assert torch.equal(every, c.bk.attend_selected(q, 0, 0.1, c.meta, 19))
    chunk = meta_to_device(grow_and_assemble(c.seqs, [2, 1], 16), DEV)
    with pytest.raises(ValueError, match="one token per sequence"):
        c.bk.attend_selected(c.rand((3, 8, 64)), 0, 0.1, chunk, 4)
    wrong = dataclasses.replace(c.meta, kv_last_page_len=c.meta.kv_last_page_len + 1, host=None)
    with pytest.raises(ValueError, match="kv_last_page_len"):
        c.bk.attend_selected(q, 0, 0.1, wrong, 4)
    plain = MI355XBackend(1, 8, 16, 2, 8, 64, device=DEV)
    for call in (lambda: plain.attend_selected(q, 0, 0.1, c.meta, 4),
                 lambda: plain.refresh_page_bounds(), lambda: plain.key_bounds):
        with pytest.raises(ValueError, match="page_bounds=True"):
            call()
    with pytest.raises(IndexError):
        c.bk.refresh_page_bounds([c.bk.num_blocks])
