"""
The 4-bit cache on the GPU: rows appended and read back give the definition's
values bit for bit; attention over it lies within the bound of its arithmetic;
block copies, swaps, streams and graphs.
"""

from __future__ import annotations

import dataclasses
import math
import random

import pytest
import torch

from llm_serving_layer_amd import (BlockAllocator, FourBitBackend, KVSwapSpace, SequenceBlocks)

from ._fourbit import attend64, held64
from ._ops64 import assert_within
from ._util import grow_and_assemble, make_meta

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


def rows(shape, dtype, seed, centre=1.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(shape, generator=g) * 0.5
    return (x + centre * torch.randn(shape[1:], generator=g)).to(dtype)


def same_bits(got, want64, dtype):
    """NaN where NaN is wanted, the same number elsewhere."""
    want = want64.to(dtype)
    got = got.cpu()
    assert torch.equal(got.isnan(), want.isnan())
    assert torch.equal(got.nan_to_num(7.0), want.nan_to_num(7.0))


class Cache:
    """Sequences over one backend, their rows kept beside it."""

    def __init__(self, lens, dtype, n_kv, n_heads, d, ps=16, seed=0, layers=1, room=64, **kw):
        self.ps, self.dtype, self.dims = ps, dtype, (n_kv, n_heads, d)
        blocks = sum(-(-(n + room) // ps) for n in lens) + 8
        self.bk = FourBitBackend(layers, blocks, ps, n_kv, n_heads, d, device=DEV, dtype=dtype,
                                 **kw)
        self.alloc = BlockAllocator(blocks, ps)
        ids = self.alloc.allocate(blocks)
        random.Random(seed).shuffle(ids)
        self.alloc.free(ids)
        self.seqs = [SequenceBlocks(self.alloc, seq_id=i) for i in range(len(lens))]
        self.k = [torch.empty(0, n_kv, d, dtype=dtype) for _ in lens]
        self.v = [torch.empty(0, n_kv, d, dtype=dtype) for _ in lens]
        self.seed = seed
        if any(lens):
            self.append(lens)

    def append(self, counts, centre=1.0):
        """Grow the sequences and append layer 0's rows; the step's meta."""
        meta = grow_and_assemble(self.seqs, counts, self.ps, device=DEV)
        n_kv, _, d = self.dims
        self.seed += 1
        k = rows((sum(counts), n_kv, d), self.dtype, 2 * self.seed, centre)
        v = rows((sum(counts), n_kv, d), self.dtype, 2 * self.seed + 1, centre / 2)
        self.bk.append_kv(0, k.to(DEV), v.to(DEV), meta)
        at = 0
        for i, n in enumerate(counts):
            self.k[i] = torch.cat([self.k[i], k[at:at + n]])
            self.v[i] = torch.cat([self.v[i], v[at:at + n]])
            at += n
        return meta

    def q(self, counts, factor=1.0):
        _, hq, d = self.dims
        g = torch.Generator().manual_seed(self.seed + 77)
        return (torch.randn((sum(counts), hq, d), generator=g) * factor).to(self.dtype)

    def check(self, got, q, counts, scale, label=""):
        got, at = got.cpu(), 0
        for i, n in enumerate(counts):
            if n:
                want, bound = attend64(q[at:at + n], self.k[i], self.v[i], scale, self.dtype)
                assert_within(got[at:at + n], want, bound, f"{label} seq {i}")
            at += n


# ------------------------------------------------------------ append, read ---

@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("n_kv,d,ps", [(8, 64, 16), (3, 128, 16), (1, 256, 32), (2, 192, 48),
                                       (2, 64, 8), (5, 80, 16), (1, 2, 1), (4, 34, 7)])
def test_rows_come_back_as_defined(dtype, n_kv, d, ps):
    print(f"rows {dtype} {n_kv} {d} {ps}", flush=True)
    lens = [1, ps, 2 * ps + 3, 40]
    c = Cache(lens, dtype, n_kv, 2 * n_kv, d, ps)
    meta = c.append([3, 1, ps, 2])
    for s, k, v in zip(c.seqs, c.k, c.v):
        slots = [s.block_ids[p // ps] * ps + p % ps for p in range(s.num_tokens)]
        gk, gv = c.bk.read_kv(0, slots)
        same_bits(gk, held64(k), dtype)
        same_bits(gv, held64(v), dtype)
    gk, _ = c.bk.read_kv(0, meta.slot_mapping)
    assert gk.dtype is dtype and gk.shape[0] == meta.n_tokens
    c.bk.check_device_errors()


def special(dtype, d):
    """Rows whose groups are the cases that go wrong."""
    g = torch.Generator().manual_seed(5)
    x = torch.randn((24, 1, d), generator=g, dtype=torch.float64)
    x[0] = 0.0
    x[1] = -0.0
    x[2] = 0.7
    x[3, 0, 1] = math.nan
    x[4, 0, d - 1] = math.inf
    x[5, 0, 0] = -math.inf
    x[6] *= 2.0 ** -20                       # subnormal steps
    x[7] *= 2.0 ** -30                       # below float16's least
    x[8] *= 40000.0
    x[9, 0, 0], x[9, 0, 1] = 65504.0, -65504.0
    x[10] = torch.arange(d) % 31 / 2.0       # every other one on a border
    x[11] = 3.0 + torch.arange(d) % 31 * 2.0 ** -7
    x[12] = 1000.0 + x[12] * 2.0 ** -4
    x[13, 0, :] = 1.0
    x[13, 0, d // 2] = 1.0 + 2.0 ** -7
    x[14] = -torch.arange(d) % 16            # whole steps
    x[15] = 2.0 ** -24
    if dtype != F16:
        x[16] *= 1e30
        x[17, 0, 0] = 3e38
        x[18] = 1e5
        x[19] = -70000.0 - torch.arange(d)
        x[20] *= 1e-30
    return x.to(dtype)


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("d", [64, 128, 80])
def test_special_rows(dtype, d):
    print(f"special {dtype} {d}", flush=True)
    x = special(dtype, d)
    n = x.shape[0]
    bk = FourBitBackend(1, 4, 16, 1, 1, d, device=DEV, dtype=dtype)
    s = SequenceBlocks(BlockAllocator(4, 16), seq_id=0)
    meta = grow_and_assemble([s], [n], 16, device=DEV)
    bk.append_kv(0, x.to(DEV), x.flip(0).to(DEV), meta)
    k, v = bk.read_kv(0, meta.slot_mapping)
    same_bits(k, held64(x), dtype)
    same_bits(v, held64(x.flip(0)), dtype)


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
def test_many_random_rows_at_borders(dtype):
    """Rows of few distinct values, so that many elements lie on or next to a
    border between codes."""
    g = torch.Generator().manual_seed(9)
    x = torch.randint(-40, 41, (4096, 2, 64), generator=g).double() / 64
    x += torch.randint(-2, 3, x.shape, generator=g) * 2.0 ** -20
    x = x.to(dtype)
    bk = FourBitBackend(1, 256, 16, 2, 2, 64, device=DEV, dtype=dtype)
    s = SequenceBlocks(BlockAllocator(256, 16), seq_id=0)
    meta = grow_and_assemble([s], [4096], 16, device=DEV)
    bk.append_kv(0, x.to(DEV), (-x).to(DEV), meta)
    k, v = bk.read_kv(0, meta.slot_mapping)
    same_bits(k, held64(x), dtype)
    same_bits(v, held64(-x), dtype)


@pytest.mark.parametrize("tokens", [1, 5])
@pytest.mark.parametrize("shift", [0, 1])
def test_slices_of_a_projection(tokens, shift):
    """Strided rows, aligned to 16 bytes or not, give what their copies give."""
    n_kv, d = 2, 64
    wide = rows((tokens, 1, 8 * n_kv * d + shift), F16, 3).to(DEV).view(tokens, -1)
    k = wide[:, shift:shift + n_kv * d].view(tokens, n_kv, d)
    v = wide[:, 3 * n_kv * d + shift:][:, :n_kv * d].view(tokens, n_kv, d)
    bk = FourBitBackend(1, 4, 16, n_kv, n_kv, d, device=DEV)
    s = SequenceBlocks(BlockAllocator(4, 16), seq_id=0)
    meta = grow_and_assemble([s], [tokens], 16, device=DEV)
    bk.append_kv(0, k, v, meta)
    gk, gv = bk.read_kv(0, meta.slot_mapping)
    same_bits(gk, held64(k), F16)
    same_bits(gv, held64(v), F16)


def test_an_append_touches_its_own_rows_only():
    c = Cache([37, 20], BF16, 2, 4, 64)
    before = c.bk._pool.clone()
    free = c.alloc.allocate(1)[0]
    meta = c.append([1, 0])
    changed = (c.bk._pool != before).flatten(2)
    page = int(meta.slot_mapping[0]) // 16
    assert changed[0, :, :].any()
    others = torch.ones(c.bk.num_blocks, dtype=torch.bool)
    others[page] = False
    assert not (c.bk._pool != before)[0, :, others].any()
    slots = [c.seqs[0].block_ids[p // 16] * 16 + p % 16 for p in range(38)]
    same_bits(c.bk.read_kv(0, slots)[1], held64(c.v[0]), BF16)
    assert free != page


def test_slots_outside_the_pool_are_flagged():
    bk = FourBitBackend(1, 4, 16, 2, 2, 64, device=DEV)
    s = SequenceBlocks(BlockAllocator(4, 16), seq_id=0)
    meta = grow_and_assemble([s], [3], 16, device=DEV)
    meta.slot_mapping[1] = 64
    x = rows((3, 2, 64), F16, 1)
    bk.append_kv(0, x.to(DEV), x.to(DEV), meta)
    with pytest.raises(IndexError, match="slot_mapping"):
        bk.check_device_errors()
    k, v = bk.read_kv(0, [0, -1, 64, 2**40])
    assert not k[1:].any() and not v[1:].any()
    same_bits(k[:1], held64(x[:1]), F16)
    with pytest.raises(IndexError):
        bk.check_device_errors()


# --------------------------------------------------------------- attention ---

GEOMS = [(8, 32, 64, 16), (2, 8, 128, 16), (1, 8, 64, 32), (3, 12, 64, 16), (2, 2, 128, 64),
         (1, 16, 128, 16), (2, 10, 64, 16), (1, 24, 64, 16), (1, 32, 128, 16),
         # generic ones
         (2, 4, 80, 16), (1, 3, 256, 16), (2, 4, 64, 8), (1, 40, 64, 16), (2, 2, 64, 48)]


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("geom", GEOMS)
def test_single_tokens(dtype, geom):
    print(f"single {dtype} {geom}", flush=True)
    n_kv, hq, d, ps = geom
    lens = [0, 15, 16, 63, 64, 65, 255, 700]
    c = Cache([n for n in lens], dtype, n_kv, hq, d, ps)
    counts = [1] * len(lens)
    meta = c.append(counts)
    q = c.q(counts)
    c.check(c.bk.attend(q.to(DEV), 0, d ** -0.5, meta), q, counts, d ** -0.5)
    c.bk.check_device_errors()


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("geom", GEOMS[:4] + GEOMS[5:7] + GEOMS[9:10])
@pytest.mark.parametrize("counts", [[2, 3, 4, 1], [5, 1, 9, 17], [40, 1, 64, 130]])
def test_several_tokens(dtype, geom, counts):
    print(f"several {dtype} {geom} {counts}", flush=True)
    n_kv, hq, d, ps = geom
    c = Cache([0, 70, 300, 129], dtype, n_kv, hq, d, ps)
    meta = c.append(counts)
    q = c.q(counts)
    c.check(c.bk.attend(q.to(DEV), 0, d ** -0.5, meta), q, counts, d ** -0.5)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("pieces", [1, 6, 100])
@pytest.mark.parametrize("new", [1, 7])
def test_pieces_of_long_sequences(d, pieces, new):
    print(f"pieces {d} {pieces} {new}", flush=True)
    c = Cache([5000, 1, 2300], F16, 2, 8, d, compute_units=pieces)
    counts = [new, 1, new]
    meta = c.append(counts)
    q = c.q(counts)
    outs = [c.bk.attend(q.to(DEV), 0, d ** -0.5, meta) for _ in range(3)]
    assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], outs[2])
    c.check(outs[0], q, counts, d ** -0.5)


@pytest.mark.parametrize("d,hq", [(64, 8), (128, 8), (64, 32), (80, 4)])
@pytest.mark.parametrize("scale", [-0.25, 0.0, 1e-30])
def test_other_scales(d, hq, scale):
    c = Cache([100, 7], F16, 2, hq, d)
    counts = [1, 3]
    meta = c.append(counts)
    q = c.q(counts)
    c.check(c.bk.attend(q.to(DEV), 0, scale, meta), q, counts, scale)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("factor", [1e-4, 30.0])
@pytest.mark.parametrize("counts,units,d", [([1, 6], None, 64), ([40, 30], 1, 64), ([40, 30], 1, 128)])
def test_peaked_and_flat_weights(dtype, factor, counts, units, d):
    """Queries so large that one key takes all, and so small that none does."""
    print(f"peaked {dtype} {factor} {counts} {d}", flush=True)
    c = Cache([900, 333], dtype, 2, 8, d, compute_units=units)
    meta = c.append(counts)
    q = c.q(counts, factor)
    c.check(c.bk.attend(q.to(DEV), 0, 0.125, meta), q, counts, 0.125)


@pytest.mark.parametrize("grow", [2.0 ** -9, 2.0 ** 9])
@pytest.mark.parametrize("new,units", [(1, None), (9, None), (40, None), (40, 1)])
def test_values_that_grow_along_the_sequence(grow, new, units):
    """Steps of V that rise or fall by 2^9 between tiles: what keeps p step in
    range follows them."""
    c = Cache([0], F16, 2, 8, 64, room=700, compute_units=units)
    c.seqs[0].append(640)
    n = 640
    k = rows((n, 2, 64), F16, 1)
    v = rows((n, 2, 64), F16, 2).double() * torch.linspace(0, 1, n).mul(math.log(grow)).exp()[:, None, None]
    c.k, c.v = [k], [v.to(F16)]
    meta = make_meta(c.seqs, [n], 16, device=DEV)
    c.bk.append_kv(0, c.k[0].to(DEV), c.v[0].to(DEV), meta)
    counts = [new]
    meta = c.append(counts)
    q = c.q(counts)
    c.check(c.bk.attend(q.to(DEV), 0, 0.125, meta), q, counts, 0.125)


@pytest.mark.parametrize("new,units", [(1, None), (9, None), (40, 1)])
@pytest.mark.parametrize("d", [64, 128])
def test_groups_without_a_step(d, new, units):
    """Constant groups have a step of 0: all of V's, then V's of the first tiles alone."""
    for last in (False, True):
        c = Cache([0], F16, 2, 8, d, room=400, compute_units=units)
        n = 200
        c.seqs[0].append(n)
        k = rows((n, 2, d), F16, 1)
        v = rows((n, 2, 1), F16, 2).expand(n, 2, d).contiguous()
        if last:
            v[-30:] = rows((30, 2, d), F16, 3) * 2.0 ** -12
        c.k, c.v = [k], [v]
        c.bk.append_kv(0, k.to(DEV), v.to(DEV), make_meta(c.seqs, [n], 16, device=DEV))
        s = c.seqs[0]
        meta = make_meta(c.seqs, [new], 16, device=DEV)      # (the last rows' queries)
        q = c.q([new])
        c.check(c.bk.attend(q.to(DEV), 0, 0.125, meta), q, [new], 0.125, f"last {last}")
        assert s.num_tokens == n


@pytest.mark.parametrize("d,hq,counts,units", [(64, 8, [1, 3], None), (64, 16, [1, 1], None),
                                               (128, 2, [4, 16], None), (64, 8, [9, 14], None),
                                               (64, 8, [60, 40], 1), (128, 8, [60, 40], 1),
                                               (80, 4, [2, 5], None)])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_a_query_that_is_not_finite_is_alone(d, hq, counts, units, bad):
    print(f"query {d} {hq} {counts} {bad}", flush=True)
    c = Cache([150, 90], F16, 2, hq, d, compute_units=units)
    meta = c.append(counts)
    q = c.q(counts)
    spoilt = q.clone()
    spoilt[1, 1, 3] = bad
    out = c.bk.attend(spoilt.to(DEV), 0, d ** -0.5, meta)
    assert out[1, 1].isnan().all()
    out[1, 1] = c.bk.attend(q.to(DEV), 0, d ** -0.5, meta)[1, 1]
    c.check(out, q, counts, d ** -0.5)


def test_blocks_past_32_bits():
    """Block ids whose bytes lie beyond 2^32."""
    n_kv, d, blocks = 8, 128, 2**32 // 36864 + 40
    bk = FourBitBackend(1, blocks, 16 * 4, n_kv, 32, d, device=DEV)
    assert bk._block_bytes * (blocks - 20) > 2**32
    alloc = BlockAllocator(blocks, 64)
    low = alloc.allocate(blocks - 20)
    s = SequenceBlocks(alloc, seq_id=0)
    meta = grow_and_assemble([s], [300], 64, device=DEV)
    assert min(s.block_ids) >= blocks - 20 and len(low) == blocks - 20
    k, v = rows((300, n_kv, d), F16, 5), rows((300, n_kv, d), F16, 6)
    bk.append_kv(0, k.to(DEV), v.to(DEV), meta)
    gk, gv = bk.read_kv(0, meta.slot_mapping)
    same_bits(gk, held64(k), F16)
    same_bits(gv, held64(v), F16)
    g = torch.Generator().manual_seed(1)
    q = torch.randn((300, 32, d), generator=g).to(F16)
    for n in (1, 4, 300):
        part = make_meta([s], [n], 64, device=DEV)
        out = bk.attend(q[:n].to(DEV), 0, d ** -0.5, part).cpu()
        want, bound = attend64(q[:n], k, v, d ** -0.5, F16)
        assert_within(out, want, bound, f"{n} tokens")


@pytest.mark.parametrize("units", [None, 1])
@pytest.mark.parametrize("d,hq", [(64, 8), (128, 2), (64, 32), (80, 4)])
def test_rows_that_no_token_sees(d, hq, units):
    """What lies behind a sequence's end in its last page, and keys behind a
    token's position, may hold NaN."""
    c = Cache([0, 0], F16, 2, hq, d, compute_units=units)
    whole = [64 + 16, 32]
    for s, n in zip(c.seqs, whole):
        s.append(n)
    bad = torch.full((sum(whole), 2, d), math.nan, dtype=F16)
    c.bk.append_kv(0, bad.to(DEV), bad.to(DEV), make_meta(c.seqs, whole, 16, device=DEV))
    for s in c.seqs:
        s.num_tokens = 0
    counts = [67, 19]
    for s, n in zip(c.seqs, counts):
        s.num_tokens = n
    k, v = rows((86, 2, d), F16, 4), rows((86, 2, d), F16, 5)
    late = [66, 85]      # the last token's own row: only it sees the NaN
    k[late[1]] = math.nan
    v[late[0]] = math.nan
    for s in c.seqs:
        s.block_ids = s.block_ids[:-(-s.num_tokens // 16)]
    meta = make_meta(c.seqs, counts, 16, device=DEV)
    c.bk.append_kv(0, k.to(DEV), v.to(DEV), meta)
    q = c.q(counts)
    out = c.bk.attend(q.to(DEV), 0, d ** -0.5, meta).cpu()
    at = 0
    for n in counts:
        want, bound = attend64(q[at:at + n - 1], k[at:at + n - 1], v[at:at + n - 1], d ** -0.5, F16)
        assert_within(out[at:at + n - 1], want, bound)
        assert out[at + n - 1].isnan().all()
        at += n


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("counts", [[150, 1], [33, 200], [17, 129]])
@pytest.mark.parametrize("units", [None, 1])
def test_prompt_chunks(d, counts, units):
    """Many rows: chunks that end inside tiles of keys and of rows, over histories
    that do, beside other rows; as wide pieces of a whole card, as tall ones of a
    compute unit."""
    for n_kv, hq in ((2, 8), (1, 3), (1, 32)):
        print(f"chunks {d} {counts} {hq}", flush=True)
        c = Cache([130, 5], BF16 if n_kv == 2 else F16, n_kv, hq, d, room=300,
                  compute_units=units)
        meta = c.append(counts)
        q = c.q(counts)
        c.check(c.bk.attend(q.to(DEV), 0, d ** -0.5, meta), q, counts, d ** -0.5)
        c.check(c.bk.attend(q.to(DEV), 0, -0.1, meta), q, counts, -0.1)
        assert (c.bk._planned.args.n_tall > 0) == (units == 1)


@pytest.mark.parametrize("new,units", [(1, None), (5, None), (40, None), (40, 1)])
def test_values_next_to_the_largest_float16(new, units):
    """A group's values may reach past 65504 by a step's rounding."""
    c = Cache([0], BF16, 1, 4, 64, compute_units=units)
    n = 70
    c.seqs[0].append(n)
    k = rows((n, 1, 64), BF16, 1)
    v = (torch.rand((n, 1, 64), generator=torch.Generator().manual_seed(2)) * 65000).to(BF16)
    v[:, 0, 0], v[:, 0, 1] = 65280.0, 0.0
    c.k, c.v = [k], [v]
    c.bk.append_kv(0, k.to(DEV), v.to(DEV), make_meta(c.seqs, [n], 16, device=DEV))
    counts = [new]
    meta = c.append(counts)
    q = c.q(counts)
    c.check(c.bk.attend(q.to(DEV), 0, 0.125, meta), q, counts, 0.125)


@pytest.mark.parametrize("n,units", [(3, None), (40, None), (40, 1)])
def test_pages_outside_the_pool_among_many_rows(n, units):
    c = Cache([200], F16, 2, 8, 64, compute_units=units)
    meta = c.append([n])
    meta.kv_indices[3] = -1
    meta = dataclasses.replace(meta, host=None)
    q = c.q([n])
    out = c.bk.attend(q.to(DEV), 0, 0.125, meta).cpu()
    k, v = c.k[0].clone(), c.v[0].clone()
    k[48:64], v[48:64] = 0, 0
    want, bound = attend64(q, k, v, 0.125, F16)
    assert_within(out, want, bound)
    with pytest.raises(IndexError, match="kv_indices"):
        c.bk.check_device_errors()


def test_pages_outside_the_pool_read_as_zeros():
    c = Cache([200], F16, 2, 8, 64)
    meta = c.append([1])
    meta.kv_indices[3] = c.bk.num_blocks + 5
    meta = dataclasses.replace(meta, host=None)      # (its host arrays hold the old page)
    q = c.q([1])
    out = c.bk.attend(q.to(DEV), 0, 0.125, meta).cpu()
    keep = torch.ones(201, dtype=torch.bool)
    keep[48:64] = False
    k, v = c.k[0].clone(), c.v[0].clone()
    k[~keep], v[~keep] = 0, 0
    want, bound = attend64(q, k, v, 0.125, F16)
    assert_within(out, want, bound)
    with pytest.raises(IndexError, match="kv_indices"):
        c.bk.check_device_errors()


def test_a_batch_of_many_sequences():
    rng = random.Random(4)
    lens = [rng.randint(0, 600) for _ in range(100)]
    c = Cache(lens, BF16, 8, 32, 128)
    counts = [rng.choice([1, 1, 1, 4]) for _ in lens]
    meta = c.append(counts)
    q = c.q(counts)
    c.check(c.bk.attend(q.to(DEV), 0, 128 ** -0.5, meta), q, counts, 128 ** -0.5)


# --------------------------------------------- blocks, streams, graphs, steps ---

def test_copied_and_swapped_blocks_hold_the_same():
    c = Cache([50, 33], F16, 2, 8, 64, layers=2)
    bk = c.bk
    x = rows((50, 2, 64), F16, 8)
    meta = make_meta(c.seqs[:1], [50], 16, device=DEV)
    bk.append_kv(1, x.to(DEV), x.to(DEV), meta)
    spare = c.alloc.allocate(4)
    bk.copy_blocks(c.seqs[0].block_ids, spare)
    slots = [spare[p // 16] * 16 + p % 16 for p in range(50)]
    same_bits(bk.read_kv(0, slots)[0], held64(c.k[0]), F16)
    same_bits(bk.read_kv(1, slots)[1], held64(x), F16)
    space = KVSwapSpace(bk)
    h = space.swap_out("r", c.seqs[0])
    assert h.nbytes == 4 * bk.block_bytes()
    new = SequenceBlocks(c.alloc, seq_id=9)
    new.append(50)
    space.swap_in(h, new)
    slots = [new.block_ids[p // 16] * 16 + p % 16 for p in range(50)]
    same_bits(bk.read_kv(1, slots)[0], held64(x), F16)
    from llm_serving_layer_amd import MI355XBackend
    other = KVSwapSpace(MI355XBackend(2, bk.num_blocks, 16, 2, 8, 64, device=DEV))
    with pytest.raises(RuntimeError, match="the pool's are"):
        other.swap_in(h, new)
    space.release(h)


def test_other_streams():
    c = Cache([900, 40], F16, 2, 8, 64, compute_units=16)
    counts = [1, 1]
    meta = c.append(counts)
    q = c.q(counts).to(DEV)
    want = c.bk.attend(q, 0, 0.125, meta)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    got = []
    for i in range(6):
        with torch.cuda.stream(side if i % 2 else torch.cuda.current_stream()):
            got.append(c.bk.attend(q, 0, 0.125, meta))
    torch.cuda.synchronize()
    assert all(torch.equal(g, want) for g in got)


def test_captured_step_replays():
    c = Cache([1500, 40, 3], F16, 2, 8, 64, compute_units=16)
    counts = [1, 3, 1]
    meta = c.append(counts)
    q = c.q(counts).to(DEV)
    k = rows((5, 2, 64), F16, 50).to(DEV)
    v = rows((5, 2, 64), F16, 51).to(DEV)
    fresh = grow_and_assemble(c.seqs, [0, 0, 1], 16, device=DEV)
    with pytest.raises(RuntimeError, match="before a graph"):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            c.bk.attend(q[:1], 0, 0.125, fresh)
    torch.cuda.synchronize()
    c.bk.append_kv(0, k, v, meta)
    want = c.bk.attend(q, 0, 0.125, meta)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        c.bk.append_kv(0, k, v, meta)
        out = c.bk.attend(q, 0, 0.125, meta)
        held = c.bk.read_kv(0, meta.slot_mapping)
    for i in range(4):
        k.copy_(rows((5, 2, 64), F16, 60 + i))
        graph.replay()
        torch.cuda.synchronize()
        same_bits(held[0], held64(k), F16)
        got = out.clone()
        other = c.bk.attend(q[:1], 0, 0.125, fresh)      # another meta's plan between
        torch.cuda.synchronize()
        c.bk.append_kv(0, k, v, meta)
        want = c.bk.attend(q, 0, 0.125, meta)
        assert torch.equal(got, want) and torch.isfinite(other).all()


def test_decode_steps_from_a_prompt():
    """A prompt in chunks, then single tokens, each step against the definition."""
    c = Cache([0, 0], BF16, 2, 8, 128)
    for counts in ([30, 100], [70, 1], [1, 1], [1, 1], [3, 1], [1, 2]):
        meta = c.append(counts)
        q = c.q(counts)
        c.check(c.bk.attend(q.to(DEV), 0, 128 ** -0.5, meta), q, counts, 128 ** -0.5, str(counts))
    c.bk.check_device_errors()
