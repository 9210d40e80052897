"""
The rotated append against the rotation in 64 bits: head layouts, odd head
and rotary dims, slices of a projection's output at any stride and address,
both pairings, one token to many, far positions; what it must leave alone,
flag and refuse; captured in a graph and on another stream.
"""

from __future__ import annotations

import dataclasses

import pytest
import torch

from llm_serving_layer_amd import BlockAllocator, RotaryTable, SequenceBlocks
from llm_serving_layer_amd.backend import MI355XBackend

from ._util import grow_and_assemble, make_meta, meta_to_device

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def turned(x, pos, table):
    """x's rotation in 64 bits, and the size of its error bound's terms."""
    r = table.rotary_dim
    f = table.frequencies64[None, :]
    z = torch.polar(torch.full((), table.factor, dtype=torch.float64, device=x.device),
                    pos.double()[:, None] * f)[:, None, :]
    y = x.double().clone()
    a, b = ((y[..., 0:r:2].clone(), y[..., 1:r:2].clone()) if table.interleaved
            else (y[..., :r // 2].clone(), y[..., r // 2:r].clone()))
    out, size = y.clone(), torch.zeros_like(y)
    ra, rb, ab = a * z.real - b * z.imag, b * z.real + a * z.imag, a.abs() + b.abs()
    for t, va, vb in ((out, ra, rb), (size, ab, ab)):
        if table.interleaved:
            t[..., 0:r:2], t[..., 1:r:2] = va, vb
        else:
            t[..., :r // 2], t[..., r // 2:r] = va, vb
    return out, size


def assert_turned(got, x, pos, table):
    """Within the one rounding to got's type (half a step of it: eps / 2 of the
    value, or half the smallest subnormal) and those of the 32-bit arithmetic:
    the table's entry, the product and the sum, 2^-24 each of at most |a| + |b|."""
    want, size = turned(x, pos, table)
    info = torch.finfo(got.dtype)
    inner = 4 * 2.0 ** -24 * abs(table.factor) * size
    bound = inner + info.eps / 2 * (want.abs() + inner) + info.tiny * info.eps / 2
    over = (got.double() - want).abs() - bound
    assert float(over.max()) <= 0, f"off by {float(over.max()):.3g} past the bound"


def table_of(n, r, interleaved=False, theta=10000.0, **kw):
    t = RotaryTable(n, r, theta=theta, interleaved=interleaved, device=DEV, **kw)
    t.frequencies64 = theta ** (-torch.arange(0, r, 2, dtype=torch.float64, device=DEV) / r)
    return t


def setup(n_heads, n_kv, d, dtype, counts, seed=0, blocks=64):
    bk = MI355XBackend(2, blocks, 16, n_kv, n_heads, d, device=DEV, dtype=dtype)
    alloc = BlockAllocator(blocks, 16)
    alloc.allocate(blocks)
    alloc.free([(7 * i) % blocks for i in range(blocks)])
    seqs = [SequenceBlocks(alloc, seq_id=i) for i in range(len(counts))]
    g = torch.Generator(device=DEV).manual_seed(seed)
    for p in (*bk.k_pool, *bk.v_pool):
        p.copy_(torch.randn(p.shape, generator=g, device=DEV))
    return bk, seqs, g


@pytest.mark.parametrize("n_heads, n_kv, d, r", [
    (32, 8, 64, 64), (32, 8, 128, 64), (8, 2, 128, 128), (4, 4, 80, 32), (8, 1, 256, 256),
    (6, 3, 24, 10), (2, 1, 3, 2), (5, 5, 72, 72)])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("layout", ["apart", "fused", "odd"])
def test_rows_turn_and_land_in_their_slots(n_heads, n_kv, d, r, dtype, interleaved, layout):
    print(f"rotated append {n_heads}/{n_kv}/{d}/{r} {dtype} {interleaved} {layout}", flush=True)
    table = table_of(700, r, interleaved)
    for counts in ([1], [130, 1, 17], [1] * 5):
        bk, seqs, g = setup(n_heads, n_kv, d, dtype, counts)
        grow_and_assemble(seqs, [20 + 9 * i for i in range(len(counts))], 16)
        meta = meta_to_device(grow_and_assemble(seqs, counts, 16), DEV)
        T, heads = sum(counts), n_heads + 2 * n_kv
        if layout == "odd":      # rows an odd number of elements apart, at an odd address
            x = torch.randn((T + 1) * (heads * d + 3), generator=g, device=DEV).to(dtype)
            x = x[1:].as_strided((T, heads * d), (heads * d + 3, 1))
        else:
            x = torch.randn((T, heads * d), generator=g, device=DEV).to(dtype)
        q, k, v = (p.view(T, -1, d) for p in x.split([n_heads * d, n_kv * d, n_kv * d], dim=1))
        if layout == "apart":
            q, k, v = q.contiguous(), k.contiguous(), v.contiguous()
        before = [(bk.k_pool[l].clone(), bk.v_pool[l].clone()) for l in range(2)]
        keep = x.clone()
        out = bk.append_kv_rotated(1, q, k, v, meta, table)
        bk.check_device_errors()
        assert out.shape == q.shape and out.dtype == dtype and out.is_contiguous()
        assert torch.equal(x, keep), "the inputs are left as they were"
        slots, pos = meta.slot_mapping.long(), meta.positions
        assert_turned(out, q, pos, table)
        kp, vp = bk.k_pool[1].view(-1, n_kv, d), bk.v_pool[1].view(-1, n_kv, d)
        assert_turned(kp[slots], k, pos, table)
        assert torch.equal(out[..., r:], q[..., r:]) and torch.equal(kp[slots][..., r:], k[..., r:])
        # every other row of both layers as it was, V copied exactly
        bk0, bv0 = before[1]
        bk0.view(-1, n_kv, d)[slots] = kp[slots]
        bv0.view(-1, n_kv, d)[slots] = v
        assert torch.equal(bk.k_pool[1], bk0) and torch.equal(bk.v_pool[1], bv0)
        assert torch.equal(bk.k_pool[0], before[0][0]) and torch.equal(bk.v_pool[0], before[0][1])


def test_far_positions_and_a_factor():
    """Positions of a long context: angles of 130 000 radians, from 64 bits."""
    bk, seqs, g = setup(8, 2, 64, torch.float32, [1], blocks=8200)
    seqs[0].append(131000)
    meta = grow_and_assemble(seqs, [33], 16, device=DEV)
    table = table_of(131033, 64, theta=500000.0, factor=1.1)
    q, k, v = (torch.randn(33, h, 64, generator=g, device=DEV) for h in (8, 2, 2))
    out = bk.append_kv_rotated(0, q, k, v, meta, table)
    assert_turned(out, q, meta.positions, table)
    assert_turned(bk.k_pool[0].view(-1, 2, 64)[meta.slot_mapping.long()], k, meta.positions, table)


def test_many_heads_share_a_token():
    """More units a token than a workgroup has threads."""
    bk, seqs, g = setup(256, 64, 128, torch.float16, [1, 1])
    meta = grow_and_assemble(seqs, [3, 1], 16, device=DEV)
    table = table_of(3, 128)
    q, k, v = (torch.randn(4, h, 128, generator=g, device=DEV).half() for h in (256, 64, 64))
    out = bk.append_kv_rotated(0, q, k, v, meta, table)
    assert_turned(out, q, meta.positions, table)
    kp = bk.k_pool[0].view(-1, 64, 128)[meta.slot_mapping.long()]
    assert_turned(kp, k, meta.positions, table)
    assert torch.equal(bk.v_pool[0].view(-1, 64, 128)[meta.slot_mapping.long()], v)


def test_other_dtypes_are_brought_to_the_pools():
    bk, seqs, g = setup(8, 2, 64, torch.bfloat16, [5])
    meta = grow_and_assemble(seqs, [5], 16, device=DEV)
    table = table_of(5, 64)
    q, k, v = (torch.randn(5, h, 64, generator=g, device=DEV) for h in (8, 2, 2))
    out = bk.append_kv_rotated(0, q, k, v, meta, table)
    same = bk.append_kv_rotated(1, q.bfloat16(), k.bfloat16(), v.bfloat16(), meta, table)
    assert torch.equal(out, same)
    slots = meta.slot_mapping.long()
    assert torch.equal(bk.k_pool[0].view(-1, 2, 64)[slots], bk.k_pool[1].view(-1, 2, 64)[slots])


@pytest.mark.parametrize("r", [64, 6])
def test_bad_slots_and_positions_are_skipped_and_flagged(r):
    """A token outside the pool or the table writes no row; one without a
    position gets a zero query; its neighbours are unharmed."""
    bk, seqs, g = setup(8, 2, 64, torch.float16, [4])
    meta = meta_to_device(make_meta(_grown(seqs, [4]), [4], 16), DEV, mirror=False)
    table = table_of(3, r)                    # position 3 has no row
    bad = meta.slot_mapping.clone()
    bad[0], bad[1] = 64 * 16, -1
    meta = dataclasses.replace(meta, slot_mapping=bad)
    q, k, v = (torch.randn(4, h, 64, generator=g, device=DEV).half() for h in (8, 2, 2))
    k0, v0 = bk.k_pool[0].clone(), bk.v_pool[0].clone()
    out = bk.append_kv_rotated(0, q, k, v, meta, table)
    with pytest.raises(IndexError, match="slot_mapping.*position outside"):
        bk.check_device_errors()
    assert_turned(out[:3], q[:3], meta.positions[:3], table)
    assert not out[3].any()
    s = int(bad[2])
    assert_turned(bk.k_pool[0].view(-1, 2, 64)[s:s + 1], k[2:3], meta.positions[2:3], table)
    k0.view(-1, 2, 64)[s], v0.view(-1, 2, 64)[s] = bk.k_pool[0].view(-1, 2, 64)[s], v[2]
    assert torch.equal(bk.k_pool[0], k0) and torch.equal(bk.v_pool[0], v0)


def _grown(seqs, counts):
    for s, n in zip(seqs, counts):
        s.append(n)
    return seqs


def test_captured_and_replayed_and_on_another_stream():
    bk, seqs, g = setup(8, 2, 64, torch.float16, [3, 40])
    meta = grow_and_assemble(seqs, [3, 40], 16, device=DEV)
    table = table_of(64, 64)
    q, k, v = (torch.randn(43, h, 64, generator=g, device=DEV).half() for h in (8, 2, 2))
    want = bk.append_kv_rotated(0, q, k, v, meta, table)
    kw, vw = bk.k_pool[0].clone(), bk.v_pool[0].clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        bk.k_pool[0].zero_()
        got = bk.append_kv_rotated(0, q, k, v, meta, table)
    torch.cuda.current_stream().wait_stream(side)
    slots = meta.slot_mapping.long()
    assert torch.equal(got, want)
    assert torch.equal(bk.k_pool[0].view(-1, 2, 64)[slots], kw.view(-1, 2, 64)[slots])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = bk.append_kv_rotated(0, q, k, v, meta, table)
    q0 = q.clone()
    for i in range(3):
        q.copy_(q0 * (i + 1))
        bk.k_pool[0].zero_()
        torch.cuda.synchronize()
        graph.replay()
        assert_turned(out, q, meta.positions, table)
        assert torch.equal(bk.k_pool[0].view(-1, 2, 64)[slots], kw.view(-1, 2, 64)[slots])
