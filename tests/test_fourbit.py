"""
The 4-bit cache without a GPU: the definition's own properties, what is refused,
and the planner.
"""

from __future__ import annotations

import ctypes as C

import numpy as np
import pytest
import torch

from llm_serving_layer_amd import _native
from llm_serving_layer_amd.fourbit import FourBitBackend

from ._fourbit import held64, quantise64


@pytest.mark.parametrize("scale", [1.0, 1e-5, 1e4])
def test_held_values_lie_half_a_step_away(scale):
    x = (torch.randn(500, 2, 128) * scale).half()
    _, step, _ = quantise64(x)
    gap = (held64(x) - x.double()).abs().reshape(500, 2, 2, 64)
    assert (gap <= step[..., None] * 0.5).all()


@pytest.mark.parametrize("n_kv,d,ps,want", [(8, 64, 16, 8 * 16 * 36), (8, 128, 16, 8 * 16 * 72),
                                            (1, 80, 16, 16 * 44), (3, 34, 7, 368 + 96),
                                            (1, 63, 16, 0), (1, 258, 16, 0), (0, 64, 16, 0)])
def test_block_bytes(n_kv, d, ps, want):
    assert _native.load().pkv_block_bytes_4bit(n_kv, d, ps) == want
    if want:
        assert FourBitBackend.estimate_pool_bytes(2, 10, ps, n_kv, d) == 2 * 2 * 10 * want


@pytest.mark.parametrize("args,kw,match", [
    ((1, 4, 16, 3, 8, 64), {}, "divisible"), ((0, 4, 16, 2, 8, 64), {}, "num_layers"),
    ((1, 4, 0, 2, 8, 64), {}, "block_size"), ((1, 4, 16, 2, 8, 63), {}, "odd"),
    ((1, 4, 16, 2, 8, 258), {}, "256"), ((1, 4, 16, 2, 8, 64), {"dtype": torch.int8}, "float16"),
    ((1, 2**28, 16, 2, 8, 64), {}, "32-bit"), ((1, 4, 16, 2, 8, 64), {"compute_units": 0}, "compute_units"),
    ((1, 4, 16, 2, 8, 64), {"device": "cpu"}, "GPU")])
def test_refused_geometries(args, kw, match):
    with pytest.raises(ValueError, match=match):
        FourBitBackend(*args, **kw)


def plan(kv_lens, query_lens, n_heads=32, n_kv=8, d=64, ps=16, dtype=_native.DTYPE_F16,
         compute_units=256, last=None, indptr=None):
    n = len(kv_lens)
    i32 = lambda a: np.ascontiguousarray(a, dtype=np.int32)  # noqa: E731
    cu = i32(np.concatenate([[0], np.cumsum(query_lens)]))
    if indptr is None:
        indptr = np.concatenate([[0], np.cumsum([-(-k // ps) for k in kv_lens])])
    indptr, kvl = i32(indptr), i32(kv_lens)
    last = i32([k % ps or ps for k in kv_lens] if last is None else last)
    ids = np.arange(int(indptr[-1]) if indptr[-1] > 0 else 1, dtype=np.int32) * 3
    args, needed = _native.FourBit(), C.c_int64()
    cap = 8
    for _ in range(2):
        items = np.empty(cap, np.int32)
        rc = _native.load().pkv_plan_4bit(
            cu.ctypes.data, indptr.ctypes.data, ids.ctypes.data, kvl.ctypes.data, last.ctypes.data, n, n_heads,
            n_kv, d, ps, dtype, compute_units, items.ctypes.data, cap, C.byref(needed),
            C.addressof(args))
        if rc != _native.ERR_CAPACITY or needed.value <= cap:
            break
        cap = needed.value
    _native.check(rc, "plan")
    return args, items[:needed.value].reshape(-1, 28).tolist()


@pytest.mark.parametrize("compute_units", [1, 16, 256, 100000])
@pytest.mark.parametrize("n_heads,n_kv", [(32, 8), (8, 8), (24, 1), (32, 1), (10, 2)])
def test_the_plan_covers_every_row_and_tile_once(compute_units, n_heads, n_kv):
    rng = np.random.default_rng(compute_units + n_heads)
    kv = [int(x) for x in rng.integers(1, 4000, 40)] + [1, 64, 65, 30000]
    ql = [int(min(k, rng.choice([1, 1, 1, 3, 8, 100]))) for k in kv]
    args, items = plan(kv, ql, n_heads, n_kv, compute_units=compute_units)
    groups = n_heads // n_kv
    assert args.n_few + args.n_wide + args.n_tall == len(items)
    seen, slots = {}, []
    cu, first = np.cumsum([0] + ql), np.cumsum([0] + [-(-k // 16) for k in kv])
    counters = {}
    # tall: the tiles along the sequence within the share of all as wide pieces
    step = max(1, 32 // groups)
    work = n_kv * sum(-(-(k - n + min(n, at + step)) // 64) for k, n in zip(kv, ql)
                      if n * groups > 64 for at in range(0, n, step))
    tall_seqs = {i for i, (k, n) in enumerate(zip(kv, ql)) if n * groups > 64
                 and 5 * -(-k // 64) * compute_units <= work}
    for i, (row, qn, pos, kvl, page, pages, t0, nt, slot, slot0, n, counter, *ids) in \
            enumerate(items):
        seq = int(np.searchsorted(cu, row, side="right")) - 1
        q = row - cu[seq]
        assert ids == [3 * (page + min(4 * t0 + u, pages - 1)) for u in range(16)]
        assert (kvl, page, pages) == (kv[seq], first[seq], -(-kv[seq] // 16))
        assert pos == kv[seq] - ql[seq] + q
        assert nt >= 1 and 1 <= qn and q + qn <= ql[seq]
        wide = i >= args.n_few
        tall = i >= args.n_few + args.n_wide
        assert wide or ql[seq] * groups <= 16
        assert tall == (seq in tall_seqs)
        assert qn * groups <= (128 if tall else 32 if wide else args.few_rows)
        assert tall or args.part_rows >= min(32 if wide else 16, qn * groups)
        assert not tall or n == 1
        assert (slot < 0) == (n == 1)
        if n > 1:
            assert slot0 <= slot < slot0 + n <= args.n_slots
            slots.append(slot)
            assert 0 <= counter < args.n_cuts and counters.setdefault(counter, slot0) == slot0
        seen.setdefault((seq, q, qn), []).append((t0, nt))
    assert sorted(slots) == list(range(args.n_slots))
    rows = {i: [] for i in range(len(kv))}
    for (seq, q, qn), tiles in seen.items():
        rows[seq].append((q, qn))
        at = 0
        for t0, nt in sorted(tiles):
            assert t0 == at
            at += nt
        assert at == -(-(kv[seq] - ql[seq] + q + qn) // 64)
    for seq, parts in rows.items():
        at = 0
        for q, qn in sorted(parts):
            assert q == at
            at += qn
        assert at == ql[seq]
    # longest first, in both parts
    for part in (items[:args.n_few], items[args.n_few:args.n_few + args.n_wide],
                 items[args.n_few + args.n_wide:]):
        assert [p[7] for p in part] == sorted((p[7] for p in part), reverse=True)
    assert len(counters) == len(set(counters.values())) == args.n_cuts
    need = _native.load().pkv_counter_bytes_4bit(args.n_cuts, n_kv) + args.n_slots * n_kv * args.part_rows * 66 * 4
    assert args.workspace_bytes == (need if args.n_slots else 0)


@pytest.mark.parametrize("kw", [{"d": 80}, {"dtype": _native.DTYPE_F32}, {"ps": 8}, {"ps": 48},
                                {"n_heads": 33, "n_kv": 1}, {"n_heads": 257, "n_kv": 257}])
def test_geometries_without_a_plan(kw):
    args, items = plan([100, 3], [1, 2], **kw)
    assert not items and args.n_few == args.n_wide == args.workspace_bytes == 0


@pytest.mark.parametrize("kw,match", [
    ({"last": [3, 3]}, "kv_last_page_len"), ({"indptr": [0, 6, 7]}, "pages"),
    ({"query_lens": [0, 1]}, "query_len"), ({"query_lens": [101, 1]}, "query_len"),
    ({"kv_lens": [0, 3], "query_lens": [0, 1], "indptr": [0, 0, 1]}, "kv_len"),
    ({"n_heads": 9}, "multiple"), ({"compute_units": 0}, "positive"), ({"d": 63}, "odd")])
def test_refused_plans(kw, match):
    kw = {"kv_lens": [100, 3], "query_lens": [1, 2], **kw}
    with pytest.raises(ValueError, match=match):
        plan(kw.pop("kv_lens"), kw.pop("query_lens"), **kw)


@pytest.mark.parametrize("change,match", [
    ({"dtype": 9}, "dtype"), ({"n_tokens": -1}, "negative"),
    ({"k": None}, "null"), ({"head_dim": 63}, "odd"), ({"n_tokens": 2**31}, "too many"),
    ({"n_tokens": 2**62}, "too many")])
def test_the_entry_refuses_before_it_launches(change, match):
    lib = _native.load()
    a = {"k_pool": 256, "v_pool": 256, "num_blocks": 4, "k": 256, "k_stride": 128, "v": 256,
         "v_stride": 128, "slots": 256, "n_tokens": 1, "n_kv": 2, "head_dim": 64, "ps": 16,
         "dtype": 0, **change}
    rc = lib.pkv_append_4bit(a["k_pool"], a["v_pool"], a["num_blocks"], a["k"], a["k_stride"],
                             a["v"], a["v_stride"], a["slots"], a["n_tokens"], a["n_kv"],
                             a["head_dim"], a["ps"], a["dtype"], None, None)
    with pytest.raises(ValueError, match=match):
        _native.check(rc, "append")


@pytest.mark.parametrize("change,match", [
    ({"items": None}, "no plan"), ({"n_few": -1, "n_wide": 2}, "no plan"),
    ({"n_slots": 2, "workspace_bytes": 8}, "workspace"), ({"n_tokens": 0}, "geometry"), ({"num_blocks": 0}, "geometry"),
    ({"kv_lens": None}, "null"), ({"head_dim": 80, "batch_indices": None}, "null")])
def test_attend_refuses_before_it_launches(change, match):
    b = _native.FourBit(num_blocks=4, n_seqs=1, n_tokens=1, n_heads=8, n_kv_heads=2, head_dim=64,
                        page_size=16, n_few=1, few_rows=4, part_rows=4)
    for f in ("cu_query_lens", "kv_indptr", "kv_indices", "kv_lens", "batch_indices", "items"):
        setattr(b, f, 256)
    for k, v in change.items():
        setattr(b, k, v)
    rc = _native.load().pkv_attend_4bit(C.addressof(b), 256, 256, 256, 256, 0.1, None)
    with pytest.raises(ValueError, match=match):
        _native.check(rc, "attend")


def host_backend():
    """A backend without a device, for the checks that come before any launch."""
    bk = object.__new__(FourBitBackend)
    bk.num_layers, bk.num_blocks, bk.block_size = 1, 8, 16
    bk.n_kv_heads, bk.n_heads, bk.head_dim, bk.groups = 2, 8, 64, 4
    bk.dtype, bk.device = torch.float16, torch.device("cpu")
    return bk


def test_refused_calls():
    from ._util import grow_and_assemble
    from llm_serving_layer_amd import BlockAllocator, SequenceBlocks
    import dataclasses
    bk = host_backend()
    s = SequenceBlocks(BlockAllocator(8, 16), seq_id=0)
    meta = grow_and_assemble([s], [3], 16)
    k = torch.zeros(3, 2, 64, dtype=torch.float16)
    for args, match in [((1, k, k, meta), "layer_idx"), ((None, k, k, meta), "layer_idx"),
                        ((0, k[:, :1], k, meta), "k has shape"), ((0, k, k[:2], meta), "v shape"),
                        ((0, k[:2], k[:2], meta), "slot_mapping"),
                        ((0, k, k, dataclasses.replace(meta, slot_mapping=None)), "slot_mapping")]:
        with pytest.raises(ValueError, match=match):
            bk.append_kv(*args)
    q = torch.zeros(3, 8, 64, dtype=torch.float16)
    for args, match in [((q, 1, 0.1, meta), "layer_idx"), ((q[:, :4], 0, 0.1, meta), "q has shape"),
                        ((q[:2], 0, 0.1, meta), "describes")]:
        with pytest.raises(ValueError, match=match):
            bk.attend(*args)
    for slots in (torch.zeros(2), torch.zeros(2, 2, dtype=torch.int32),
                  torch.zeros(2, dtype=torch.bool)):
        with pytest.raises(ValueError, match="slots"):
            bk.read_kv(0, slots)
    with pytest.raises(ValueError, match="layer_idx"):
        bk.read_kv(3, [0])
