"""
The rotation table and the refusals of the rotated append, without a GPU.
"""

from __future__ import annotations

import math

import pytest
import torch

from llm_serving_layer_amd import RotaryTable, _native
from llm_serving_layer_amd.backend import MI355XBackend

from ._util import make_meta


def test_table_holds_cosines_and_sines_of_angles_in_64_bits():
    t = RotaryTable(131072, 128, theta=500000.0, device="cpu")
    assert t.table.shape == (131072, 2, 64) and t.table.dtype == torch.float32
    for p in (0, 1, 777, 131071):
        for i in (0, 1, 31, 63):
            a = p * 500000.0 ** (-2 * i / 128)
            # one rounding to 32 bits, and the angle's own in 64 (131071 radians: 2^-36)
            assert abs(float(t.cos[p, i]) - math.cos(a)) <= 2 ** -24 * abs(math.cos(a)) + 1e-10
            assert abs(float(t.sin[p, i]) - math.sin(a)) <= 2 ** -24 * abs(math.sin(a)) + 1e-10


def test_table_takes_frequencies_and_a_factor():
    f = [1.0, 0.25, 0.01]
    t = RotaryTable(10, 6, frequencies=f, factor=1.25, interleaved=True, device="cpu")
    want = 1.25 * torch.cos(torch.arange(10, dtype=torch.float64)[:, None]
                            * torch.tensor(f, dtype=torch.float64))
    assert torch.equal(t.cos, want.float()) and t.interleaved


@pytest.mark.parametrize("args, kw, match", [
    ((0, 8), {}, "max_positions"), ((4, 7), {}, "rotary_dim"), ((4, 0), {}, "rotary_dim"),
    ((4, 8), {"theta": 0.0}, "theta"), ((4, 8), {"frequencies": [1.0, 2.0]}, "frequencies")])
def test_table_refusals(args, kw, match):
    with pytest.raises(ValueError, match=match):
        RotaryTable(*args, device="cpu", **kw)


def test_library_refusals():
    """Refused on the host: nothing is launched, no pointer is followed."""
    lib = _native.load()

    def call(k_pool=16, max_positions=4, rotary_dim=8, n_heads=4, head_dim=8, dtype=0):
        return lib.pkv_append_rotated(k_pool, 16, 64, 16, 32, 16, 16, 32, 16, 32, 16, 16, 1, 16,
                                      max_positions, rotary_dim, 0, n_heads, 4, head_dim, dtype,
                                      None, None)
    for kw, match in (({"rotary_dim": 7}, "rotary_dim"), ({"rotary_dim": 10}, "rotary_dim"),
                      ({"rotary_dim": 0}, "rotary_dim"), ({"dtype": 9}, "dtype"),
                      ({"n_heads": 0}, "geometry"), ({"max_positions": 0}, "geometry"),
                      ({"k_pool": None}, "null")):
        with pytest.raises(ValueError, match=match):
            _native.check(call(**kw), "append_kv_rotated")


def _host_backend():
    bk = object.__new__(MI355XBackend)
    bk._lib = _native.load()
    bk.device = torch.device("cpu")
    bk.num_layers, bk.num_blocks, bk.block_size = 1, 64, 16
    bk.n_kv_heads, bk.n_heads, bk.head_dim = 2, 4, 8
    bk._planned, bk._slot_cache, bk._pending = None, None, None
    return bk


def test_backend_refusals():
    import dataclasses

    from llm_serving_layer_amd import (BlockAllocator, ScheduledSeq, SequenceBlocks,
                                       build_batch_meta)

    bk = _host_backend()
    s = SequenceBlocks(BlockAllocator(64, 16), seq_id=0)
    s.append(20)
    meta = build_batch_meta([ScheduledSeq(s, [0] * 20)], "cpu", 16)
    table = RotaryTable(32, 8, device="cpu")
    q, k = torch.zeros(20, 4, 8), torch.zeros(20, 2, 8)
    for args, kind, match in (
            ((1, q, k, k, meta, table), ValueError, "layer_idx"),
            ((0, q[:, :3], k, k, meta, table), ValueError, "q has shape"),
            ((0, q, k[:, :1], k, meta, table), ValueError, "k has shape"),
            ((0, q, k, k[:19], meta, table), ValueError, "v has shape"),
            ((0, q[:19], k[:19], k[:19], meta, table), ValueError, "tokens"),
            ((0, q, k, k, dataclasses.replace(meta, slot_mapping=None), table), ValueError,
             "slot_mapping"),
            ((0, q, k, k, meta, table.table), TypeError, "RotaryTable"),
            ((0, q, k, k, meta, RotaryTable(32, 10, device="cpu")), ValueError, "rotary_dim"),
            ((0, q, k, k, meta, RotaryTable(19, 8, device="cpu")), ValueError, "position 19")):
        with pytest.raises(kind, match=match):
            bk.append_kv_rotated(*args)
    bk.device = torch.device("meta")
    with pytest.raises(ValueError, match="rotation table is on"):
        bk.append_kv_rotated(0, q, k, k, meta, table)
    assert make_meta([s], [20], 16).host_arrays() is None   # (no mirror: the kernel flags it)
