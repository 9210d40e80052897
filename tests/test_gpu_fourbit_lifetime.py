"""Slots of the 4-bit cache's calls: those that a graph reads stay, and those past 32
bits are none of the pool's. Every launch is the backend's device's."""

from __future__ import annotations

import contextlib
import dataclasses
import gc

import pytest
import torch

from ._fourbit import held64
from .test_gpu_fourbit import DEV, F16, Cache, rows, same_bits

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
def test_a_captured_append_keeps_its_slots(dtype):
    """The meta goes once the graph is captured, and its memory is written over."""
    c = Cache([30, 7], F16, 2, 8, 64)
    meta = c.append([3, 2])
    slots = meta.slot_mapping.tolist()
    meta = dataclasses.replace(meta, slot_mapping=meta.slot_mapping.to(dtype).clone(), host=None)
    k, v = rows((5, 2, 64), F16, 50).to(DEV), rows((5, 2, 64), F16, 51).to(DEV)
    asked = torch.tensor(slots, dtype=dtype, device=DEV)
    c.bk.append_kv(0, k, v, meta)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        c.bk.append_kv(0, k, v, meta)
        held = c.bk.read_kv(0, asked)
    del meta, asked
    gc.collect()
    over = [torch.zeros(n, dtype=t, device=DEV) for t in (torch.int32, torch.int64)
            for n in (1, 2, 3, 5, 8) for _ in range(40)]
    torch.cuda.synchronize()
    for i in range(3):
        k.copy_(rows((5, 2, 64), F16, 60 + i))
        v.copy_(rows((5, 2, 64), F16, 70 + i))
        graph.replay()
        torch.cuda.synchronize()
        for got, want in ((held[0], k), (held[1], v), (c.bk.read_kv(0, slots)[0], k)):
            same_bits(got, held64(want), F16)
    assert len(over) == 400
    c.bk.check_device_errors()


def test_slots_past_32_bits_are_flagged():
    c = Cache([20], F16, 2, 8, 64)
    meta = c.append([2])
    before = c.bk._pool.clone()
    wide = torch.tensor([2**32 + 3, -2**32 + 4], device=DEV)
    x = rows((2, 2, 64), F16, 9).to(DEV)
    c.bk.append_kv(0, x, x, dataclasses.replace(meta, slot_mapping=wide, host=None))
    assert torch.equal(c.bk._pool, before)
    with pytest.raises(IndexError, match="slot_mapping"):
        c.bk.check_device_errors()
    k, v = c.bk.read_kv(0, wide)
    assert not k.any() and not v.any()
    with pytest.raises(IndexError):
        c.bk.check_device_errors()


def test_every_launch_is_made_on_the_backends_device():
    """The plan's upload too. (With one device: inside what makes it the current one.)"""
    c = Cache([40], F16, 2, 8, 64)
    meta = c.append([2])
    q = c.q([2])
    bk, inside, seen = c.bk, [0], []

    @contextlib.contextmanager
    def here():
        inside[0] += 1
        yield
        inside[0] -= 1

    def watched(name, call):
        def f(*args):
            seen.append((name, inside[0] > 0))
            return call(*args)
        return f

    class Library:
        def __init__(self, lib):
            self._lib = lib

        def __getattr__(self, name):
            return watched(name, getattr(self._lib, name))

    bk._on_device, bk._lib = here, Library(bk._lib)
    bk._upload = watched("upload", bk._upload)
    out = bk.attend(q.to(DEV), 0, 0.125, meta)
    bk.read_kv(0, meta.slot_mapping)
    c.check(out, q, [2], 0.125)
    assert {n for n, _ in seen} >= {"upload", "pkv_attend_4bit", "pkv_read_4bit"}
    assert all(ok for _, ok in seen), seen
