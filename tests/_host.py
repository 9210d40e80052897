"""
A backend without a GPU: CPU tensors stand in for the device's, the library's
planners run, and its launches are recorded instead of made, for tests of what
the host hands to them and in which order.
"""

from __future__ import annotations

import numpy as np
import torch

from llm_serving_layer_amd import BlockAllocator, SequenceBlocks, _native, backend
from llm_serving_layer_amd.backend import MI355XBackend

from ._util import grow_and_assemble

LAUNCHES = ("pkv_append_kv", "pkv_append_batch", "pkv_append_rotated_batch", "pkv_attend_batch",
            "pkv_attend_shared_batch", "pkv_attend_selected_batch", "pkv_page_bounds",
            "pkv_copy_blocks")
STREAM = 7   # the stand-in for the current stream's handle


class HostLib:
    """The library, with each launch noted in ``calls`` as (name, arguments, the
    struct it was given by address)."""

    def __init__(self):
        self._lib = _native.load()
        self.calls = []

    def __getattr__(self, name):
        if name not in LAUNCHES:
            return getattr(self._lib, name)
        kind = {"pkv_append_batch": _native.Batch, "pkv_attend_batch": _native.Batch,
                "pkv_append_rotated_batch": _native.Rotated,
                "pkv_attend_shared_batch": _native.Shared,
                "pkv_attend_selected_batch": _native.Selected}.get(name)

        def launch(*args):
            held = kind.from_buffer_copy(kind.from_address(args[0])) if kind else None
            self.calls.append((name, args, held))
            return _native.OK
        return launch


def host_backend(monkeypatch, n_heads=32, n_kv=8, d=64, dtype=torch.float16, blocks=512, ps=16,
                 layers=1, page_bounds=False, part_pages=17) -> MI355XBackend:
    monkeypatch.setattr(backend, "_raw_stream", lambda index: STREAM)
    monkeypatch.setattr(backend, "_current_stream", lambda device: STREAM)
    monkeypatch.setattr(backend, "_current_device", lambda: None)
    monkeypatch.setattr(backend, "_capturing", lambda: False)
    bk = object.__new__(MI355XBackend)
    bk._lib = HostLib()
    bk.device = torch.device("cpu")
    bk.num_layers, bk.num_blocks, bk.block_size = layers, blocks, ps
    bk.n_kv_heads, bk.n_heads, bk.head_dim = n_kv, n_heads, d
    bk.dtype, bk.groups, bk.part_pages = dtype, n_heads // n_kv, part_pages
    bk._code = backend._DTYPES[dtype]
    bk._prefill_tile = bk._lib.pkv_prefill_q_tile(n_heads, n_kv, d, ps, bk._code)
    bk.q_tile = bk._prefill_tile or backend.DEFAULT_Q_TILE
    bk._fast_decode = bool(bk._lib.pkv_decode_fast_path(n_heads, n_kv, d, ps, bk._code,
                                                        part_pages))
    bk._fuse_append = bk._fast_decode and not page_bounds
    bk._split_mixed = bk._fast_decode and bk._prefill_tile > 0
    bk._decode_wgs = 512             # what pkv_decode_workgroups gives on 256 compute units
    bk._pool = torch.zeros((layers, 2, blocks, ps, n_kv, d), dtype=dtype)
    bk._k_pool, bk._v_pool = ([bk._pool[l, i] for l in range(layers)] for i in range(2))
    bk._k_ptr, bk._v_ptr = ([t.data_ptr() for t in p] for p in (bk._k_pool, bk._v_pool))
    bk._block_bytes = ps * n_kv * d * bk._pool.element_size()
    bk._plane_bytes = blocks * bk._block_bytes
    bk._status = torch.zeros(1, dtype=torch.int32)
    bk._status_ptr = bk._status.data_ptr()
    bk._planned = bk._slot_cache = bk._pending = None
    bk._set_workspace(torch.zeros(0, dtype=torch.uint8))
    bk._captured = []
    bk.n_plans = bk.n_runs = 0
    if page_bounds:
        bk._bounds = torch.zeros((layers, 2, blocks, n_kv, d), dtype=dtype)
        bk._bounds_ptr = [(b[0].data_ptr(), b[1].data_ptr()) for b in bk._bounds]
    bk._upload = lambda a: torch.from_numpy(np.array(a))
    return bk


def sharing_batch(bk, pages=20, n=3):
    """A decode step of n sequences that begin with the same pages."""
    alloc = BlockAllocator(bk.num_blocks, bk.block_size)
    head = alloc.allocate(pages)
    seqs = []
    for i in range(n):
        s = SequenceBlocks(alloc, seq_id=i)
        alloc.incref(head)
        s.block_ids, s.num_tokens = list(head), pages * bk.block_size
        seqs.append(s)
    return grow_and_assemble(seqs, [1] * n, bk.block_size)
