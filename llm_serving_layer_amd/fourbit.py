"""
FourBitBackend — the attention-backend contract over a cache held in 4 bits:
``append_kv`` quantises, ``attend`` reads the codes. A pool of the same bytes
holds 3.6 times the tokens of a 16-bit one (head_dim 64: 36 bytes a row for 128),
and a decode step reads that much less.

Format: a row of a KV head is cut into groups of 64 elements (one group where
head_dim is no multiple of 64). A group keeps

* its zero: the largest float16 not above its least element;
* its step: the least float16 not below (largest element - zero) / 15;
* a 4-bit code an element: (x - zero) / step rounded to the nearest whole number
  (ties to even), at most 15;

and holds ``zero + code * step``, at most half a step from its element. Elements
beyond +-65504 are brought to that first; a group with a NaN or an infinity reads
as NaN throughout. Codes are decided in 64 bits, so they do not depend on the
kernel that writes them.

The same calls in the same order as ``MI355XBackend`` (``append_kv`` then
``attend``, per layer), the same checks, streams, capture rules and device error
word; ``copy_block(s)`` and ``KVSwapSpace`` move its blocks. ``k_pool`` /
``v_pool`` are the blocks' bytes; ``read_kv`` gives the values that slots hold.
Matrix-core kernels for head_dim 64 and 128, float16 and bfloat16, pages of 16
rows times a power of two, up to 32 query heads a KV head and 256 KV heads; others
(any even head_dim up to 256, float32, any page size) run generic ones.
"""

from __future__ import annotations

import ctypes as C

import numpy as np
import torch

from . import _native
from .backend import _DTYPES, PagedPool, _capturing, _current_stream
from .contract import BatchMeta

__all__ = ["FourBitBackend"]

class _Plan:
    """What ``attend`` keeps for one BatchMeta."""

    __slots__ = ("meta", "args", "ptr", "buffers", "stream")


class FourBitBackend(PagedPool):
    """Paged KV storage in 4 bits plus attention on gfx950 kernels."""

    _planned: _Plan | None = None

    def __init__(self, num_layers: int, num_blocks: int, block_size: int, n_kv_heads: int,
                 n_heads: int, head_dim: int, device: str | torch.device = "cuda:0",
                 dtype: torch.dtype = torch.float16, *, compute_units: int | None = None):
        if n_heads % n_kv_heads != 0:
            raise ValueError(
                f"n_heads={n_heads} must be divisible by n_kv_heads={n_kv_heads}; "
                "GQA maps query head h to KV head h // (n_heads // n_kv_heads)."
            )
        for name, val in (("num_layers", num_layers), ("num_blocks", num_blocks),
                          ("block_size", block_size), ("n_kv_heads", n_kv_heads),
                          ("n_heads", n_heads), ("head_dim", head_dim)):
            if val <= 0:
                raise ValueError(f"{name} must be positive, got {val}")
        if dtype not in _DTYPES:
            raise ValueError(f"FourBitBackend supports float16, bfloat16 and float32 rows, "
                             f"got {dtype}")
        if head_dim > 256 or head_dim % 2:
            raise ValueError(f"head_dim={head_dim} is odd or > 256: not supported")
        if num_blocks * block_size > 2**31 - 1:
            raise ValueError(f"{num_blocks} blocks of {block_size} rows pass the 32-bit slots")
        if compute_units is not None and compute_units < 1:
            raise ValueError(f"compute_units={compute_units} must be positive")
        try:
            self._lib = _native.load()
        except RuntimeError as exc:
            raise RuntimeError(f"FourBitBackend requires the gfx950 paged-KV library: {exc}"
                               ) from exc
        self.device = torch.device(device)
        if self.device.type != "cuda":
            raise ValueError(f"FourBitBackend requires a GPU device, got {self.device}")
        if self.device.index is None:
            self.device = torch.device("cuda", torch.cuda.current_device())
        self.num_layers, self.num_blocks, self.block_size = num_layers, num_blocks, block_size
        self.n_kv_heads, self.n_heads, self.head_dim = n_kv_heads, n_heads, head_dim
        self.dtype, self.groups = dtype, n_heads // n_kv_heads
        self._code = _DTYPES[dtype]
        # (what long sequences are cut to fill; the device's own by default)
        self.compute_units = compute_units or torch.cuda.get_device_properties(
            self.device).multi_processor_count
        self._block_bytes = self._bytes_of_block(n_kv_heads, head_dim, block_size)
        self._plane_bytes = num_blocks * self._block_bytes
        self._pool = torch.zeros((num_layers, 2, num_blocks, self._block_bytes),
                                 dtype=torch.uint8, device=self.device)
        self.k_pool = [self._pool[l, 0] for l in range(num_layers)]
        self.v_pool = [self._pool[l, 1] for l in range(num_layers)]
        self._k_ptr = [t.data_ptr() for t in self.k_pool]
        self._v_ptr = [t.data_ptr() for t in self.v_pool]
        self._status = torch.zeros(1, dtype=torch.int32, device=self.device)
        self._status_ptr = self._status.data_ptr()
        self._captured: list = []
        self.n_plans = 0
        self.n_runs = 0

    # -- accounting ---------------------------------------------------------------

    @staticmethod
    def _bytes_of_block(n_kv_heads: int, head_dim: int, block_size: int) -> int:
        size = int(_native.load().pkv_block_bytes_4bit(n_kv_heads, head_dim, block_size))
        if size <= 0:
            raise ValueError(f"no 4-bit block of {block_size} rows of {n_kv_heads} x {head_dim}")
        return size

    @staticmethod
    def estimate_pool_bytes(num_layers: int, num_blocks: int, block_size: int,
                            n_kv_heads: int, head_dim: int) -> int:
        return num_layers * 2 * num_blocks * FourBitBackend._bytes_of_block(
            n_kv_heads, head_dim, block_size)

    def workspace_bytes(self) -> int:
        """Partial results and arrival counters of the latest plan."""
        return 0 if self._planned is None else int(self._planned.args.workspace_bytes)

    # -- write path ---------------------------------------------------------------

    def _slots(self, slots: torch.Tensor) -> torch.Tensor:
        """Slots in 32 bits on the device; one that does not fit them is none of the
        pool's, and stays so."""
        if slots.dtype is torch.int64:
            slots = slots.clamp(-1, 2**31 - 1)
        return self._dev_i32(slots)

    def append_kv(self, layer_idx: int, k: torch.Tensor, v: torch.Tensor,
                  meta: BatchMeta) -> None:
        """
        Quantise this step's K/V into the pool through ``meta.slot_mapping`` (no
        two tokens may share a slot). ``k`` and ``v`` may be slices of one
        projection's output: any stride between tokens, heads one after another.
        Slots that a captured append reads stay as long as the backend does.
        """
        if layer_idx is None or not 0 <= layer_idx < self.num_layers:
            self._check_layer(layer_idx)
        slots = meta.slot_mapping
        if slots is None:
            raise ValueError("FourBitBackend.append_kv requires meta.slot_mapping")
        tokens = k.shape[0]
        if k.shape != (tokens, self.n_kv_heads, self.head_dim):
            raise ValueError(f"k has shape {tuple(k.shape)}, expected "
                             f"({tokens}, {self.n_kv_heads}, {self.head_dim})")
        if v.shape != k.shape:
            raise ValueError(f"v shape {tuple(v.shape)} != k shape {tuple(k.shape)}")
        if slots.shape[0] != tokens:
            raise ValueError(f"slot_mapping has {slots.shape[0]} entries but {tokens} tokens "
                             "were supplied")
        if not tokens:
            return
        k, v, slots = self._token_rows(k), self._token_rows(v), self._slots(slots)
        if k.data_ptr() % 16:
            k = k.clone(memory_format=torch.contiguous_format)
        if v.data_ptr() % 16:
            v = v.clone(memory_format=torch.contiguous_format)
        if _capturing():
            self._keep(meta.slot_mapping)
        row = self.n_kv_heads * self.head_dim   # (a single row's stride may be anything)
        with self._on_device():
            rc = self._lib.pkv_append_4bit(
                self._k_ptr[layer_idx], self._v_ptr[layer_idx], self.num_blocks, k.data_ptr(),
                k.stride(0) if tokens > 1 else row, v.data_ptr(),
                v.stride(0) if tokens > 1 else row, slots.data_ptr(), tokens, self.n_kv_heads,
                self.head_dim, self.block_size, self._code, self._status_ptr,
                _current_stream(self.device))
        if rc:
            _native.check(rc, "append_kv (4 bits)")

    def read_kv(self, layer_idx: int, slots) -> tuple[torch.Tensor, torch.Tensor]:
        """
        The values that the flat pool slots ``slots`` (``meta.slot_mapping``, or
        any 1-d tensor or list of ids) hold: two new ``(len(slots), n_kv_heads,
        head_dim)`` tensors in the backend's dtype, rounded to it once. Slots
        outside the pool give zeros and are flagged for ``check_device_errors``.
        """
        if layer_idx is None or not 0 <= layer_idx < self.num_layers:
            self._check_layer(layer_idx)
        if not isinstance(slots, torch.Tensor):
            slots = torch.tensor(slots, dtype=torch.int64)
        if slots.dim() != 1 or slots.is_floating_point() or slots.is_complex() \
                or slots.dtype is torch.bool:
            raise ValueError(f"slots must be a 1-d tensor of whole numbers, got {slots.dtype} of "
                             f"shape {tuple(slots.shape)}")
        if _capturing():
            self._keep(slots)
        slots = self._slots(slots)
        n = slots.shape[0]
        k = torch.empty((n, self.n_kv_heads, self.head_dim), dtype=self.dtype, device=self.device)
        v = torch.empty_like(k)
        if n:
            with self._on_device():
                rc = self._lib.pkv_read_4bit(
                    self._k_ptr[layer_idx], self._v_ptr[layer_idx], self.num_blocks,
                    slots.data_ptr(), n, k.data_ptr(), v.data_ptr(), self.n_kv_heads,
                    self.head_dim, self.block_size, self._code, self._status_ptr,
                    _current_stream(self.device))
            if rc:
                _native.check(rc, "read_kv")
        return k, v

    # -- read path ----------------------------------------------------------------

    def attend(self, q: torch.Tensor, layer_idx: int, scale: float,
               meta: BatchMeta) -> torch.Tensor:
        """
        Causal GQA attention over each sequence's full paged history, any number
        of new tokens a sequence. The result depends, in its last bits, on what
        shares the batch (long sequences are cut to fill the device), and on the
        keys that a token sees alone: NaN where one of them is.

        Weights times steps of V are rounded to float16, the matrix cores' input:
        by 2^-11 of a product at most, or, of products below some 2^-13 of the
        largest weight times the largest step among the token's keys, by 2^-24 of
        that. Scores (times scale) have to stay below some 2^26: from there on a
        reference in 32 bits lies a unit and more off the largest one, and with the
        matrix-core kernels an output may be NaN.

        To capture a graph, call it with the meta before, with no other meta's
        call between. Graphs captured with one meta share its buffers: neither
        their replays nor eager calls with it may overlap.
        """
        if layer_idx is None or not 0 <= layer_idx < self.num_layers:
            self._check_layer(layer_idx)
        tokens = q.shape[0]
        if q.shape != (tokens, self.n_heads, self.head_dim):
            raise ValueError(f"q has shape {tuple(q.shape)}, expected "
                             f"({tokens}, {self.n_heads}, {self.head_dim})")
        if meta.n_tokens != tokens:
            raise ValueError(f"meta describes {meta.n_tokens} tokens but q has {tokens}")
        p = self._planned
        if p is None or p.meta is not meta:
            with self._on_device():
                p = self._plan(meta)
        stream = self._enter(p)
        q = self._as_pool(q)
        if q.data_ptr() % 16:
            q = q.clone()
        out = torch.empty_like(q)
        with self._on_device():
            rc = self._lib.pkv_attend_4bit(p.ptr, q.data_ptr(), out.data_ptr(),
                                           self._k_ptr[layer_idx], self._v_ptr[layer_idx],
                                           float(scale), stream)
        if rc:
            _native.check(rc, "attend (4 bits)")
        self.n_runs += 1
        return out

    def _plan(self, meta: BatchMeta) -> _Plan:
        """The meta's launch plan, made at most once per forward pass."""
        self._refuse_capture("attend")
        ql, cu, kvl, indptr, last, indices, _ = self._host_index(meta, False)
        n = int(ql.shape[0])
        if n == 0:
            raise ValueError("attend needs at least one sequence")
        for name, field, want in (("cu_query_lens", cu, n + 1), ("kv_lens", kvl, n),
                                  ("kv_indptr", indptr, n + 1), ("kv_last_page_len", last, n)):
            if field.shape[0] != want:
                raise ValueError(f"{name} has {field.shape[0]} entries for {n} sequences")
        if bool(meta.is_prefill) != bool((ql > 1).any()):
            raise ValueError(
                f"BatchMeta.is_prefill={meta.is_prefill} disagrees with query_lens "
                f"(max={int(ql.max())}). is_prefill must be True iff some sequence "
                "contributes more than one token."
            )
        if int(cu[-1]) != meta.n_tokens:
            raise ValueError(f"cu_query_lens ends at {int(cu[-1])} but meta has "
                             f"{meta.n_tokens} positions")
        if int(meta.batch_indices.shape[0]) != meta.n_tokens:
            raise ValueError(f"batch_indices has {int(meta.batch_indices.shape[0])} entries "
                             f"for {meta.n_tokens} tokens")
        self._check_pages(kvl, indptr, last, int(indices.shape[0]))
        i32 = lambda a: np.ascontiguousarray(a, dtype=np.int32)  # noqa: E731
        arrays = [i32(a) for a in (cu, indptr, indices, kvl, last)]
        args = _native.FourBit()
        needed = C.c_int64()
        cap = 28 * (16 * self.compute_units + 2 * n + meta.n_tokens * self.groups // 16)
        while True:
            items = np.empty(cap, np.int32)
            rc = self._lib.pkv_plan_4bit(
                *(a.ctypes.data for a in arrays), n, self.n_heads, self.n_kv_heads,
                self.head_dim, self.block_size, self._code, self.compute_units, items.ctypes.data, cap,
                C.byref(needed), C.addressof(args))
            if rc != _native.ERR_CAPACITY or needed.value <= cap:
                break
            cap = needed.value
        _native.check(rc, "plan (4 bits)")
        p = _Plan()
        p.args = args
        fields = [self._dev_i32(t) for t in (meta.cu_query_lens, meta.kv_indptr, meta.kv_indices,
                                             meta.kv_lens, meta.batch_indices)]
        p.buffers = [*fields, self._upload(items[:max(needed.value, 1)])]
        at = [t.data_ptr() for t in p.buffers]
        (args.cu_query_lens, args.kv_indptr, args.kv_indices, args.kv_lens, args.batch_indices,
         args.items) = at
        if args.workspace_bytes:   # (the plan's own: its counters stay zero between launches)
            ws = torch.empty(args.workspace_bytes, dtype=torch.uint8, device=self.device)
            ws[:self._lib.pkv_counter_bytes_4bit(args.n_cuts, self.n_kv_heads)].zero_()
            args.workspace = ws.data_ptr()
            p.buffers.append(ws)
        args.num_blocks, args.status_word = self.num_blocks, self._status_ptr
        args.n_seqs, args.n_tokens = n, meta.n_tokens
        args.n_heads, args.n_kv_heads, args.head_dim = self.n_heads, self.n_kv_heads, self.head_dim
        args.page_size, args.dtype = self.block_size, self._code
        p.ptr = C.addressof(args)
        p.stream = _current_stream(self.device)
        p.meta = meta
        self._planned = p
        self.n_plans += 1
        return p

    def invalidate_plan(self) -> None:
        """Force the next ``attend`` to re-plan (and drop the cached meta)."""
        self._planned = None

    def reset(self) -> None:
        """Zero every pool and drop the plan. Tests only."""
        self._pool.zero_()
        self.invalidate_plan()

    def __repr__(self) -> str:
        mib = self.pool_bytes() / (1024 * 1024)
        return (f"FourBitBackend(layers={self.num_layers}, blocks={self.num_blocks}, "
                f"block_size={self.block_size}, kv_heads={self.n_kv_heads}, "
                f"heads={self.n_heads}, head_dim={self.head_dim}, dtype={self.dtype}, "
                f"device={self.device}, pool={mib:.1f} MiB)")
