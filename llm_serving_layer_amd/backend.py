"""
MI355XBackend — a third implementation of the attention-backend contract,
next to the reference's PagedTorchBackend (serving/backends/paged_torch.py)
and FlashInferBackend (serving/backends/flashinfer_backend.py), running on
hand-written gfx950 kernels through the C ABI in include/pagedkv.h.

Drop-in surface (same as both reference backends):

* constructor ``(num_layers, num_blocks, block_size, n_kv_heads, n_heads,
  head_dim, device="cuda:0", dtype=torch.float16, *, ...)`` with the same
  validation and messages (paged_torch.py:95-109), checked BEFORE the native
  library is touched so errors do not depend on the machine
  (flashinfer_backend.py:271-300);
* ``k_pool[l]`` / ``v_pool[l]``: per-layer contiguous
  ``[num_blocks, block_size, n_kv_heads, head_dim]`` tensors
  (paged_torch.py:127-137). Here they are views of ONE allocation laid out
  ``[num_layers, 2, num_blocks, block_size, n_kv_heads, head_dim]`` so that a
  whole-block copy across every layer, or a swap, is one kernel launch;
* ``append_kv`` / ``attend`` / ``copy_block`` and the accounting methods
  (paged_torch.py:139-207), plus ``workspace_bytes()``, ``invalidate_plan()``
  and the ``n_plans`` / ``n_runs`` counters (flashinfer_backend.py:354-394,
  678-688);
* plan once per ``BatchMeta`` identity, run once per layer
  (flashinfer_backend.py:566-676), including the ``is_prefill`` cross-check.

Beyond the reference's surface: ``append_kv_rotated`` (the position rotation
with the append), ``attend_shared`` (decode attention that reads shared pages
once) and, with ``page_bounds=True``, ``attend_selected`` (decode attention over
the pages whose key bounds allow the largest scores), ``key_bounds``,
``refresh_page_bounds`` and ``bounds_bytes``.

One launch per layer on decode steps: for a decode-shaped batch on the fast
geometry, ``append_kv`` records its rows and the following ``attend`` of the
same layer performs the append inside the attention kernel (the result is
exactly append-then-attend). Anything else that could observe the pool --
reading ``k_pool`` / ``v_pool``, another append or attend, ``copy_block(s)``,
``reset``, swapping, ``check_device_errors`` -- first launches the recorded
append on its own. A caller must not modify ``k`` / ``v`` in place between
``append_kv`` and the next backend call; that is detected (tensor version
counters) and raises.

Everything runs on torch's current stream of the backend's device. Not
thread-safe and not re-entrant, like the reference backends.
"""

from __future__ import annotations

import contextlib
import copy
import ctypes as C
from array import array
from operator import eq, index

import numpy as np
import torch

from . import _native
from .contract import BatchMeta
from .rotary import RotaryTable
from .upload import uploader
from .sizing import DEFAULT_PART_PAGES  # split-K pieces: 17 pages = 272 tokens

__all__ = ["MI355XBackend", "is_available", "unavailable_reason"]

_DTYPES = {torch.float16: _native.DTYPE_F16, torch.bfloat16: _native.DTYPE_BF16,
           torch.float32: _native.DTYPE_F32}

MAX_PART_PAGES = 64      # a partition's page ids are read by one wavefront
SELECTED_PART_PAGES = 8  # of chosen pages; what their kernel stages at a time
# Pieces (of 8 pages, were every list as long as the longest) up to which each of
# them gets a workgroup of its own; the streaming kernel takes more. us a call, workgroups against streaming: 64 pieces
# 20.4 and 29.7, 512 20.0 and 26.8, 1024 26.9 and 29.3 (head_dim 64) or 36.2 and
# 36.7 (128), 2048 40.7 and 34.5.
SELECTED_PIECES = 1024
# What attend_shared must save to be worth its tiles and its merge: a run of
# shared pages at least 4 pages long, in bytes a KV head more than 25 KiB a
# sequence (the part it adds), all runs together 16 MiB. us a call, attend against
# shared (8 KV heads of 64): 6 sequences over 96 pages 10.0 and 10.7, 200 over 8
# 28.5 and 30.4, 32 over 32 16.8 and 13.8, 256 over 128 130 and 39. The least lies
# on the side of attend: 2 over 512, 15.9 and 14.3, save 15.6 MiB and run it.
SHARED_MIN_PAGES, SHARED_PART_BYTES, SHARED_LEAST_BYTES = 4, 25 << 10, 16 << 20
SHARED_TILES = 256       # workgroups that share the work on a batch's shared pages
DEFAULT_Q_TILE = 64      # prefill tile when the geometry has no matrix-core kernel


def block_ids(ids) -> np.ndarray:
    """Block ids as an int64 array (one C loop over the list)."""
    if not isinstance(ids, (list, tuple)):
        ids = list(ids)
    try:
        return np.frombuffer(array("q", ids), dtype=np.int64)
    except (TypeError, OverflowError):   # not all Python integers
        ids = [int(i) for i in ids]
        try:
            return np.array(ids, dtype=np.int64).reshape(-1)
        except OverflowError:            # beyond 64 bits: no pool has such a block
            return np.array([min(max(i, -1), 2**63 - 1) for i in ids], dtype=np.int64)


# Pairs up to which a copy's ids are checked as Python lists. Host time of the
# checks, lists against arrays: 1 pair 5 and 15 us, 32 pairs 13 and 15 us, 64
# pairs 21 and 17 us, 4096 pairs 1130 and 170 us.
SHORT_COPY = 32


def copy_ids(src, dst, num_blocks: int) -> torch.Tensor:
    """The pairs of a block copy as int32 ids, every source and then every
    destination, pairs that copy a block onto itself left out; refuses ids
    outside the pool, repeated destinations and destinations that are also
    sources. The cost depends on the pairs alone, not on the pool: its blocks
    are marked in an array only where the pairs are many for its size
    (0.1 us a thousand blocks against 0.05 us a pair for a set)."""
    if not isinstance(src, (list, tuple)):
        src = list(src)
    if not isinstance(dst, (list, tuple)):
        dst = list(dst)
    short = len(src) <= SHORT_COPY
    if short:
        src, dst = [int(s) for s in src], [int(d) for d in dst]
    else:
        src, dst = block_ids(src), block_ids(dst)
    n = len(src)
    if n != len(dst):
        raise ValueError(f"{n} sources but {len(dst)} destinations")
    if n == 0:
        return torch.empty(0, dtype=torch.int32)
    if short:
        ids = src + dst
        outside = min(ids) < 0 or max(ids) >= num_blocks
    else:
        outside = (src.min() < 0 or src.max() >= num_blocks or dst.min() < 0
                   or dst.max() >= num_blocks)
    if outside:
        s, d = next((int(s), int(d)) for s, d in zip(src, dst)
                    if not (0 <= s < num_blocks and 0 <= d < num_blocks))
        raise IndexError(f"copy_block({s} -> {d}) outside [0, {num_blocks})")
    if short:
        if any(map(eq, src, dst)):
            pairs = [(s, d) for s, d in zip(src, dst) if s != d]
            src, dst = [s for s, _ in pairs], [d for _, d in pairs]
            ids = src + dst
        to = set(dst)
        clash = len(to) != len(dst) or not to.isdisjoint(src)
    else:
        move = src != dst
        if not move.all():
            src, dst = src[move], dst[move]
        if num_blocks <= 256 * n:
            written = np.zeros(num_blocks, dtype=bool)
            written[dst] = True
            clash = np.count_nonzero(written) != len(dst) or written[src].any()
        else:
            to = set(dst.tolist())
            clash = len(to) != len(dst) or not to.isdisjoint(src.tolist())
    if clash:
        raise ValueError("copy_blocks needs distinct destinations that are not also sources")
    if short:
        return torch.tensor(ids, dtype=torch.int32)
    return torch.from_numpy(np.concatenate([src, dst]).astype(np.int32))


def is_available() -> bool:
    """True if the gfx950 library loads in this process (says nothing of a GPU)."""
    return _native.available()


def unavailable_reason() -> str | None:
    return _native.reason()


_HERE = contextlib.nullcontext()
# (the plain queries: torch.cuda's own check first whether it is initialised)
_current_device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)
_capturing = getattr(torch._C, "_cuda_isCurrentStreamCapturing",
                     torch.cuda.is_current_stream_capturing)

_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def _current_stream(device: torch.device) -> int:
    """Handle of torch's current stream on ``device`` (the raw-handle query
    skips building a Stream object on every launch)."""
    if _raw_stream is not None and device.index is not None:
        return _raw_stream(device.index)
    return torch.cuda.current_stream(device).cuda_stream


class _Plan:
    """Device-side metadata and launch plan for one BatchMeta (one step)."""

    __slots__ = ("meta", "use_prefill", "slots", "indptr", "indices", "kv_lens", "cu_q",
                 "bidx", "plan", "n_work", "n_slots", "stride", "n_tokens", "n_seqs", "fusable",
                 "dec", "batch", "batch_ptr")


class _DecodeRows:
    """The one-token sequences of a mixed batch, run through the decode kernel:
    their decode plan as a batch of their own, whose items name their token
    rows in the whole batch's q and out (the plan is all the kernel reads)."""

    __slots__ = ("plan", "n", "n_work", "n_slots", "stride")


class _Pending:
    """An append_kv whose rows will be written by the next launch."""

    __slots__ = ("layer", "k", "v", "meta", "slots", "stream", "kver", "vver")


class _Rows:
    """Where one BatchMeta's new rows go, on the device (``append_kv_rotated``)."""

    __slots__ = ("meta", "slots", "positions", "complete", "table", "args", "ptr", "buffers",
                 "stream")


class _Shared:
    """What ``attend_shared`` keeps for one BatchMeta. Where nothing is worth
    sharing ``n_tiles`` is 0; ``whole`` is the plan ``attend`` ran it by, once it
    has."""

    __slots__ = ("meta", "n", "n_tiles", "n_merges", "tiles", "plan", "indices", "slots", "n_work", "n_slots",
                 "stride", "ws", "fusable", "args", "ptr", "buffers", "stream", "whole")


class _Selected:
    """What ``attend_selected`` keeps for one BatchMeta and page budget."""

    __slots__ = ("meta", "asked", "n", "max_pages", "indptr", "indices", "kv_lens", "scores",
                 "ids", "ordinals", "words", "places", "plan", "part", "ws", "width", "args", "ptr", "buffers", "stream")


class PagedPool:
    """What the backends share: one pool ``[num_layers, 2, num_blocks, ...]`` whose
    blocks move as bytes, the checks of a meta's index fields, and the order of
    launches on streams and in graphs."""

    _bounds: torch.Tensor | None = None

    def _flush(self) -> None:
        """Launch what an earlier call left to a later one."""

    def pool_bytes(self) -> int:
        return self.num_layers * 2 * self._plane_bytes

    def block_bytes(self) -> int:
        return self.pool_bytes() // self.num_blocks

    def tokens_capacity(self) -> int:
        return self.num_blocks * self.block_size

    def _check_layer(self, layer_idx) -> None:
        if layer_idx is None or not 0 <= layer_idx < self.num_layers:
            raise ValueError(f"layer_idx {layer_idx} out of range [0, {self.num_layers})")

    def _dev_i32(self, t: torch.Tensor) -> torch.Tensor:
        # (as it is, without conversion calls, where nothing is to be done)
        if t.dtype is torch.int32 and t.get_device() == self.device.index and t.is_contiguous():
            return t
        return t.to(device=self.device, dtype=torch.int32).contiguous()

    def _as_pool(self, x: torch.Tensor) -> torch.Tensor:
        # (a tensor already in the pool dtype, contiguous and on this device is
        # used as it is, without a conversion call per launch)
        if x.dtype is self.dtype and x.get_device() == self.device.index and x.is_contiguous():
            return x
        return x.to(device=self.device, dtype=self.dtype).contiguous()

    def check_device_errors(self) -> None:
        """
        Declared check point: synchronise and raise if any kernel since the
        last check skipped an out-of-range slot, page or block id.
        """
        self._flush()
        bits = int(self._status.item())
        if bits:
            self._status.zero_()
            what = []
            if bits & _native.STATUS_BAD_SLOT:
                what.append("slot_mapping entry outside the pool")
            if bits & _native.STATUS_BAD_PAGE:
                what.append("kv_indices entry outside [0, num_blocks)")
            if bits & _native.STATUS_BAD_BLOCK:
                what.append("block id outside [0, num_blocks)")
            if bits & _native.STATUS_BAD_POSITION:
                what.append("position outside the rotation table")
            raise IndexError("device kernels skipped invalid ids: " + "; ".join(what))

    def copy_block(self, src: int, dst: int) -> None:
        """Duplicate one block's KV in every layer (copy-on-write)."""
        if not (0 <= src < self.num_blocks and 0 <= dst < self.num_blocks):
            raise IndexError(f"copy_block({src} -> {dst}) outside [0, {self.num_blocks})")
        if src == dst:
            return
        self.copy_blocks([src], [dst])

    def copy_blocks(self, src, dst) -> None:
        """
        Batched ``copy_block``: one launch for every (src, dst) pair, every
        layer, K and V. Destinations must be distinct and must not appear among
        the sources (so the result cannot depend on the order of the pairs).
        """
        ids = copy_ids(src, dst, self.num_blocks)
        n = ids.shape[0] // 2
        if n == 0:
            return
        self._flush()
        # pinned, so the upload queues on the stream without a host wait
        ids = ids.pin_memory().to(self.device, non_blocking=True)
        with self._on_device():
            self._launch_copy(self._pool.data_ptr(), self._plane_bytes, self._block_bytes, ids, n)
            if self._bounds is not None:
                row = self._block_bytes // self.block_size
                self._launch_copy(self._bounds.data_ptr(), self.num_blocks * row, row, ids, n)

    def _launch_copy(self, pool: int, plane: int, block: int, ids: torch.Tensor, n: int) -> None:
        rc = self._lib.pkv_copy_blocks(pool, self.num_layers, plane, block, self.num_blocks,
                                       ids.data_ptr(), ids.data_ptr() + 4 * n, n,
                                       self._status.data_ptr(), _current_stream(self.device))
        _native.check(rc, "copy_blocks")

    def _token_rows(self, x: torch.Tensor) -> torch.Tensor:
        """x in the pool dtype on this device, heads contiguous in each token's
        row, rows any distance apart."""
        if x.dtype is self.dtype and x.get_device() == self.device.index:
            _, head, one = x.stride()
            if one == 1 and head == self.head_dim:
                return x
        return x.to(device=self.device, dtype=self.dtype).contiguous()

    def _on_device(self):
        """Launches go to this backend's device, whichever is current."""
        if _current_device() == self.device.index:
            return _HERE
        return torch.cuda.device(self.device)

    def _counted_workspace(self, need: int, n: int) -> torch.Tensor:
        """A workspace whose arrival counters (at its front) are zero."""
        ws = torch.empty(need, dtype=torch.uint8, device=self.device)
        if need:
            ws[:4 * n * self.n_kv_heads].zero_()
        return ws

    def _check_pages(self, kvl, indptr, last, n_pages: int) -> None:
        """Every sequence's page list fits its length (ValueError naming the first
        that does not)."""
        ps = self.block_size
        if int(indptr[0]) != 0 or int(indptr[-1]) != n_pages:
            raise ValueError(f"kv_indptr spans [{int(indptr[0])}, {int(indptr[-1])}) but "
                             f"kv_indices holds {n_pages} pages")
        need = (kvl + ps - 1) // ps
        bad = (kvl < 1) | (np.diff(indptr) != need) | (last != kvl - (need - 1) * ps)
        if bad.any():
            i = int(np.argmax(bad))
            raise ValueError(f"seq {i}: kv_len={int(kvl[i])} with "
                             f"{int(indptr[i + 1] - indptr[i])} pages of {ps} and "
                             f"kv_last_page_len={int(last[i])} disagree")

    def _refuse_capture(self, what: str) -> None:
        """What a plan uploads while a graph is captured is there only once the
        graph has run, but the plan stays for eager calls too."""
        if _capturing():
            raise RuntimeError(f"{what} has to plan this meta before a graph is captured: call "
                               "it once with the meta (and the same arguments), then capture")

    def _enter(self, p, slots=None) -> int:
        """The current stream's handle, ordered behind the plan's last launch:
        launches of one plan share its buffers. A plan that a graph captures, and
        the slots of an append that it landed, stay as long as the backend does."""
        stream = _current_stream(self.device)
        if _capturing():
            self._keep(p)
            if slots is not None:
                self._keep(slots)
        elif p.stream != stream:
            cur, ev = torch.cuda.current_stream(self.device), torch.cuda.Event()
            ev.record(torch.cuda.ExternalStream(p.stream, device=self.device))
            cur.wait_event(ev)
            for t in p.buffers:     # not reused before this stream is done with them
                t.record_stream(cur)
            p.stream = stream
        return stream

    def _keep(self, read) -> None:
        """What a graph being captured reads stays as long as the backend does."""
        if not any(c is read for c in self._captured):
            self._captured.append(read)

    @staticmethod
    def _host_index(meta: BatchMeta, with_slots: bool) -> tuple:
        """The meta's index fields on the host: query_lens, cu_query_lens,
        kv_lens, kv_indptr, kv_last_page_len, kv_indices and, if asked for,
        slot_mapping (else None)."""
        names = ["query_lens", "cu_query_lens", "kv_lens", "kv_indptr", "kv_last_page_len",
                 "kv_indices"] + ["slot_mapping"] * with_slots
        mirror = meta.host_arrays()
        if mirror is not None:
            # the assembler's own host arrays: no device read-back
            out = [mirror[k] for k in names]
        else:
            # ONE device->host transfer for everything the host plan reads.
            parts = [getattr(meta, k).reshape(-1).to(torch.int64) for k in names]
            host = torch.cat(parts).cpu().numpy()
            out = np.split(host, np.cumsum([t.shape[0] for t in parts])[:-1])
        return (*out, *[None] * (not with_slots))

    def _upload(self, a: np.ndarray) -> torch.Tensor:
        """Host array to the device through a pinned ring buffer, uploaded by a
        kernel on the current stream without a host wait (upload.py)."""
        return uploader(self.device).array(a)


class MI355XBackend(PagedPool):
    """Paged KV storage plus attention on gfx950 kernels."""

    _rows: _Rows | None = None
    _selected: _Selected | None = None
    _budgets: tuple[_Selected, ...] = ()   # the latest meta's plans, one a page budget
    _shared: _Shared | None = None

    def __init__(self, num_layers: int, num_blocks: int, block_size: int, n_kv_heads: int,
                 n_heads: int, head_dim: int, device: str | torch.device = "cuda:0",
                 dtype: torch.dtype = torch.float16, *,
                 part_pages: int = DEFAULT_PART_PAGES, q_tile: int | None = None,
                 fuse_append: bool = True, decode_workgroups_per_cu: int = 2,
                 decode_workgroups: int | None = None, decode_workspace_bytes: int = 0,
                 page_bounds: bool = False):
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
            raise ValueError(f"MI355XBackend supports float16, bfloat16 and float32 pools, "
                             f"got {dtype}")
        if head_dim > 256:
            raise ValueError(f"head_dim={head_dim} > 256 is not supported")
        if q_tile is not None and q_tile < 1:
            raise ValueError(f"q_tile={q_tile} must be positive")
        if not 1 <= part_pages <= MAX_PART_PAGES:
            raise ValueError(f"part_pages={part_pages} must be in [1, {MAX_PART_PAGES}]")
        if decode_workgroups_per_cu < 1:
            raise ValueError(f"decode_workgroups_per_cu={decode_workgroups_per_cu} must be "
                             "positive")
        if decode_workgroups is not None and decode_workgroups < 1:
            raise ValueError(f"decode_workgroups={decode_workgroups} must be positive")
        if decode_workspace_bytes < 0:
            raise ValueError(f"decode_workspace_bytes={decode_workspace_bytes} must be >= 0")
        try:
            self._lib = _native.load()
        except RuntimeError as exc:
            raise RuntimeError(
                f"MI355XBackend requires the gfx950 paged-KV library: {exc}\n"
                "Use PagedTorchBackend (the correctness oracle) instead, or build the "
                "library. Check availability without raising via "
                "llm_serving_layer_amd.backend.is_available()."
            ) from exc
        self.device = torch.device(device)
        if self.device.type != "cuda":
            raise ValueError(f"MI355XBackend requires a GPU device, got {self.device}. "
                             "PagedTorchBackend is the CPU path.")
        if self.device.index is None:
            self.device = torch.device("cuda", torch.cuda.current_device())

        self.num_layers, self.num_blocks, self.block_size = num_layers, num_blocks, block_size
        self.n_kv_heads, self.n_heads, self.head_dim = n_kv_heads, n_heads, head_dim
        self.dtype = dtype
        self.groups = n_heads // n_kv_heads
        self.part_pages = part_pages
        # The matrix-core prefill kernel owns 128 query rows (tokens x heads)
        # of one KV head; other geometries run the generic kernel.
        self._prefill_tile = int(self._lib.pkv_prefill_q_tile(
            n_heads, n_kv_heads, head_dim, block_size, _DTYPES[dtype]))
        self.q_tile = q_tile or self._prefill_tile or DEFAULT_Q_TILE
        self._code = _DTYPES[dtype]
        self._fast_decode = bool(self._lib.pkv_decode_fast_path(
            n_heads, n_kv_heads, head_dim, block_size, self._code, part_pages))
        # (with page bounds the append runs first: the bounds follow from its rows)
        self._fuse_append = fuse_append and self._fast_decode and not page_bounds
        # The decode grid: every bin of the plan a resident workgroup (per
        # group of KV heads), so none waits for a slot. ``decode_workgroups``
        # overrides the count (tests force many sequences into a bin with it).
        self._decode_wgs = 0
        if self._fast_decode:
            with torch.cuda.device(self.device):
                self._decode_wgs = int(self._lib.pkv_decode_workgroups(
                    n_heads, n_kv_heads, head_dim, self._code, decode_workgroups_per_cu))
            if self._decode_wgs <= 0:
                raise RuntimeError("pkv_decode_workgroups found no resident decode workgroup "
                                   "on this device")
            if decode_workgroups is not None:
                self._decode_wgs = decode_workgroups
        # A mixed batch (prefill chunks beside one-token decodes) runs its
        # decodes through the decode kernel, so a decode step's bits do not
        # depend on whether prefills share its batch.
        self._split_mixed = self._fast_decode and self.q_tile == self._prefill_tile > 0

        self._pool = torch.zeros((num_layers, 2, num_blocks, block_size, n_kv_heads, head_dim),
                                 dtype=dtype, device=self.device)
        self._k_pool = [self._pool[l, 0] for l in range(num_layers)]
        self._v_pool = [self._pool[l, 1] for l in range(num_layers)]
        # the pools never move: their addresses are taken once
        self._k_ptr = [t.data_ptr() for t in self._k_pool]
        self._v_ptr = [t.data_ptr() for t in self._v_pool]
        self._block_bytes = block_size * n_kv_heads * head_dim * self._pool.element_size()
        self._plane_bytes = num_blocks * self._block_bytes
        self._status = torch.zeros(1, dtype=torch.int32, device=self.device)
        self._status_ptr = self._status.data_ptr()
        # The split-K workspace. A pool sized by sizing.plan_kv_pool passes its
        # workspace_bytes here, so no batch within that plan's limits ever
        # allocates at run time; a plan that needs more grows it.
        self._planned: _Plan | None = None
        self._set_workspace(torch.zeros(decode_workspace_bytes, dtype=torch.uint8,
                                        device=self.device))
        # Per page and KV head the elementwise minimum and maximum of its keys
        # (attend_selected's cheap score), laid out like a pool of one-row pages.
        if page_bounds:
            self._bounds = torch.zeros((num_layers, 2, num_blocks, n_kv_heads, head_dim),
                                       dtype=dtype, device=self.device)
            half = self._bounds.stride(1) * self._bounds.element_size()
            at = self._bounds.data_ptr()
            self._bounds_ptr = [(at + 2 * l * half, at + (2 * l + 1) * half)
                                for l in range(num_layers)]
        # what graphs were captured with: it stays as long as the backend
        self._captured: list = []
        self._slot_cache: tuple[BatchMeta, torch.Tensor] | None = None
        self._pending: _Pending | None = None
        self.n_plans = 0
        self.n_runs = 0

    # -- the pools (reading them first lands any deferred append) ---------------

    @property
    def k_pool(self) -> list[torch.Tensor]:
        self._flush()
        return self._k_pool

    @property
    def v_pool(self) -> list[torch.Tensor]:
        self._flush()
        return self._v_pool

    @property
    def key_bounds(self) -> list[torch.Tensor]:
        """Per layer ``(2, num_blocks, n_kv_heads, head_dim)``: the elementwise
        minimum and maximum of each page's keys, renewed when an append
        completes the page, when blocks are copied and swapped in, and by
        ``refresh_page_bounds``. Needs ``page_bounds=True``."""
        self._need_bounds("key_bounds")
        self._flush()
        return list(self._bounds.unbind(0))

    def _need_bounds(self, what: str) -> None:
        if self._bounds is None:
            raise ValueError(f"{what} needs a backend built with page_bounds=True")

    def bounds_bytes(self) -> int:
        """Device bytes of the page bounds (beside ``pool_bytes``)."""
        return 0 if self._bounds is None else self._bounds.numel() * self._bounds.element_size()

    # -- pool construction / accounting ---------------------------------------

    def zeros_like_pool(self) -> torch.Tensor:
        return torch.zeros_like(self._k_pool[0])

    def workspace_bytes(self) -> int:
        """Split-K partials and arrival counters; grows with the largest batch
        planned, not with the pool."""
        return self._workspace.numel()

    @staticmethod
    def estimate_pool_bytes(num_layers: int, num_blocks: int, block_size: int,
                            n_kv_heads: int, head_dim: int,
                            dtype: torch.dtype = torch.float16) -> int:
        elem = torch.empty((), dtype=dtype).element_size()
        return num_layers * 2 * num_blocks * block_size * n_kv_heads * head_dim * elem

    # -- helpers -----------------------------------------------------------------

    def _set_workspace(self, ws: torch.Tensor) -> None:
        self._workspace = ws
        self._ws_ptr = ws.data_ptr() if ws.numel() else None
        self._ws_bytes = ws.numel()
        if self._planned is not None:   # described again, with this workspace
            self._planned.batch = self._planned.batch_ptr = None
        # leading bytes known to be zero between launches (a new workspace
        # is zero-filled)
        self._ws_zero = ws.numel()

    # -- write path -----------------------------------------------------------------

    def refresh_page_bounds(self, blocks=None) -> None:
        """
        Renew every layer's key bounds of ``blocks`` (all of the pool by
        default) from the pool: for a caller that wrote ``k_pool`` itself.
        Appends, block copies and swaps keep the bounds by themselves.
        """
        self._need_bounds("refresh_page_bounds")
        self._flush()
        if blocks is None:
            return self._renew_bounds(None, self.num_blocks, _current_stream(self.device))
        ids = block_ids(blocks)
        if ids.shape[0] == 0:
            return
        if ids.min() < 0 or ids.max() >= self.num_blocks:
            raise IndexError(f"block id outside [0, {self.num_blocks})")
        ids = torch.from_numpy(ids.astype(np.int32)).pin_memory().to(self.device,
                                                                     non_blocking=True)
        self._renew_bounds(ids, ids.shape[0], _current_stream(self.device))

    def _renew_bounds(self, ids, n: int, stream: int, layer: int | None = None) -> None:
        """Bounds of the blocks ``ids`` (device int32; None: the pool's first
        ``n``) in one layer or in all of them."""
        l = layer or 0
        lo, hi = self._bounds_ptr[l]
        with self._on_device():
            rc = self._lib.pkv_page_bounds(
                self._k_ptr[l], 2 * self._plane_bytes, lo, hi, 2 * (hi - lo),
                self.num_layers if layer is None else 1, self.num_blocks,
                None if ids is None else ids.data_ptr(), n, self.n_kv_heads, self.head_dim,
                self.block_size, self._code, self._status_ptr, stream)
        _native.check(rc, "page bounds")

    def append_kv(self, layer_idx: int, k: torch.Tensor, v: torch.Tensor,
                  meta: BatchMeta) -> None:
        """Scatter this step's K/V into the pool through ``meta.slot_mapping``."""
        # (checks and conversions inlined: this runs once per layer per step)
        if layer_idx is None or not 0 <= layer_idx < self.num_layers:
            self._check_layer(layer_idx)
        if meta.slot_mapping is None:
            raise ValueError("MI355XBackend.append_kv requires meta.slot_mapping")
        ks = k.shape
        tokens = ks[0]
        if ks != (tokens, self.n_kv_heads, self.head_dim):
            raise ValueError(f"k has shape {tuple(ks)}, expected "
                             f"({tokens}, {self.n_kv_heads}, {self.head_dim})")
        if v.shape != ks:
            raise ValueError(f"v shape {tuple(v.shape)} != k shape {tuple(ks)}")
        if meta.slot_mapping.shape[0] != tokens:
            raise ValueError(f"slot_mapping has {meta.slot_mapping.shape[0]} entries but "
                             f"{tokens} tokens were supplied")
        if self._pending is not None:
            self._flush()
        dt, di = self.dtype, self.device.index
        if not (k.dtype is dt and k.get_device() == di and k.is_contiguous()):
            k = self._as_pool(k)
        if not (v.dtype is dt and v.get_device() == di and v.is_contiguous()):
            v = self._as_pool(v)
        stream = _raw_stream(di) if _raw_stream is not None else _current_stream(self.device)
        if self._fuse_append:
            p = self._planned
            if p is None or p.meta is not meta:
                if _capturing():   # no plan is made here: the rows are appended on their own
                    slots = self._slots_for(meta)
                    self._keep(slots)
                    return self._launch_append(layer_idx, k, v, slots, stream)
                try:
                    p = self._ensure_planned(meta)
                except ValueError:
                    p = None  # inconsistent paging metadata: append now, attend will raise
            if p is not None and p.fusable:
                pend = _Pending()
                pend.layer, pend.k, pend.v, pend.meta = layer_idx, k, v, meta
                pend.slots, pend.stream = p.slots, stream
                pend.kver, pend.vver = k._version, v._version
                self._pending = pend
                return
            if p is not None and p.n_tokens == tokens and tokens:
                rc = self._lib.pkv_append_batch(
                    p.batch_ptr or self._describe(p), self._k_ptr[layer_idx],
                    self._v_ptr[layer_idx], k.data_ptr(), v.data_ptr(), stream)
                if rc:
                    _native.check(rc, "append_kv")
                return
        if self._bounds is None:
            return self._launch_append(layer_idx, k, v, self._slots_for(meta), stream)
        r = self._rows
        if r is None or r.meta is not meta:
            r = self._rows_for(meta)
        stream = self._enter(r)   # (before the rows: behind the upload of their slots)
        self._launch_append(layer_idx, k, v, r.slots, stream)
        if r.complete is not None:
            self._renew_bounds(r.complete, r.complete.shape[0], stream, layer_idx)

    def append_kv_rotated(self, layer_idx: int, q: torch.Tensor, k: torch.Tensor,
                          v: torch.Tensor, meta: BatchMeta, table: RotaryTable) -> torch.Tensor:
        """
        Rotate this step's queries and keys by ``meta.positions`` and scatter
        the rotated K and V into the pool through ``meta.slot_mapping``, in one
        launch; returns the rotated queries (a new ``(tokens, n_heads,
        head_dim)`` tensor), ready for an ``attend``.

        ``q``, ``k`` and ``v`` may be slices of one projection's output: any
        stride between tokens, heads one after another. Rotation in 32 bits,
        rounded once to the pool dtype; inputs of another dtype are brought to
        it first, as ``append_kv`` does. A position past the table is refused
        where the meta's host mirror holds it, and else flagged for
        ``check_device_errors`` (its row is not written, its query is zero).
        To capture a graph, call it with the meta before, with no other meta's
        call between.
        """
        if layer_idx is None or not 0 <= layer_idx < self.num_layers:
            self._check_layer(layer_idx)
        if meta.slot_mapping is None:
            raise ValueError("MI355XBackend.append_kv_rotated requires meta.slot_mapping")
        tokens, d, hkv = q.shape[0], self.head_dim, self.n_kv_heads
        if q.shape != (tokens, self.n_heads, d):
            raise ValueError(f"q has shape {tuple(q.shape)}, expected "
                             f"({tokens}, {self.n_heads}, {d})")
        if k.shape != (tokens, hkv, d):
            raise ValueError(f"k has shape {tuple(k.shape)}, expected ({tokens}, {hkv}, {d})")
        if v.shape != k.shape:
            raise ValueError(f"v has shape {tuple(v.shape)}, expected ({tokens}, {hkv}, {d})")
        if meta.slot_mapping.shape[0] != tokens or meta.n_tokens != tokens:
            raise ValueError(f"meta describes {meta.n_tokens} tokens and "
                             f"{meta.slot_mapping.shape[0]} slots but {tokens} tokens were "
                             "supplied")
        r = self._rows
        if r is None or r.meta is not meta or r.table is not table:
            r = self._rows_for(meta, table)
        pend = self._pending
        if pend is not None:
            self._flush()
        q, k, v = self._token_rows(q), self._token_rows(k), self._token_rows(v)
        stream = self._enter(r, pend.slots if pend is not None else None)
        out = torch.empty((tokens, self.n_heads, d), dtype=self.dtype, device=self.device)
        lo, hi = self._bounds_ptr[layer_idx] if r.complete is not None else (None, None)
        with self._on_device():
            rc = self._lib.pkv_append_rotated_batch(
                r.ptr, self._k_ptr[layer_idx], self._v_ptr[layer_idx], q.data_ptr(), q.stride(0),
                out.data_ptr(), k.data_ptr(), k.stride(0), v.data_ptr(), v.stride(0), lo, hi,
                stream)
        if rc:
            _native.check(rc, "append_kv_rotated")
        return out

    def _check_table(self, meta: BatchMeta, table) -> None:
        if not isinstance(table, RotaryTable):
            raise TypeError(f"table must be a RotaryTable, got {type(table).__name__}")
        if table.device != self.device:
            raise ValueError(f"the rotation table is on {table.device}, the pool on "
                             f"{self.device}")
        if table.rotary_dim > self.head_dim:
            raise ValueError(f"rotary_dim={table.rotary_dim} exceeds head_dim={self.head_dim}")
        pos = meta.host_positions()   # (without them the kernel flags it)
        if pos is not None and pos.shape[0]:
            far = int(pos.view(np.uint64).max())   # (a negative one is the farthest)
            if far >= table.max_positions:
                raise ValueError(f"position {far - (far >> 63 << 64)} is outside the rotation "
                                 f"table of {table.max_positions} positions")

    def _rows_for(self, meta: BatchMeta, table: RotaryTable | None = None) -> _Rows:
        """The meta's slots, positions and completed pages on the device, once
        per meta, described for appends that rotate by ``table``."""
        if table is not None:
            self._check_table(meta, table)
        r = self._rows
        if r is None or r.meta is not meta:
            self._refuse_capture("append_kv_rotated (or append_kv, with page bounds)")
            r = _Rows()
            r.slots = self._slots_for(meta)
            r.positions = meta.positions.to(device=self.device, dtype=torch.int64).contiguous()
            r.complete = None
            if self._bounds is not None:
                pages = self._completed_pages(meta)
                if pages.shape[0]:
                    r.complete = self._upload(pages)
            r.buffers = [t for t in (r.slots, r.positions, r.complete) if t is not None]
            r.stream = _current_stream(self.device)
            r.meta = meta
        else:   # another table: what a captured launch read stays described as it was
            old, r = r, _Rows()
            for name in ("meta", "slots", "positions", "complete", "stream"):
                setattr(r, name, getattr(old, name))
            r.buffers = [t for t in (r.slots, r.positions, r.complete) if t is not None]
        r.table = table
        r.args = r.ptr = None
        if table is not None:
            r.buffers.append(table.table)
            if table.stream != _current_stream(self.device) and not _capturing():
                table.table.record_stream(torch.cuda.current_stream(self.device))
            r.args = _native.Rotated(
                num_blocks=self.num_blocks, n_tokens=r.positions.shape[0],
                max_positions=table.max_positions,
                n_complete=0 if r.complete is None else r.complete.shape[0],
                slot_mapping=r.slots.data_ptr(), positions=r.positions.data_ptr(),
                table=table.table.data_ptr(),
                complete=None if r.complete is None else r.complete.data_ptr(),
                status_word=self._status_ptr, n_heads=self.n_heads, n_kv_heads=self.n_kv_heads,
                head_dim=self.head_dim, page_size=self.block_size, dtype=self._code,
                rotary_dim=table.rotary_dim, interleaved=table.interleaved)
            r.ptr = C.addressof(r.args)
        self._rows = r
        return r

    def _completed_pages(self, meta: BatchMeta) -> np.ndarray:
        """Pages whose last row this meta's append writes: the bounds of a page
        are those of all its rows, and only whole pages are ever chosen by them.
        Rows that go elsewhere than the page table says renew their pages each
        time."""
        ql, cu, kvl, indptr, last, indices, slots = self._host_index(meta, True)
        ps = self.block_size
        seq = np.repeat(np.arange(ql.shape[0]), ql)
        pos = np.arange(seq.shape[0]) + (kvl - ql - cu[:-1])[seq]
        at = indptr[:-1][seq] + pos // ps
        if at.shape[0] == slots.shape[0] and (at < indices.shape[0]).all() and (pos >= 0).all():
            pages = indices[at]
            if (pages * ps + pos % ps == slots).all():
                return np.ascontiguousarray(pages[pos % ps == ps - 1], dtype=np.int32)
        pages = np.unique(slots // ps)
        return pages[(pages >= 0) & (pages < self.num_blocks)].astype(np.int32)

    def _slots_for(self, meta: BatchMeta) -> torch.Tensor:
        p = self._planned
        if p is not None and p.meta is meta:
            return p.slots
        sc = self._slot_cache
        if sc is not None and sc[0] is meta:
            return sc[1]
        slots = self._dev_i32(meta.slot_mapping)
        if not _capturing():   # (what a graph converts is there only once it has run)
            self._slot_cache = (meta, slots)
        return slots

    def _launch_append(self, layer, k, v, slots, stream) -> None:
        rc = self._lib.pkv_append_kv(
            self._k_ptr[layer], self._v_ptr[layer],
            self.num_blocks * self.block_size, k.data_ptr(), v.data_ptr(), slots.data_ptr(),
            k.shape[0], self.n_kv_heads, self.head_dim, self._code, self._status_ptr,
            stream)
        _native.check(rc, "append_kv")

    def _check_pending_intact(self, pend: _Pending) -> None:
        if pend.k._version != pend.kver or pend.v._version != pend.vver:
            self._pending = None
            raise RuntimeError(
                "k/v passed to append_kv were modified in place before the rows were "
                "written; pass tensors that stay unchanged until the next backend call"
            )

    def _flush(self) -> None:
        """Launch a deferred append on its own (on the stream it was issued on)."""
        pend = self._pending
        if pend is None:
            return
        self._check_pending_intact(pend)
        self._pending = None
        self._launch_append(pend.layer, pend.k, pend.v, pend.slots, pend.stream)
        cur = _current_stream(self.device)
        if cur != pend.stream:  # later work on this stream must see the rows
            ev = torch.cuda.Event()
            ev.record(torch.cuda.ExternalStream(pend.stream, device=self.device))
            torch.cuda.current_stream(self.device).wait_event(ev)

    # -- read path ------------------------------------------------------------------

    def attend(self, q: torch.Tensor, layer_idx: int, scale: float,
               meta: BatchMeta) -> torch.Tensor:
        """Causal GQA attention over each sequence's full paged history."""
        if layer_idx is None or not 0 <= layer_idx < self.num_layers:
            self._check_layer(layer_idx)
        qs = q.shape
        tokens = qs[0]
        if qs != (tokens, self.n_heads, self.head_dim):
            raise ValueError(f"q has shape {tuple(qs)}, expected "
                             f"({tokens}, {self.n_heads}, {self.head_dim})")
        if meta.n_tokens != tokens:
            raise ValueError(f"meta describes {meta.n_tokens} tokens but q has {tokens}")
        p = self._planned
        if p is None or p.meta is not meta:
            p = self._ensure_planned(meta)
        return self._attend_by(p, q, layer_idx, scale, meta)

    def _attend_by(self, p: _Plan, q: torch.Tensor, layer_idx: int, scale: float,
                   meta: BatchMeta) -> torch.Tensor:
        """``attend`` by the meta's plan ``p``."""
        di = self.device.index
        stream = _raw_stream(di) if _raw_stream is not None else _current_stream(self.device)
        pend = self._pending
        fused = (pend is not None and pend.layer == layer_idx and pend.meta is meta
                 and pend.stream == stream and p.fusable)
        if fused:
            self._check_pending_intact(pend)
            self._pending = None
        elif pend is not None:
            self._flush()
        if not (q.dtype is self.dtype and q.get_device() == di and q.is_contiguous()):
            q = self._as_pool(q)
        q_ptr = q.data_ptr()
        if q_ptr % 16 and p.dec is not None and not C.c_float(float(scale)).value > 0:
            # such a scale sends the chunks to the generic kernel, which takes
            # any address; the decode kernel reads 16 bytes at a time
            q = q.clone()
            q_ptr = q.data_ptr()
        out = torch.empty_like(q)
        kp = self._k_ptr[layer_idx]
        vp = self._v_ptr[layer_idx]
        self.n_runs += 1
        rc = self._lib.pkv_attend_batch(
            p.batch_ptr or self._describe(p), q_ptr, out.data_ptr(), kp, vp, float(scale),
            pend.k.data_ptr() if fused else None, pend.v.data_ptr() if fused else None, stream)
        if rc:
            _native.check(rc, "attend (prefill)" if p.use_prefill else "attend (decode)")
        return out

    def attend_shared(self, q: torch.Tensor, layer_idx: int, scale: float,
                      meta: BatchMeta) -> torch.Tensor:
        """
        ``attend`` for a decode batch whose sequences begin with the same
        pages (a system prompt, a document, the branches of a search): the
        shared pages, found by their ids in the page lists, are read once for
        all the sequences that begin with them, and so are the pages that some
        of those share further on. The result is ``attend``'s up to rounding,
        and depends, in its last bits, on what shares the batch.

        Batches with prompt chunks, geometries without the fast decode path, a
        scale that is not positive and batches that share too little to gain
        by it run as ``attend`` runs them. To capture a graph, call it with the
        meta (and a scale of the same sign) before, with no other meta's call
        between. Graphs captured with one meta share its buffers: neither their
        replays nor eager calls with it may overlap.
        """
        if layer_idx is None or not 0 <= layer_idx < self.num_layers:
            self._check_layer(layer_idx)
        tokens = q.shape[0]
        if q.shape != (tokens, self.n_heads, self.head_dim):
            raise ValueError(f"q has shape {tuple(q.shape)}, expected "
                             f"({tokens}, {self.n_heads}, {self.head_dim})")
        if meta.n_tokens != tokens:
            raise ValueError(f"meta describes {meta.n_tokens} tokens but q has {tokens}")
        p = self._shared
        if p is None or p.meta is not meta:
            p = self._plan_shared(meta)
        if not p.n_tiles or not C.c_float(float(scale)).value > 0:   # (as the kernels take it)
            with self._on_device():
                if _capturing():
                    return self._attend_in_graph(p, q, layer_idx, scale, meta)
                out = self.attend(q, layer_idx, scale, meta)
            if p.whole is None:
                p.whole = self._planned
            return out
        pend = self._pending
        fused = (pend is not None and pend.layer == layer_idx and pend.meta is meta
                 and pend.stream == _current_stream(self.device) and p.fusable
                 and not (pend.k.data_ptr() | pend.v.data_ptr()) % 16)
        if fused:
            self._check_pending_intact(pend)
            self._pending = None
        elif pend is not None:
            self._flush()
        stream = self._enter(p, pend.slots if pend is not None else None)
        if not (q.dtype is self.dtype and q.get_device() == self.device.index
                and q.is_contiguous()):
            q = self._as_pool(q)
        q_ptr = q.data_ptr()
        if q_ptr % 16:
            q = q.clone()
            q_ptr = q.data_ptr()
        out = torch.empty_like(q)
        with self._on_device():
            rc = self._lib.pkv_attend_shared_batch(
                p.ptr, q_ptr, out.data_ptr(), self._k_ptr[layer_idx], self._v_ptr[layer_idx],
                float(scale), pend.k.data_ptr() if fused else None,
                pend.v.data_ptr() if fused else None, stream)
        if rc:
            _native.check(rc, "attend_shared")
        self.n_runs += 1
        return out

    def _plan_shared(self, meta: BatchMeta) -> _Shared:
        self._refuse_capture("attend_shared")
        n = meta.n_seqs
        with_slots = (meta.slot_mapping is not None and meta.slot_mapping.shape[0] == n
                      and meta.kv_indices.shape[0] > 0)
        ql, cu, kvl, indptr, last, indices, slots = self._host_index(meta, with_slots)
        p = _Shared()
        p.n, p.n_tiles, p.buffers, p.whole = n, 0, [], None
        if self._split_mixed and n > 1 and not (ql != 1).any() and n == meta.n_tokens:
            self._check_pages(kvl, indptr, last, int(indices.shape[0]))
            self._fill_shared(p, meta, *(np.ascontiguousarray(a, dtype=np.int32)
                                         for a in (indptr, indices, kvl, last)))
            # (as for attend: each new row at the end of its own page list)
            p.fusable = with_slots and bool(
                (slots == indices[indptr[1:] - 1] * self.block_size + last - 1).all())
        p.stream = _current_stream(self.device)
        p.meta = meta
        self._shared = p
        return p

    def _attend_in_graph(self, p: _Shared, q, layer_idx, scale, meta) -> torch.Tensor:
        """``attend`` within a capture, by the plan of its eager call, which stays
        with ``p``, and a workspace of the graph's own, cleared by it. (In the
        backend's, which each plan lays out anew, other plans' partials would lie on
        this one's arrival counters between replays.)"""
        if p.whole is None:
            self._refuse_capture("attend_shared")
        self._keep(p)
        if self._pending is not None:
            self._keep(self._pending.slots)
        w = copy.copy(p.whole)
        n, d = (w.n_seqs, w) if w.dec is None else (w.dec.n, w.dec)
        ws = self._counted_workspace(self._lib.pkv_decode_workspace_bytes(
            n, d.n_slots, self.n_heads, self.n_kv_heads, self.head_dim), n)
        self._describe(w, ws)
        return self._attend_by(w, q, layer_idx, scale, meta)

    def _fill_shared(self, p: _Shared, meta: BatchMeta, indptr, indices, kvl, last) -> None:
        """Plan the batch's shared runs and own pages (pkv_plan_shared)."""
        ptr = lambda a: a.ctypes.data  # noqa: E731
        n_work, n_slots, stride, n_tiles, n_merges = (C.c_int32() for _ in range(5))
        needed, tiles_needed = C.c_int64(), C.c_int64()
        cap = 10 * self._decode_wgs + 2 * int(indptr[-1]) + 24 * p.n + 128
        tiles_cap = 8 * SHARED_TILES + 16 * p.n
        part = self.part_pages
        while True:
            for _ in range(3):
                buf, tiles = np.empty(cap, np.int32), np.empty(tiles_cap, np.int32)
                rc = self._lib.pkv_plan_shared(
                    ptr(indptr), ptr(indices), ptr(kvl), ptr(last), p.n, self.block_size,
                    self.num_blocks, self.n_heads, self.n_kv_heads, part, self._decode_wgs,
                    SHARED_MIN_PAGES, self._block_bytes * 2 // self.n_kv_heads, SHARED_PART_BYTES,
                    SHARED_LEAST_BYTES, SHARED_TILES, ptr(buf), cap, C.byref(needed),
                    C.byref(n_work), C.byref(n_slots), C.byref(stride), ptr(tiles), tiles_cap,
                    C.byref(tiles_needed), C.byref(n_tiles), C.byref(n_merges))
                if rc != _native.ERR_CAPACITY or (needed.value <= cap
                                                  and tiles_needed.value <= tiles_cap):
                    break
                cap, tiles_cap = max(cap, needed.value), max(tiles_cap, tiles_needed.value)
            _native.check(rc, "plan (shared)")
            need = self._lib.pkv_decode_workspace_bytes(p.n, n_slots.value, self.n_heads,
                                                        self.n_kv_heads, self.head_dim)
            if need < 2**31 or part >= MAX_PART_PAGES:
                break
            part = min(2 * part, MAX_PART_PAGES)
        if not n_tiles.value or need >= 2**31:
            return
        p.n_tiles, p.n_work, p.n_slots = n_tiles.value, n_work.value, n_slots.value
        p.stride, p.n_merges = stride.value, n_merges.value
        p.plan = self._upload(buf[:needed.value])
        p.tiles = self._upload(tiles[:tiles_needed.value])
        p.indices = self._dev_i32(meta.kv_indices)
        p.slots = self._dev_i32(meta.slot_mapping) if meta.slot_mapping is not None else None
        p.ws = self._counted_workspace(need, p.n)
        p.buffers = [t for t in (p.plan, p.tiles, p.indices, p.slots, p.ws) if t is not None]
        p.args = _native.Shared(
            num_blocks=self.num_blocks, workspace_bytes=need, kv_indices=p.indices.data_ptr(),
            tiles=p.tiles.data_ptr(), plan=p.plan.data_ptr(),
            slot_mapping=None if p.slots is None else p.slots.data_ptr(),
            workspace=p.ws.data_ptr(), status_word=self._status_ptr, n_seqs=p.n,
            n_heads=self.n_heads, n_kv_heads=self.n_kv_heads, head_dim=self.head_dim,
            page_size=self.block_size, dtype=self._code, n_tiles=p.n_tiles, n_merges=p.n_merges,
            n_work=p.n_work, n_slots=p.n_slots, plan_stride=p.stride)
        p.ptr = C.addressof(p.args)
        self.n_plans += 1

    def attend_selected(self, q: torch.Tensor, layer_idx: int, scale: float, meta: BatchMeta,
                        pages: int, return_pages: bool = False):
        """
        Attention of a decode batch over at most ``pages`` pages a sequence
        and KV head: the sequence's last page and, of the others, those whose
        key bounds allow the largest score (the largest over the KV head's
        query heads of ``sum_d max(q_d lo_d, q_d hi_d)``, summed in 64 bits;
        equal scores: the earlier page; a NaN beats every number). Sequences of
        at most ``pages`` pages are attended whole, as ``attend`` does.

        Needs ``page_bounds=True``, one token per sequence and a positive
        scale. With ``return_pages`` also returns the chosen pages' indices in
        each sequence's page list, int32 ``(n_seqs, n_kv_heads, min(pages,
        longest list))``, ascending, -1 behind a shorter list. To capture a
        graph, call it with the meta and ``pages`` before, with no other meta's
        call between. Graphs captured with one meta share its buffers: neither
        their replays nor eager calls with it may overlap.
        """
        if layer_idx is None or not 0 <= layer_idx < self.num_layers:
            self._check_layer(layer_idx)
        self._need_bounds("attend_selected")
        tokens = q.shape[0]
        if q.shape != (tokens, self.n_heads, self.head_dim):
            raise ValueError(f"q has shape {tuple(q.shape)}, expected "
                             f"({tokens}, {self.n_heads}, {self.head_dim})")
        if meta.n_tokens != tokens:
            raise ValueError(f"meta describes {meta.n_tokens} tokens but q has {tokens}")
        pages = index(pages)
        if pages < 1:
            raise ValueError(f"pages must be positive, got {pages}")
        if not float(scale) > 0:
            raise ValueError(f"attend_selected needs a positive scale, got {scale}: the bounds "
                             "are of the largest score")
        p = self._selected
        if p is None or p.meta is not meta or p.asked != pages:
            p = self._selected_for(meta, pages)
        self._flush()
        stream = self._enter(p)
        if not (q.dtype is self.dtype and q.get_device() == self.device.index
                and q.is_contiguous()):
            q = self._as_pool(q)
        q_ptr = q.data_ptr()
        if q_ptr % 16:
            q = q.clone()
            q_ptr = q.data_ptr()
        out = torch.empty_like(q)
        ordinals = p.ordinals
        if return_pages:
            ordinals = torch.empty((p.n, self.n_kv_heads, p.width), dtype=torch.int32,
                                   device=self.device)
        lo, hi = self._bounds_ptr[layer_idx]
        with self._on_device():
            rc = self._lib.pkv_attend_selected_batch(
                p.ptr, q_ptr, out.data_ptr(), self._k_ptr[layer_idx], self._v_ptr[layer_idx],
                lo, hi, ordinals.data_ptr(), float(scale), stream)
        if rc:
            _native.check(rc, "attend_selected")
        self.n_runs += 1
        return (out, ordinals) if return_pages else out

    def _selected_for(self, meta: BatchMeta, pages: int) -> _Selected:
        """The meta's plan for this budget, made once (a step's layers may differ
        in theirs)."""
        known = tuple(p for p in self._budgets if p.meta is meta)
        p = next((p for p in known if p.asked == pages), None)
        if p is None:
            p = self._plan_selected(meta, pages)
            known += (p,)
        self._budgets, self._selected = known, p
        return p

    def _plan_selected(self, meta: BatchMeta, pages: int) -> _Selected:
        self._refuse_capture("attend_selected")
        ql, cu, kvl, indptr, last, indices, _ = self._host_index(meta, False)
        n = int(ql.shape[0])
        if n == 0:
            raise ValueError("attend_selected needs at least one sequence")
        if (ql != 1).any() or n != meta.n_tokens:
            raise ValueError("attend_selected takes decode batches: one token per sequence "
                             f"(query_lens up to {int(ql.max())} over {meta.n_tokens} tokens)")
        self._check_pages(kvl, indptr, last, int(indices.shape[0]))
        p = _Selected()
        p.asked, p.n, p.max_pages = pages, n, int(np.diff(indptr).max())
        pages = width = p.width = min(pages, p.max_pages)   # (the longest list: all of it)
        dev = {"device": self.device}
        p.indptr = self._dev_i32(meta.kv_indptr)
        p.indices = self._dev_i32(meta.kv_indices)
        p.kv_lens = self._dev_i32(meta.kv_lens)
        many = n * self.n_kv_heads
        p.scores = torch.empty(many * p.max_pages if p.max_pages > pages else 0,
                               dtype=torch.float64, **dev)
        p.ids = torch.empty(many * width, dtype=torch.int32, **dev)
        p.ordinals = torch.empty(many * width, dtype=torch.int32, **dev)
        p.plan = p.places = p.words = None
        n_work = n_slots = stride = 0
        pieces = many * -(-width // SELECTED_PART_PAGES)
        if self._fast_decode and pieces > SELECTED_PIECES:
            p.part = self.part_pages
            plan, places, n_work, n_slots, stride, need = self._plan_chosen(kvl, pages, p)
            p.plan, p.places = self._upload(plan), self._upload(places)
            p.words = torch.empty(self.n_kv_heads * plan.shape[0], dtype=torch.int32, **dev)
        else:
            p.part = min(self.part_pages, SELECTED_PART_PAGES)
            while True:   # partials take 32-bit offsets: longer pieces where they pass 2 GiB
                need = self._lib.pkv_selected_workspace_bytes(
                    n, p.max_pages, pages, p.part, self.n_heads, self.n_kv_heads, self.head_dim,
                    self.block_size, self.num_blocks, self._code)
                if need < 2**31 or p.part >= MAX_PART_PAGES:
                    break
                p.part = min(2 * p.part, MAX_PART_PAGES)
        p.ws = self._counted_workspace(need, n)
        p.buffers = [t for t in (p.indptr, p.indices, p.kv_lens, p.scores, p.ids, p.ordinals,
                                 p.words, p.places, p.plan, p.ws) if t is not None]
        at = lambda t: t.data_ptr() if t is not None and t.numel() else None  # noqa: E731
        p.args = _native.Selected(
            num_blocks=self.num_blocks, workspace_bytes=need,
            head_words=0 if p.plan is None else p.plan.shape[0], kv_indptr=at(p.indptr),
            kv_indices=at(p.indices), kv_lens=at(p.kv_lens), scores=at(p.scores), ids=at(p.ids),
            words=at(p.words), places=at(p.places), plan=at(p.plan), workspace=at(p.ws),
            status_word=self._status_ptr, n_seqs=n, max_pages=p.max_pages, pages=pages,
            part_pages=p.part, n_heads=self.n_heads, n_kv_heads=self.n_kv_heads,
            head_dim=self.head_dim, page_size=self.block_size, dtype=self._code, n_work=n_work,
            n_slots=n_slots, plan_stride=stride)
        p.ptr = C.addressof(p.args)
        p.stream = _current_stream(self.device)
        p.meta = meta
        self.n_plans += 1
        return p

    def _plan_chosen(self, kvl, pages: int, p: _Selected) -> tuple:
        """Plan the chosen lists for the streaming kernel (pkv_plan_selected):
        (plan, places, n_work, n_slots, stride, workspace bytes)."""
        lens = np.ascontiguousarray(kvl, dtype=np.int32)
        n_work, n_slots, stride = (C.c_int32() for _ in range(3))
        needed, places_needed = C.c_int64(), C.c_int64()
        listed = p.n * p.width
        cap = 10 * self._decode_wgs + 2 * listed + 24 * p.n + 128
        places_cap = 4 * p.n + listed
        ptr = lambda a: a.ctypes.data  # noqa: E731
        while True:
            for _ in range(3):
                plan, places = np.empty(cap, np.int32), np.empty(places_cap, np.int32)
                rc = self._lib.pkv_plan_selected(
                    ptr(lens), p.n, pages, self.n_heads, self.n_kv_heads, self.head_dim,
                    self._code, p.part, self._decode_wgs, ptr(plan), cap, C.byref(needed),
                    C.byref(n_work), C.byref(n_slots), C.byref(stride), ptr(places), places_cap,
                    C.byref(places_needed))
                if rc != _native.ERR_CAPACITY or (needed.value <= cap
                                                  and places_needed.value <= places_cap):
                    break
                cap, places_cap = max(cap, needed.value), max(places_cap, places_needed.value)
            _native.check(rc, "plan (selected)")
            need = self._lib.pkv_decode_workspace_bytes(p.n, n_slots.value, self.n_heads,
                                                        self.n_kv_heads, self.head_dim)
            if need < 2**31 or p.part >= MAX_PART_PAGES:
                break
            p.part = min(2 * p.part, MAX_PART_PAGES)
        return (plan[:needed.value], places[:places_needed.value], n_work.value, n_slots.value,
                stride.value, need)

    # -- planning ---------------------------------------------------------------

    def _ensure_planned(self, meta: BatchMeta) -> _Plan:
        """
        Build the launch plan for ``meta`` at most once per forward pass.
        Keyed on the object identity of the (frozen) BatchMeta, with a strong
        reference held so the identity cannot be recycled. The softmax scale
        is a launch argument, not part of the plan.
        """
        pl = self._planned
        if pl is not None and pl.meta is meta:
            return pl
        n = meta.n_seqs
        with_slots = (meta.slot_mapping is not None and meta.slot_mapping.shape[0] == n
                      and meta.kv_indices.shape[0] > 0 and meta.kv_indptr.shape[0] == n + 1)
        n_pages = int(meta.kv_indices.shape[0])
        ql, cu, kvl, indptr, last, indices, new_slot = self._host_index(meta, with_slots)
        if with_slots:  # for the fused append: each sequence's last page id
            last_page = indices[np.clip(indptr[1:] - 1, 0, n_pages - 1)]
        use_prefill = bool((ql > 1).any())
        if bool(meta.is_prefill) != use_prefill:
            raise ValueError(
                f"BatchMeta.is_prefill={meta.is_prefill} disagrees with query_lens "
                f"(max={int(ql.max())}). is_prefill must be True iff some sequence "
                "contributes more than one token."
            )
        p = _Plan()
        p.meta, p.use_prefill = meta, use_prefill
        # Fusing the append into attention is exact only if every sequence's
        # new row lands at the last slot of its own page list (then no other
        # sequence of the launch reads that slot).
        p.fusable = False
        if with_slots and not use_prefill:
            p.fusable = bool((new_slot == last_page * self.block_size + last - 1).all())
        p.n_seqs, p.n_tokens = n, int(cu[-1])
        if p.n_tokens != meta.n_tokens:
            raise ValueError(f"cu_query_lens ends at {p.n_tokens} but meta has "
                             f"{meta.n_tokens} positions")
        if int(indptr[0]) != 0 or int(indptr[-1]) != int(meta.kv_indices.shape[0]):
            raise ValueError(f"kv_indptr spans [{int(indptr[0])}, {int(indptr[-1])}) but "
                             f"kv_indices holds {int(meta.kv_indices.shape[0])} pages")
        if int(meta.batch_indices.shape[0]) != p.n_tokens:
            raise ValueError(f"batch_indices has {int(meta.batch_indices.shape[0])} entries "
                             f"for {p.n_tokens} tokens")
        i32 = lambda a: np.ascontiguousarray(a, dtype=np.int32)  # noqa: E731
        kvl32, indptr32, last32, cu32 = i32(kvl), i32(indptr), i32(last), i32(cu)
        ptr = lambda a: a.ctypes.data  # noqa: E731
        decodes = None
        p.stride = 0
        if not use_prefill:
            plan, p.n_work, p.n_slots, p.stride = self._plan_decode(indptr32, i32(indices),
                                                                    kvl32, last32, n)
        else:
            n_work = C.c_int32()
            cap = 4 * (int(cu[-1]) // self.q_tile + n + 1)
            buf = np.empty(cap, dtype=np.int32)
            rc = self._lib.pkv_plan_prefill(ptr(cu32), ptr(indptr32), ptr(kvl32), ptr(last32),
                                            n, self.block_size, self.q_tile, ptr(buf), cap,
                                            C.byref(n_work))
            _native.check(rc, "plan (prefill)")
            tiles = buf[:4 * n_work.value].reshape(-1, 4)
            if self._split_mixed and bool((ql == 1).any()):
                decodes = np.flatnonzero(ql == 1)
                tiles = tiles[ql[tiles[:, 0]] > 1]  # the decode kernel takes the rest
            plan, p.n_work, p.n_slots = tiles.reshape(-1).copy(), tiles.shape[0], 0
        p.plan = self._upload(plan)
        p.indptr = self._dev_i32(meta.kv_indptr)
        p.indices = self._dev_i32(meta.kv_indices)
        p.kv_lens = self._dev_i32(meta.kv_lens)
        p.dec = None
        if decodes is not None:
            p.dec = self._decode_rows(decodes, cu, indptr, kvl, last, indices)
        p.cu_q = self._dev_i32(meta.cu_query_lens)
        p.bidx = self._dev_i32(meta.batch_indices)
        p.slots = (self._dev_i32(meta.slot_mapping) if meta.slot_mapping is not None
                   else None)
        p.batch = p.batch_ptr = None
        self._planned = p
        self.n_plans += 1
        return p

    def _describe(self, p: _Plan, ws: torch.Tensor | None = None) -> int:
        """Address of the plan's ``pkv_batch``: the arguments its launches share,
        converted once instead of per layer; with ``ws`` in place of the backend's
        workspace."""
        own = ws is not None
        at = lambda t: t.data_ptr() if t is not None else None  # noqa: E731
        d = p.dec or p
        p.batch = _native.Batch(
            num_blocks=self.num_blocks, cu_query_lens=at(p.cu_q), kv_indptr=at(p.indptr),
            kv_indices=at(p.indices), kv_lens=at(p.kv_lens), batch_indices=at(p.bidx),
            slot_mapping=at(p.slots), prefill_plan=at(p.plan), decode_plan=at(d.plan),
            workspace=ws.data_ptr() if own else self._ws_ptr,
            workspace_bytes=ws.numel() if own else self._ws_bytes,
            status_word=self._status_ptr, n_seqs=p.n_seqs, n_tokens=p.n_tokens, n_heads=self.n_heads,
            n_kv_heads=self.n_kv_heads, head_dim=self.head_dim, page_size=self.block_size,
            dtype=self._code, is_prefill=p.use_prefill, n_tiles=p.n_work, q_tile=self.q_tile,
            n_decodes=p.dec.n if p.dec is not None else 0, n_work=d.n_work, n_slots=d.n_slots,
            plan_stride=d.stride)
        p.batch_ptr = C.addressof(p.batch)
        return p.batch_ptr

    def _plan_decode(self, indptr32, indices32, kvl32, last32, n):
        """Host decode plan (pkv_plan_decode) plus a workspace large enough for it.
        Returns (plan, n_work, n_slots, stride)."""
        if not self._fast_decode:  # the generic kernel reads the CSR, not a plan
            return np.zeros(4, dtype=np.int32), 1, 0, 4
        ptr = lambda a: a.ctypes.data  # noqa: E731
        n_work, n_slots, stride = C.c_int32(), C.c_int32(), C.c_int32()
        needed = C.c_int64()
        cap = 10 * self._decode_wgs + 2 * int(indptr32[-1]) + 24 * n + 128
        counter_bytes = (4 * n * self.n_kv_heads + 255) // 256 * 256
        part_pages = self.part_pages
        while True:
            for _ in range(2):
                buf = np.empty(cap, dtype=np.int32)
                rc = self._lib.pkv_plan_decode(
                    ptr(indptr32), ptr(indices32), ptr(kvl32), ptr(last32), n,
                    self.block_size, self.num_blocks, self.n_kv_heads, part_pages,
                    self._decode_wgs, ptr(buf), cap, C.byref(needed), C.byref(n_work),
                    C.byref(n_slots), C.byref(stride))
                if rc == _native.ERR_CAPACITY and needed.value > cap:
                    cap = int(needed.value)
                    continue
                break
            _native.check(rc, "plan (decode)")
            need = self._lib.pkv_decode_workspace_bytes(n, n_slots.value, self.n_heads,
                                                        self.n_kv_heads, self.head_dim)
            # The kernel addresses the partials with 32-bit buffer offsets
            # (at most 2 GiB). A batch whose partials would not fit is cut
            # into larger pieces for this launch only (its bits then differ
            # from a solo run's, which is cut at part_pages).
            if need - counter_bytes < 2**31 - 1 or part_pages >= MAX_PART_PAGES:
                break
            part_pages = min(2 * part_pages, MAX_PART_PAGES)
        if need > self._workspace.numel():
            # zero-filled (the arrival counters at the front start at zero),
            # with room to spare: a running batch's plans grow step by step
            # as its sequences do, and each regrowth is an allocation
            grown = max(need, self._workspace.numel() * 5 // 4)
            self._set_workspace(torch.zeros(grown, dtype=torch.uint8, device=self.device))
        elif counter_bytes > self._ws_zero:
            # the counters now reach over bytes an earlier layout used for
            # partials: clear what is new (every counter is zero after a launch)
            self._workspace[self._ws_zero:counter_bytes].zero_()
        # after this plan's launch the bytes past its counters hold partials
        self._ws_zero = counter_bytes
        return (buf[:int(needed.value)].copy(), n_work.value, n_slots.value, stride.value)

    def _decode_rows(self, dec, cu, indptr, kvl, last, indices) -> _DecodeRows:
        """The decode-kernel batch of a mixed batch's one-token sequences
        ``dec``: a plan over their own pages, each item's row set to the
        sequence's token row in the whole batch, so the kernel reads q and
        writes out in place."""
        npg = indptr[dec + 1] - indptr[dec]
        sub_ptr = np.concatenate([[0], np.cumsum(npg)])
        # position in the batch's kv_indices of every page of the sub-batch
        page_ix = np.repeat(indptr[dec] - sub_ptr[:-1], npg) + np.arange(int(sub_ptr[-1]))
        i32 = lambda a: np.ascontiguousarray(a, dtype=np.int32)  # noqa: E731
        rows = cu[dec]
        d = _DecodeRows()
        d.n = int(dec.shape[0])
        plan, d.n_work, d.n_slots, d.stride = self._plan_decode(
            i32(sub_ptr), i32(indices[page_ix]), i32(kvl[dec]), i32(last[dec]), d.n)
        # item i of a bin: 8 (i + 1) ints before the bin's end; its sequence
        # first, its flags (last-page bit, then the row) last
        blocks = plan[:plan.shape[0] // d.stride * d.stride].reshape(-1, d.stride)
        count = blocks[:, 0]
        bins = np.repeat(np.arange(blocks.shape[0]), count)
        first = np.repeat(np.cumsum(count) - count, count)
        at = (bins + 1) * d.stride - 8 * (np.arange(bins.shape[0]) - first + 1)
        plan[at + 7] = (plan[at + 7] & 1) | (rows[plan[at]] << 1)
        d.plan = self._upload(plan)
        return d

    def invalidate_plan(self) -> None:
        """Force the next ``attend`` to re-plan (and drop the cached meta)."""
        self._flush()
        self._planned = None
        self._slot_cache = None
        self._rows = self._selected = self._shared = None
        self._budgets = ()

    # -- misc -------------------------------------------------------------------------

    def reset(self) -> None:
        """Zero every pool and drop the plan. Tests only."""
        self._pending = None
        self._pool.zero_()
        if self._bounds is not None:
            self._bounds.zero_()
        self.invalidate_plan()

    def __repr__(self) -> str:
        mib = self.pool_bytes() / (1024 * 1024)
        return (f"MI355XBackend(layers={self.num_layers}, blocks={self.num_blocks}, "
                f"block_size={self.block_size}, kv_heads={self.n_kv_heads}, "
                f"heads={self.n_heads}, head_dim={self.head_dim}, dtype={self.dtype}, "
                f"device={self.device}, pool={mib:.1f} MiB)")
