"""
The scheduler step's sampling and timing points on the device.

The reference scheduler ends every step with ``logits = model.forward_varlen(
tokens, meta, backend)`` and ``torch.argmax(logits, dim=-1).tolist()``
(serving/scheduler/scheduler.py:743-757), and times GPU work with events on
the stream rather than the host clock, because ``forward_varlen`` returns a
device tensor (docs/ADR.md:954-989, ADR-023). Here:

* ``greedy(logits)`` is that argmax on the device through the library's
  ``pkv_argmax_rows`` kernel (one int64 per row comes back, not the logits);
* ``StepTimer`` brackets a step with HIP events on torch's current stream
  (where the backend launches) and reads the elapsed time only at a declared
  synchronisation point;
* ``verify_drafts(logits, tokens, meta, uniforms)`` checks a step's drafted
  tokens against the target's logits and draws the token behind them (the
  reference decodes greedily: no counterpart);
* ``greedy_step`` is the forward-and-sample part of ``Scheduler.step``:
  metadata, tokens, forward, greedy pick, and one device-to-host copy of the
  picked ids, the step's only synchronisation.
"""

from __future__ import annotations

from itertools import accumulate

import torch

from . import _native
from .assembly import ScheduledSeq, build_batch_meta, build_token_tensor
from .backend import _DTYPES, _HERE, _capturing, _current_device, _current_stream
from .contract import BatchMeta

__all__ = ["greedy", "verify_drafts", "StepTimer", "greedy_step"]


def rows_for_kernel(logits: torch.Tensor) -> torch.Tensor:
    """
    ``logits`` itself when the argmax kernel can read it in place -- unit
    element stride and rows that do not overlap (row stride >= vocab, or a
    single row) -- else a contiguous copy. A view whose rows overlap (an
    ``expand`` has row stride 0) would otherwise make the kernel read rows
    1..n-1 past the end of the allocation.
    """
    n, vocab = logits.shape
    unit = logits.stride(1) == 1 or vocab == 1
    apart = n <= 1 or logits.stride(0) >= vocab
    return logits if unit and apart else logits.contiguous()


def greedy(logits: torch.Tensor) -> torch.Tensor:
    """
    ``torch.argmax(logits, dim=-1)`` for a (n_rows, vocab) f16, bf16 or f32
    device tensor whose rows are contiguous: an int64 device tensor of
    n_rows greedy ids (torch's order: a NaN beats every number, of equal
    values the first wins). Asynchronous on torch's current stream.
    """
    if logits.dim() != 2:
        raise ValueError(f"logits must be (n_rows, vocab), got shape {tuple(logits.shape)}")
    if logits.device.type != "cuda":
        raise ValueError(f"logits must be on the GPU, got {logits.device}")
    if logits.dtype not in _DTYPES:
        raise ValueError(f"logits dtype {logits.dtype} is not float16, bfloat16 or float32")
    n, vocab = logits.shape
    if vocab == 0:
        raise ValueError("argmax of an empty row: vocab is 0")
    logits = rows_for_kernel(logits)
    out = torch.empty(n, dtype=torch.int64, device=logits.device)
    if n == 0:
        return out
    lib = _native.load()
    # (one row: its stride is never used, and may be anything, e.g. 0)
    row_stride = logits.stride(0) if n > 1 else vocab
    rc = lib.pkv_argmax_rows(logits.data_ptr(), n, vocab, row_stride,
                             _DTYPES[logits.dtype], out.data_ptr(),
                             _current_stream(logits.device))
    _native.check(rc, "greedy argmax")
    return out


def _step_lengths(meta: BatchMeta, rows: int) -> list[int]:
    """Every sequence's rows of a step, checked against what the kernels read of the
    meta on the device."""
    n = meta.n_seqs
    if meta.cu_query_lens.shape != (n + 1,) or meta.batch_indices.shape != (rows,):
        raise ValueError(f"cu_query_lens has shape {tuple(meta.cu_query_lens.shape)} and "
                         f"batch_indices {tuple(meta.batch_indices.shape)} for {n} sequences "
                         f"and {rows} tokens")
    arrays = meta.host_arrays()
    if arrays is not None:
        lens = arrays["query_lens"].tolist()     # (a list: numpy's reductions cost 1 us each)
    elif _capturing():
        raise RuntimeError("verify_drafts reads a meta without host arrays from the device: not "
                           "while a graph is captured")
    else:
        lens = meta.query_lens.tolist()
        if meta.cu_query_lens.tolist() != [0, *accumulate(lens)]:
            raise ValueError("cu_query_lens are not the sums of query_lens")
    if min(lens) < 1 or sum(lens) != rows:
        raise ValueError(f"query_lens ({min(lens)} at least, {sum(lens)} in all) do "
                         f"not make up {rows} rows")
    return lens


def verify_drafts(logits: torch.Tensor, tokens: torch.Tensor, meta: BatchMeta,
                  uniforms: torch.Tensor, *, draft_probs: torch.Tensor | None = None,
                  temperature=1.0) -> tuple[torch.Tensor, torch.Tensor]:
    """
    Verify a step's drafted tokens: each sequence of ``meta`` contributes its
    last accepted token and its drafts (none or more), ``tokens`` (``(T,)``
    int64, as ``build_token_tensor`` gives them) are the step's tokens and
    ``logits`` (``(T, vocab)`` f16, bf16 or f32) the target's for what follows
    each. Draft x behind row r stands if ``uniforms[r] * q(x) < p(x)``: p the
    softmax of the row over ``temperature`` (a number, or a float32 tensor of one
    a sequence; as a float32, at most the largest finite one), q the drafting
    distribution (``draft_probs``, ``(T - n_seqs, vocab)``, a row a draft in order;
    None: 1 at the draft). The first that does not stand ends a sequence's run and
    is replaced by a token drawn from ``max(p - q, 0)`` (p where that is nothing);
    behind a run that stands whole one is drawn from the last row's p. Drawn is the
    first token whose running sum of weights exceeds the sequence's last number
    times their sum, so the ``(T,)`` float32 ``uniforms`` in [0, 1) serve all
    decisions once each.

    Returns ``(ids, accepted)``, int64: per sequence the drafts that stand, one
    more token, -1 behind it (``(n_seqs, max(query_lens))``), and how many stand.

    Decisions are those of 64-bit arithmetic. At a temperature of 0 or below a
    draft stands if it is the row's ``greedy`` id, which is taken otherwise; a
    row without a distribution (a NaN, +inf, nothing but -inf) lets no draft
    stand and gives its ``greedy`` id; a draft outside [0, vocab) falls.
    Asynchronous on torch's current stream; every call has a workspace of its
    own, so calls may overlap and be captured; a captured call reads ``meta``'s
    ``cu_query_lens`` and ``batch_indices``, which have to stay as long as the graph
    does. A meta without host arrays is read back from the device (not in a capture).
    """
    if logits.dim() != 2:
        raise ValueError(f"logits must be (n_tokens, vocab), got shape {tuple(logits.shape)}")
    if logits.device.type != "cuda":
        raise ValueError(f"logits must be on the GPU, got {logits.device}")
    if logits.dtype not in _DTYPES:
        raise ValueError(f"logits dtype {logits.dtype} is not float16, bfloat16 or float32")
    dev, (rows, vocab), n = logits.device, logits.shape, meta.n_seqs
    if vocab == 0:
        raise ValueError("verify_drafts of empty rows: vocab is 0")
    if meta.n_tokens != rows:
        raise ValueError(f"meta describes {meta.n_tokens} tokens but logits has {rows} rows")
    if n == 0 or rows < n:
        raise ValueError(f"verify_drafts needs a row a sequence, got {rows} for {n}")
    for name, x, dtype in (("tokens", tokens, torch.int64), ("uniforms", uniforms, torch.float32)):
        if x.shape != (rows,) or x.dtype is not dtype or x.device != dev:
            raise ValueError(f"{name} must be ({rows},) {dtype} on {dev}, got "
                             f"{tuple(x.shape)} {x.dtype} on {x.device}")
    if draft_probs is not None:
        if draft_probs.shape != (rows - n, vocab):
            raise ValueError(f"draft_probs has shape {tuple(draft_probs.shape)}, expected "
                             f"({rows - n}, {vocab}): one row a draft")
        if draft_probs.dtype not in _DTYPES or draft_probs.device != dev:
            raise ValueError(f"draft_probs must be float16, bfloat16 or float32 on {dev}, got "
                             f"{draft_probs.dtype} on {draft_probs.device}")
        draft_probs = rows_for_kernel(draft_probs)
        if rows == n:
            draft_probs = None
    temps = None
    if isinstance(temperature, torch.Tensor):
        if (temperature.shape != (n,) or temperature.dtype is not torch.float32
                or temperature.device != dev):
            raise ValueError(f"temperature must be a number or ({n},) float32 on {dev}, got "
                             f"{tuple(temperature.shape)} {temperature.dtype} on "
                             f"{temperature.device}")
        temps, temperature = temperature.contiguous(), 1.0
    elif not 0.0 <= float(temperature) < float("inf"):
        raise ValueError(f"temperature must be finite and not negative, got {temperature}")
    lens = _step_lengths(meta, rows)
    width = max(lens)
    logits, tokens, uniforms = rows_for_kernel(logits), tokens.contiguous(), uniforms.contiguous()
    cu, owner = meta.cu_query_lens, meta.batch_indices
    if not (cu.dtype is owner.dtype is torch.int32 and cu.device == owner.device == dev
            and cu.is_contiguous() and owner.is_contiguous()):
        cu, owner = (t.to(device=dev, dtype=torch.int32).contiguous() for t in (cu, owner))
    ids = torch.empty((n, width), dtype=torch.int64, device=dev)
    accepted = torch.empty(n, dtype=torch.int64, device=dev)
    lib, code = _native.load(), _DTYPES[logits.dtype]
    ws = torch.empty(lib.pkv_verify_workspace_bytes(rows, n, vocab, code), dtype=torch.uint8,
                     device=dev)
    here = _HERE if _current_device() == dev.index else torch.cuda.device(dev)
    with here:
        rc = lib.pkv_verify_drafts(
            logits.data_ptr(), rows, vocab, logits.stride(0) if rows > 1 else vocab, code,
            tokens.data_ptr(), cu.data_ptr(), owner.data_ptr(), n, uniforms.data_ptr(),
            None if draft_probs is None else draft_probs.data_ptr(),
            vocab if draft_probs is None or rows - n < 2 else draft_probs.stride(0),
            0 if draft_probs is None else _DTYPES[draft_probs.dtype],
            None if temps is None else temps.data_ptr(), float(temperature), ids.data_ptr(),
            width, accepted.data_ptr(), ws.data_ptr(), ws.numel(), _current_stream(dev))
    if rc:
        _native.check(rc, "verify_drafts")
    return ids, accepted


class StepTimer:
    """
    GPU time of a step from two HIP events on torch's current stream of
    ``device``: ``start()`` and ``stop()`` only record; ``elapsed_ms()``
    waits for the stop event (the declared synchronisation point) and
    returns the milliseconds between them. ``history`` keeps every step read.
    """

    def __init__(self, device="cuda:0"):
        self.device = torch.device(device)
        self._start = torch.cuda.Event(enable_timing=True)
        self._stop = torch.cuda.Event(enable_timing=True)
        self._armed = False
        self.history: list[float] = []

    def start(self) -> None:
        self._start.record(torch.cuda.current_stream(self.device))
        self._armed = True

    def stop(self) -> None:
        if not self._armed:
            raise RuntimeError("StepTimer.stop() without start()")
        self._stop.record(torch.cuda.current_stream(self.device))
        self._armed = False

    def elapsed_ms(self) -> float:
        self._stop.synchronize()
        ms = self._start.elapsed_time(self._stop)
        self.history.append(ms)
        return ms


def greedy_step(model, scheduled: list[ScheduledSeq], backend, page_size: int,
                timer: StepTimer | None = None) -> list[int]:
    """
    The forward-and-sample part of the reference's ``Scheduler.step``
    (serving/scheduler/scheduler.py:743-757): block tables already grown by
    the caller, then metadata and token ids for ``scheduled`` (in that
    order), ``model.forward_varlen(tokens, meta, backend)`` -> (n_seqs,
    vocab) device logits, the greedy id of every sequence on the device, and
    ONE device-to-host copy of those ids, which is also where a ``timer``'s
    stop event is known to have passed.
    """
    meta = build_batch_meta(scheduled, device=backend.device, page_size=page_size)
    tokens = build_token_tensor(scheduled, device=backend.device)
    if timer is not None:
        timer.start()
    logits = model.forward_varlen(tokens, meta, backend)
    if tuple(logits.shape[:1]) != (len(scheduled),):
        raise ValueError(f"forward_varlen returned {tuple(logits.shape)} logits for "
                         f"{len(scheduled)} sequences")
    ids = greedy(logits)
    if timer is not None:
        timer.stop()
    return ids.tolist()
