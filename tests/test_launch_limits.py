"""Calls that would take 2^32 threads or more in one launch are refused before
anything is launched."""

from __future__ import annotations

import ctypes as C

import numpy as np
import pytest

from llm_serving_layer_amd import _native


@pytest.mark.parametrize("tokens,n_kv,d,ps", [(2**23, 4, 80, 16), (2**26, 4, 64, 16),
                                              (2**25, 1, 64, 8)])
def test_append(tokens, n_kv, d, ps):
    stride = n_kv * d
    rc = _native.load().pkv_append_4bit(256, 256, 4, 256, stride, 256, stride, 256, tokens, n_kv,
                                        d, ps, 0, None, None)
    with pytest.raises(ValueError, match="too many rows"):
        _native.check(rc, "append")


@pytest.mark.parametrize("kw,match", [
    ({"head_dim": 80, "n_tokens": 2**23}, "query rows"),
    ({"n_few": 2**23, "few_waves": 1}, "pieces"), ({"n_few": 2**23, "few_waves": 4}, "pieces"),
    ({"n_few": 0, "n_wide": 2**23}, "pieces"), ({"n_few": 0, "n_tall": 2**23}, "row tiles")])
def test_attend(kw, match):
    b = _native.FourBit(num_blocks=4, n_seqs=1, n_tokens=1, n_heads=32, n_kv_heads=8, head_dim=64,
                        page_size=16, n_few=1, few_rows=4, part_rows=4)
    for f in ("cu_query_lens", "kv_indptr", "kv_indices", "kv_lens", "batch_indices", "items"):
        setattr(b, f, 256)
    for k, v in kw.items():
        setattr(b, k, v)
    rc = _native.load().pkv_attend_4bit(C.addressof(b), 256, 256, 256, 256, 0.1, None)
    with pytest.raises(ValueError, match=match):
        _native.check(rc, "attend")


@pytest.mark.parametrize("rows,seqs,vocab", [(2**24, 1, 2), (2**24 - 1, 2**23, 2),
                                             (2**20, 2**20, 2**21)])
def test_verify(rows, seqs, vocab):
    lib = _native.load()
    size = lib.pkv_verify_workspace_bytes(rows, seqs, vocab, 0)
    rc = lib.pkv_verify_drafts(256, rows, vocab, vocab, 0, 256, 256, 256, seqs, 256, None, 0, 0,
                               None, 1.0, 256, 1, 256, 256, size, None)
    with pytest.raises(ValueError, match="too many"):
        _native.check(rc, "verify")


@pytest.mark.parametrize("kv", [2**31 - 1, 2**31 - 16, 2**31 - 100])
@pytest.mark.parametrize("d", [64, 80])
def test_a_plan_of_lengths_next_to_the_largest(kv, d):
    """Tiles are counted past a sequence's end, in 32 bits."""
    ps, i32 = 16, lambda *a: np.array(a, dtype=np.int32)
    cu, pages, lens = i32(0, 1), -(-kv // ps), i32(kv)
    indptr, ids, last = i32(0, pages), np.zeros(pages, np.int32), i32(kv - (pages - 1) * ps)
    needed, args = C.c_int64(), _native.FourBit()
    items = np.empty(28 * 1024, np.int32)
    rc = _native.load().pkv_plan_4bit(
        cu.ctypes.data, indptr.ctypes.data, ids.ctypes.data, lens.ctypes.data, last.ctypes.data, 1,
        1, 1, d, ps, 0, 4, items.ctypes.data, items.size, C.byref(needed), C.addressof(args))
    with pytest.raises(ValueError, match="kv_len"):
        _native.check(rc, "plan")
