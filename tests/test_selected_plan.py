"""
The plan over chosen pages on the host: every list's words have places of their
own, where the decode plan's items expect them; refusals.
"""

from __future__ import annotations

import ctypes as C
import random

import numpy as np
import pytest

from llm_serving_layer_amd import _native

from ._util import expected_cut


def plan_selected(lens, pages, *, n_heads=32, n_kv=8, d=64, dtype=0, part=17, wgs=512, cap=None):
    lib = _native.load()
    kv = np.array(lens, np.int32)
    p = lambda a: a.ctypes.data_as(C.c_void_p)  # noqa: E731
    nw, ns, st = (C.c_int32() for _ in range(3))
    need, pneed = C.c_int64(), C.c_int64()
    cap = pcap = 1
    for _ in range(3):
        buf, places = np.zeros(cap, np.int32), np.zeros(pcap, np.int32)
        rc = lib.pkv_plan_selected(p(kv), len(lens), pages, n_heads, n_kv, d, dtype, part, wgs,
                                   p(buf), cap, C.byref(need), C.byref(nw), C.byref(ns),
                                   C.byref(st), p(places), pcap, C.byref(pneed))
        if rc != _native.ERR_CAPACITY:
            break
        cap, pcap = max(cap, need.value), max(pcap, pneed.value)
    _native.check(rc, "plan")
    return buf[:need.value], places[:pneed.value], nw.value, ns.value, st.value


@pytest.mark.parametrize("seed", range(8))
def test_every_word_has_its_place(seed):
    rng = random.Random(seed)
    n, pages, part = rng.choice([1, 5, 90]), rng.choice([1, 2, 18, 64, 500]), rng.choice([1, 3, 17])
    lens = [rng.randint(1, 9000) for _ in range(n)]
    n_kv = rng.choice([1, 2, 3, 8])
    buf, places, nw, ns, S = plan_selected(lens, pages, n_kv=n_kv, n_heads=4 * n_kv, part=part,
                                           wgs=rng.choice([1, 64, 512]))
    per_wg = 4 if n_kv % 4 == 0 else 2 if n_kv % 2 == 0 else 1
    words = {}
    for b in range(nw // (n_kv // per_wg)):
        blk, at = buf[b * S:(b + 1) * S], 4
        for i in range(int(blk[0])):
            seq, np_, tok0, kv, *_ = (int(x) for x in blk[S - 8 * (i + 1):][:8])
            chosen = min(pages, -(-lens[seq] // 16))
            assert kv == (chosen - 1) * 16 + (lens[seq] - 1) % 16 + 1
            for j in range(np_):
                words[b * S + at + j] = (seq, tok0 // 16 + j)
            at += np_
    assert sorted(words.values()) == [(i, j) for i, k in enumerate(lens)
                                      for j in range(min(pages, -(-k // 16)))]
    for i, k in enumerate(lens):
        first, count = places[2 * i:2 * i + 2]
        cut = expected_cut(min(pages, -(-k // 16)), part)
        assert count == len(cut)
        at = places[2 * n + first:2 * n + first + count]
        for piece, size in enumerate(cut):
            for j in range(size):
                assert words[int(at[piece]) + j] == (i, piece * part + j)


def test_refusals():
    for kw, match in (({"d": 80}, "fast decode path"), ({"dtype": 2}, "fast decode path"),
                      ({"n_heads": 24}, "fast decode path"), ({"n_heads": 30}, "multiple"),
                      ({"part": 0}, "part_pages")):
        with pytest.raises(ValueError, match=match):
            plan_selected([100, 200], 4, **kw)
    with pytest.raises(ValueError, match="kv_len"):
        plan_selected([100, 0], 4)
    with pytest.raises(ValueError, match="positive"):
        plan_selected([100], 0)
