"""
The shared-prefix plan on the host: every page of every sequence is read
exactly once, in a shared tile or in a piece of its own; partial slots and
arrival counts fit; refusals.
"""

from __future__ import annotations

import ctypes as C
import random

import numpy as np
import pytest

from llm_serving_layer_amd import _native


def plan_shared(tables, tails, *, n_kv=8, G=4, part=17, wgs=512, min_pages=4, target=512, ps=16,
                blocks=1 << 20, page_bytes=4096, part_bytes=0, least=0):
    """Plan and parse: (ids, n_slots, tiles, merges, members, items)."""
    lib = _native.load()
    indptr = np.concatenate([[0], np.cumsum([len(t) for t in tables])]).astype(np.int32)
    ids = np.array([b for t in tables for b in t], np.int32)
    kvl = np.array([(len(t) - 1) * ps + x for t, x in zip(tables, tails)], np.int32)
    last = np.array(tails, np.int32)
    p = lambda a: a.ctypes.data_as(C.c_void_p)  # noqa: E731
    nw, ns, st, nt, nm = (C.c_int32() for _ in range(5))
    need, tneed = C.c_int64(), C.c_int64()
    cap = tcap = 1
    for _ in range(4):
        buf, tiles = np.zeros(cap, np.int32), np.zeros(tcap, np.int32)
        rc = lib.pkv_plan_shared(p(indptr), p(ids), p(kvl), p(last), len(tables), ps, blocks,
                                 n_kv * G, n_kv, part, wgs, min_pages, page_bytes, part_bytes,
                                 least, target, p(buf), cap, C.byref(need), C.byref(nw), C.byref(ns), C.byref(st), p(tiles),
                                 tcap, C.byref(tneed), C.byref(nt), C.byref(nm))
        if rc != _native.ERR_CAPACITY:
            break
        cap, tcap = max(cap, need.value), max(tcap, tneed.value)
    _native.check(rc, "plan")
    if not nt.value:     # nothing is shared: no plan either
        assert not any((nw.value, ns.value, st.value, nm.value, need.value, tneed.value))
        none = np.zeros((0, 8), np.int32)
        return ids, 0, none, none[:, :4], none[:, :2], []
    per_wg = 4 if n_kv % 4 == 0 else 2 if n_kv % 2 == 0 else 1
    bins, S, items = nw.value // (n_kv // per_wg), st.value, []
    for b in range(bins):
        blk, at = buf[b * S:(b + 1) * S], 4
        for i in range(int(blk[0])):
            f = [int(x) for x in blk[S - 8 * (i + 1):][:8]]
            items.append((f, [int(w) & ((1 << 27) - 1) for w in blk[at:at + f[1]]],
                          [(int(w) >> 27 & 15) + 1 for w in blk[at:at + f[1]]]))
            at += f[1]
    t = tiles[:8 * nt.value].reshape(-1, 8)
    at = 8 * nt.value + 4 * nm.value
    merges = tiles[8 * nt.value:at].reshape(-1, 4)
    return ids, ns.value, t, merges, tiles[at:tneed.value].reshape(-1, 2), items


def tree(rng, n, depth, ps_pages):
    """Page lists of a random tree."""
    count = iter(range(10 ** 6))

    def grow(members, head, d):
        if d == 0 or len(members) == 1 or rng.random() < 0.2:
            return {i: head + [next(count) for _ in range(rng.randint(1, 30))] for i in members}
        head = head + [next(count) for _ in range(rng.randint(0, ps_pages))]
        kids = rng.randint(1, 3)
        out = {}
        for k in range(kids):
            part = members[k::kids]
            if part:
                out.update(grow(part, head, d - 1))
        return out
    lists = grow(list(range(n)), [], depth)
    return [lists[i] for i in range(n)]


def check(tables, tails, **kw):
    ids, n_slots, tiles, merges, members, items = plan_shared(tables, tails, **kw)
    G, min_pages = kw.get("G", 4), kw.get("min_pages", 4)
    if not len(tiles):
        return tiles, members, min_pages
    read = {i: [] for i in range(len(tables))}
    slots = {i: [] for i in range(len(tables))}
    for first, pages, at, count, split, *rest in tiles.tolist():
        assert 1 <= count <= 128 // G and pages >= 1 and not any(rest)
        run = ids[first:first + pages].tolist()
        for seq, slot in members[at:at + count].tolist():
            read[seq] += run
            slots[seq].append(slot + split)
    shared = {i: len(s) for i, s in slots.items()}
    own = {i: [] for i in read}
    for (seq, np_, tok0, kv, slot, parts, slot0, flags), pages, live in items:
        own[seq].append((tok0, pages, live, kv))
        assert flags >> 1 == seq
        if slot < 0:
            assert not shared[seq] and parts == 1
        else:
            slots[seq].append(slot)
            assert parts >= 2
    for i, (t, tail) in enumerate(zip(tables, tails)):
        mine = [p for _, pages, _, _ in sorted(own[i]) for p in pages]
        assert sorted(read[i] + mine) == sorted(t), "every page once"
        assert mine[-1] == t[-1], "the last page is the sequence's own"
        assert [x for _, _, live, _ in sorted(own[i]) for x in live] == \
            [16] * (len(mine) - 1) + [tail]
        assert all(kv == (len(mine) - 1) * 16 + tail for _, _, _, kv in own[i])
        parts = [f[5] for f, _, _ in items if f[0] == i]
        if slots[i]:     # dense slots: the shared parts, then the pieces in order
            assert sorted(slots[i]) == list(range(min(slots[i]), min(slots[i]) + len(slots[i])))
            assert set(parts) == {len(slots[i])}
            assert {f[6] for f, _, _ in items if f[0] == i} == {min(slots[i])}
    assert merges.tolist() == [[i, len(slots[i]), min(slots[i]), 0] for i in shared if shared[i]]
    used = sorted(s for v in slots.values() for s in v)
    assert used == list(range(n_slots)), "no two parts share a slot"
    return tiles, members, min_pages


@pytest.mark.parametrize("seed", range(12))
def test_every_page_is_read_once(seed):
    rng = random.Random(seed)
    n = rng.choice([1, 2, 3, 17, 90])
    tables = tree(rng, n, 3, rng.choice([3, 20, 200]))
    check(tables, [rng.randint(1, 16) for _ in range(n)], G=rng.choice([1, 2, 4, 8, 16]),
          n_kv=rng.choice([1, 2, 3, 8]), part=rng.choice([1, 3, 17, 64]),
          wgs=rng.choice([1, 40, 512]), min_pages=rng.choice([1, 4, 9]),
          target=rng.choice([1, 64, 512]))


def test_runs_below_the_least_length_stay_the_sequences_own():
    head = list(range(100, 103))                      # three pages shared by all
    tables = [head + list(range(200, 220)) + [1], head + list(range(200, 220)) + [2],
              head + [3, 4], head + [5]]
    tiles, members, _ = check(tables, [1, 16, 7, 8], min_pages=4, target=1)
    # the two first sequences' further run of 20 pages is shared, the head is not
    assert tiles[:, 1].tolist() == [20] and members[:, 0].tolist() == [0, 1]
    tiles, _, _ = check(tables, [1, 16, 7, 8], min_pages=3, target=1)
    assert sorted(tiles[:, 1].tolist()) == [3, 20]


def test_equal_lists_and_lists_that_are_heads_of_others():
    """The last page of the shortest list bounds the run; equal lists share all
    but their last page, a batch without shared pages nothing."""
    a = list(range(50, 80))
    for tables in ([a, a, a], [a, a[:10], a[:11]], [a[:1], a[:1]], [a[:2], a[:2]]):
        check(tables, [5] * len(tables), min_pages=1)
    tiles, _, _ = check([a, a, a], [16] * 3, min_pages=1, target=1)
    assert tiles[:, 1].sum() == 29
    tiles, _, _ = check([[1, 2, 3, 4, 5, 6]], [4])
    assert len(tiles) == 0
    tiles, _, _ = check([list(range(i, i + 9)) for i in range(0, 90, 9)], [4] * 10)
    assert len(tiles) == 0


def test_what_saves_too_little_is_not_shared():
    """A run must save more than its members' parts cost, all runs together the
    least; else the batch stays whole (no tiles, no plan)."""
    head, more = list(range(100, 110)), list(range(200, 260))
    tables = [head + more + [1], head + more + [2], head + [3]]
    # two members save 60 pages of the further run, three 20 of the head
    def runs(**kw):
        return sorted(set(plan_shared(tables, [1, 1, 1], target=1, **kw)[2][:, 1].tolist()))
    assert runs() == [10, 60]
    assert runs(part_bytes=20 * 4096 // 3) == [10, 60]
    assert runs(part_bytes=20 * 4096 // 3 + 1) == [60]
    assert runs(part_bytes=30 * 4096) == [60] and runs(part_bytes=30 * 4096 + 1) == []
    assert runs(least=8 * 80 * 4096) == [10, 60] and runs(least=8 * 80 * 4096 + 1) == []
    assert plan_shared(tables, [1, 1, 1], least=1 << 40)[1] == 0
    check(tables, [1, 5, 16], part_bytes=20 * 4096 // 3 + 1)


def test_splits_are_even_and_bounded():
    a = list(range(1000))
    tables = [a + [2000 + i] for i in range(40)]
    for target in (1, 8, 64, 512, 4096):
        tiles, _, _ = check(tables, [3] * 40, target=target)
        sizes = sorted(set(tiles[:, 1].tolist()))
        assert sum(tiles[:, 1].tolist()) == 2 * 1000      # two row tiles of 32 and 8
        assert all(x % 2 == 0 and x >= 8 for x in sizes[1:]) and len(sizes) <= 2


def test_refusals():
    with pytest.raises(ValueError, match="kv_last_page_len"):
        lib = _native.load()
        one = (C.c_int32 * 2)(0, 2)
        ids, kv, last = (C.c_int32 * 2)(1, 2), (C.c_int32 * 1)(20), (C.c_int32 * 1)(5)
        _native.check(lib.pkv_plan_shared(one, ids, kv, last, 1, 16, 8, 8, 2, 17, 4, 4, 0, 0, 0,
                                          8, None, 0, None, None, None, None, None, 0, None, None,
                                          None), "plan")
    for kw, match in (({"G": 3}, "not supported"), ({"min_pages": 0}, "not supported"),
                      ({"target": 0}, "not supported"), ({"part": 0}, "part_pages")):
        with pytest.raises(ValueError, match=match):
            plan_shared([[*range(8), 20], [*range(8), 30]], [1, 1], **kw)


def test_launch_refusals():
    lib = _native.load()

    def call(n_heads=8, d=64, page=16, dtype=0, scale=0.1, q=16, tiles=16, n_slots=4, ws=0):
        return lib.pkv_attend_shared(q, 16, 16, 16, 8, 16, 2, n_heads, 2, d, page, scale, dtype,
                                     tiles, 1, 1, 16, 1, n_slots, 72, None, None, None, None, ws,
                                     None, None)
    for kw, match in (({"d": 80}, "fast decode path"), ({"dtype": 2}, "fast decode path"),
                      ({"page": 8}, "fast decode path"), ({"n_heads": 6}, "fast decode path"),
                      ({"scale": 0.0}, "positive scale"), ({"scale": float("nan")}, "positive"),
                      ({"q": 8}, "aligned"), ({"q": None}, "null"), ({"tiles": None}, "tiles"),
                      ({"n_slots": 0}, "slots"), ({}, "workspace")):
        with pytest.raises(ValueError, match=match):
            _native.check(call(**kw), "attend_shared")
