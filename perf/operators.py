"""
Performance cases of the operators around the paged cache beyond the plain
append and attention: the append with the position rotation on the way, the
attention of a batch that shares prefixes, and the attention over the pages a
cheap bound selects. Three kinds of case:

* ``rotate``    one layer's append: q and k turned by their positions, k and v
  written to the pages of the cache; with ``bounds`` the cache also keeps each
  page's key bounds, renewed for the pages the step completes.
* ``shared``    one layer's attention of a decode batch whose sequences begin
  with the same pages: ``root`` tokens shared by all, ``branch`` more by each
  of ``groups`` groups, then every sequence's own.
* ``selected``  one layer's attention of a decode batch over at most ``pages``
  pages a sequence: its last page, and those whose bounds (elementwise minimum
  and maximum of the page's keys) allow the largest score.

With ``own`` false everything is elementary torch in 32 bits (64 for angles
and for the scores that decide between pages); with ``own`` true the calls of
``MI355XBackend``. Lengths are fixed by the case; page tables, cache contents
and activations come from the seed.
"""

from __future__ import annotations

import math
import random

import torch

own = False

DEV = "cuda:0"
PAGE = 16
THETA = 10000.0
DTYPES = {"float16": torch.float16, "bfloat16": torch.bfloat16, "float32": torch.float32}

# 32 query heads over 8 KV heads at head_dim 64, the benchmark's geometry
BASE = {"n_kv": 8, "n_heads": 32, "head_dim": 64}
D128 = {"n_kv": 8, "n_heads": 32, "head_dim": 128}


def _rotate(name, dtype, *, n=0, lo=0, hi=0, n_chunk=0, chunk_lo=0, chunk_hi=0, history=0,
            rotary_dim=None, interleaved=False, fused=True, bounds=False, lens_seed=20260731,
            **geom):
    geom = {**BASE, **geom}
    case = {"kind": "rotate", "dtype": dtype, **geom, "n": n, "lo": lo, "hi": hi,
            "n_chunk": n_chunk, "chunk_lo": chunk_lo, "chunk_hi": chunk_hi, "history": history,
            "rotary_dim": rotary_dim or geom["head_dim"], "interleaved": interleaved,
            "fused": fused, "bounds": bounds, "lens_seed": lens_seed}
    return {"name": name, **case} if name else case


def _shared(name, dtype, *, n, root, groups=1, branch=0, law="uniform", mean=0, lo=1, hi=1,
            lens_seed=20260731, **geom):
    case = {"kind": "shared", "dtype": dtype, **BASE, **geom, "n": n, "root": root,
            "groups": groups, "branch": branch, "law": law, "mean": mean, "lo": lo, "hi": hi,
            "lens_seed": lens_seed}
    return {"name": name, **case} if name else case


def _selected(name, dtype, *, n, lo, hi, pages, lens_seed=20260731, **geom):
    case = {"kind": "selected", "dtype": dtype, **BASE, **geom, "n": n, "lo": lo, "hi": hi,
            "pages": pages, "lens_seed": lens_seed}
    return {"name": name, **case} if name else case


def listed():
    return [
        # one user alone: the new token's q, k, v of one layer
        _rotate("rotate_single", "float16", n=1, lo=1371, hi=1371),
        # a batch-256 decode step of a model with head_dim 128, in bf16
        _rotate("rotate_decode", "bfloat16", n=256, lo=16, hi=400, **D128),
        # one prompt chunk behind a cached history, pages bounded for selection
        _rotate("rotate_prompt", "float16", n_chunk=1, chunk_lo=777, chunk_hi=777, history=720,
                bounds=True),
        # chunked prefill of eight requests at once, half the dims rotated, in pairs
        _rotate("rotate_chunks", "bfloat16", n_chunk=8, chunk_lo=512, chunk_hi=1000, history=135,
                rotary_dim=64, interleaved=True, **D128),
        # a handful of requests over one system prompt
        _shared("shared_few", "float16", n=6, root=1536, lo=3, hi=90),
        # the headline decode batch behind a cached system prompt
        _shared("shared_batch", "float16", n=256, root=2048, law="lognormal", mean=258),
        # six few-shot tasks over one common preamble
        _shared("shared_tree", "bfloat16", n=96, root=512, groups=6, branch=784, lo=20, hi=400,
                **D128),
        # many questions about one long document
        _shared("shared_document", "bfloat16", n=128, root=16384, lo=100, hi=700, **D128),
        # one user with a long history
        _selected("selected_single", "float16", n=1, lo=32749, hi=32749, pages=64),
        # conversations partly shorter than the budget, 8 query heads a KV head
        _selected("selected_short", "float16", n=128, lo=100, hi=1500, pages=32, n_kv=4),
        # a decode batch of medium histories
        _selected("selected_batch", "bfloat16", n=48, lo=2000, hi=8000, pages=64, **D128),
        # long documents
        _selected("selected_long", "bfloat16", n=16, lo=20000, hi=60000, pages=128, **D128),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


GEOMS = [(8, 32, 64), (8, 32, 64), (8, 32, 128), (2, 8, 128), (8, 8, 64), (4, 8, 64), (2, 32, 64),
         (4, 32, 128), (1, 8, 64), (3, 12, 64)]


def draw(rng):
    kind = rng.choices(["rotate", "shared", "selected"], [1, 1, 1])[0]
    n_kv, n_heads, d = rng.choice(GEOMS)
    geom = {"n_kv": n_kv, "n_heads": n_heads, "head_dim": d}
    seed = rng.randrange(1 << 30)
    if kind == "rotate":
        dtype = rng.choices(["float16", "bfloat16", "float32"], [4, 4, 2])[0]
        rot = rng.choice([d, d, d // 2, 2 * rng.randint(1, d // 2)])
        opts = {"rotary_dim": rot, "interleaved": rng.random() < 0.4,
                "fused": rng.random() < 0.6, "bounds": rng.random() < 0.3, "lens_seed": seed}
        if rng.random() < 0.5:
            hi = _log(rng, 2, 4000)
            n = min(_log(rng, 1, 1000), max(1, 100000 // hi))
            return _rotate(None, dtype, n=n, lo=max(1, hi // 8), hi=hi, **opts, **geom)
        hi, n = _log(rng, 2, 2500), rng.randint(1, 4)
        hi = hi // 2 if dtype == "float32" else hi
        return _rotate(None, dtype, n_chunk=n, chunk_lo=max(1, hi // 2), chunk_hi=max(1, hi // n),
                       history=rng.choice([0, rng.randint(1, 1500)]), **opts, **geom)
    dtype = rng.choice(["float16", "bfloat16"])
    if kind == "shared":
        n, root = _log(rng, 2, 200), _log(rng, 2, 600) * PAGE
        groups = rng.choice([1, 1, rng.randint(1, min(n, 8))])
        branch = rng.choice([0, _log(rng, 1, 60) * PAGE])
        hi = _log(rng, 2, 700)
        return _shared(None, dtype, n=n, root=root, groups=groups, branch=branch,
                       lo=max(1, hi // 8), hi=hi, lens_seed=seed, **geom)
    n, pages = _log(rng, 1, 160), _log(rng, 1, 128)
    hi = min(_log(rng, 60, 50000), 400000 // n)
    pages = min(pages, max(1, 32768 // PAGE // n))   # as many pages read as by the largest
    return _selected(None, dtype, n=n, lo=max(1, hi // 3), hi=hi, pages=pages, lens_seed=seed,
                     **geom)


# ------------------------------------------------------------------ inputs ---

def _pages(n):
    return -(-n // PAGE)


def _lengths(case):
    """(history, new tokens) of every sequence."""
    rng = random.Random(case["lens_seed"])
    if case["kind"] == "rotate":
        out = [(rng.randint(case["lo"], case["hi"]) - 1, 1) for _ in range(case["n"])]
        lo, hi = min(case["chunk_lo"], case["chunk_hi"]), max(case["chunk_lo"], case["chunk_hi"])
        return out + [(case["history"], rng.randint(lo, hi)) for _ in range(case["n_chunk"])]
    if case["kind"] == "shared":
        pre = case["root"] + case["branch"]
        mu = math.log(max(case["mean"], 1)) - 0.8 ** 2 / 2.0
        return [(pre + max(1, min(2048, int(round(rng.lognormvariate(mu, 0.8)))
                           if case["law"] == "lognormal"
                           else rng.randint(case["lo"], case["hi"]))) - 1, 1)
                for _ in range(case["n"])]
    return [(rng.randint(case["lo"], case["hi"]) - 1, 1) for _ in range(case["n"])]


def _tables(case, seed):
    """(blocks of the pool, page ids of every sequence)."""
    lens = _lengths(case)
    shared = case["kind"] == "shared"
    root = case["root"] // PAGE if shared else 0
    branch = case["branch"] // PAGE if shared else 0
    groups = case["groups"] if shared else 0
    own_pages = [_pages(h + n) - root - branch for h, n in lens]
    used = root + groups * branch + sum(own_pages)
    nb = used + max(8, used // 16)
    order = list(range(nb))
    random.Random(seed).shuffle(order)
    at = root + groups * branch
    tables = []
    for i, k in enumerate(own_pages):
        g = i % groups if shared else 0
        tables.append(order[:root] + order[root + g * branch:root + (g + 1) * branch]
                      + order[at:at + k])
        at += k
    return nb, tables


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _values(shape, dtype, g):
    return torch.randn(shape, generator=g, device=DEV).mul_(0.5).to(dtype)


def _inputs(case, seed):
    """The cache's K and V and the step's activations. The keys of a page lie
    around a centre of their own, as neighbouring tokens' do."""
    dt, d, hkv = DTYPES[case["dtype"]], case["head_dim"], case["n_kv"]
    nb, tables = _tables(case, seed)
    g = _gen(seed)
    k = _values((nb, PAGE, hkv, d), dt, g)
    if case["kind"] == "selected":
        k += _values((nb, 1, hkv, d), dt, g)
    v = _values((nb, PAGE, hkv, d), dt, g)
    tokens = sum(n for _, n in _lengths(case))
    heads = case["n_heads"] + (2 * hkv if case["kind"] == "rotate" else 0)
    return nb, tables, k, v, _values((tokens, heads * d), dt, g)


def _frequencies(case):
    r = case["rotary_dim"]
    return THETA ** (-torch.arange(0, r, 2, dtype=torch.float64, device=DEV) / r)


def _bounds(k):
    """Elementwise minimum and maximum of every page's keys."""
    return k.amin(dim=1), k.amax(dim=1)


def prepare(case, seed):
    nb, tables, k, v, x = _inputs(case, seed)
    lens = _lengths(case)
    hq, hkv, d = case["n_heads"], case["n_kv"], case["head_dim"]
    state = {"case": case, "scale": d ** -0.5}
    if case["kind"] == "rotate":
        # the slices of one projection's output, as a model has them, or apart
        parts = [t.view(-1, h, d) for t, h in zip(x.split([hq * d, hkv * d, hkv * d], dim=1),
                                                  (hq, hkv, hkv))]
        if not case["fused"]:
            parts = [t.contiguous() for t in parts]
        state["qkv"] = parts
        far = max(h + n for h, n in lens)
    else:
        state["q"] = x.view(-1, hq, d)
    if own:
        from llm_serving_layer_amd import (BlockAllocator, MI355XBackend, RotaryTable,
                                           ScheduledSeq, SequenceBlocks, build_batch_meta)
        bounded = case["kind"] == "selected" or case.get("bounds", False)
        bk = MI355XBackend(1, nb, PAGE, hkv, hq, d, device=DEV, dtype=DTYPES[case["dtype"]],
                           page_bounds=bounded)
        bk.k_pool[0].copy_(k)
        bk.v_pool[0].copy_(v)
        if bounded:
            bk.refresh_page_bounds()
        alloc = BlockAllocator(nb, PAGE)
        alloc.allocate(nb)
        seqs = []
        for i, ((h, n), ids) in enumerate(zip(lens, tables)):
            s = SequenceBlocks(alloc, seq_id=i)
            s.block_ids, s.num_tokens = list(ids), h + n
            seqs.append(ScheduledSeq(s, [0] * n))
        state.update(bk=bk, meta=build_batch_meta(seqs, DEV, PAGE))
        if case["kind"] == "rotate":
            state["table"] = RotaryTable(far, case["rotary_dim"], theta=THETA,
                                         interleaved=case["interleaved"], device=DEV)
            state["cache"] = {"k": bk.k_pool[0], "v": bk.v_pool[0]}
            if bounded:
                state["cache"].update(lo=bk.key_bounds[0][0], hi=bk.key_bounds[0][1])
        return state
    state.update(k=k, v=v, ids=[torch.tensor(t, device=DEV) for t in tables],
                 lens=[h + n for h, n in lens])
    if case["kind"] == "rotate":
        angle = torch.arange(far, device=DEV).double()[:, None] * _frequencies(case)
        state["cos"], state["sin"] = angle.cos().float(), angle.sin().float()
        pos = [torch.arange(h, h + n, device=DEV) for h, n in lens]
        state["pos"] = torch.cat(pos)
        state["slots"] = torch.cat([t[p // PAGE] * PAGE + p % PAGE
                                    for t, p in zip(state["ids"], pos)])
        # the pages that this step's tokens complete
        state["done"] = torch.cat([t[h // PAGE:(h + n) // PAGE]
                                   for t, (h, n) in zip(state["ids"], lens)])
    if case["kind"] == "selected" or case.get("bounds", False):
        state["lo"], state["hi"] = _bounds(k)
    return state


# --------------------------------------------------------------- plain form ---

def _turn(x, cos, sin, case):
    """x turned by its positions, in 32 bits."""
    r = case["rotary_dim"]
    y = x.float()
    out = y.clone()
    a, b = ((y[..., 0:r:2], y[..., 1:r:2]) if case["interleaved"]
            else (y[..., :r // 2], y[..., r // 2:r]))
    c, s = cos[:, None, :], sin[:, None, :]
    ra, rb = a * c - b * s, b * c + a * s
    if case["interleaved"]:
        out[..., 0:r:2], out[..., 1:r:2] = ra, rb
    else:
        out[..., :r // 2], out[..., r // 2:r] = ra, rb
    return out.to(x.dtype)


def _attend_rows(q, k, v, scale):
    """(Hq, D) queries of one token over (N, Hkv, D) keys and values, 32 bits."""
    hkv, d = k.shape[1], k.shape[2]
    kk = k.float().permute(1, 2, 0).contiguous()
    vv = v.float().permute(1, 0, 2).contiguous()
    s = torch.matmul(q.float().view(hkv, -1, d), kk) * scale
    p = torch.exp(s - s.amax(dim=-1, keepdim=True))
    o = torch.matmul(p, vv) / p.sum(dim=-1, keepdim=True)
    return o.reshape(-1, d).to(q.dtype)


def _plain_rotate(st):
    case = st["case"]
    q, k, v = st["qkv"]
    cos, sin = st["cos"][st["pos"]], st["sin"][st["pos"]]
    rq = _turn(q, cos, sin, case)
    st["k"].flatten(0, 1)[st["slots"]] = _turn(k, cos, sin, case)
    st["v"].flatten(0, 1)[st["slots"]] = v
    out = {"q": rq, "k": st["k"], "v": st["v"]}
    if case["bounds"]:
        lo, hi = _bounds(st["k"][st["done"]])
        st["lo"][st["done"]], st["hi"][st["done"]] = lo, hi
        out.update(lo=st["lo"], hi=st["hi"])
    return out


def _plain_shared(st):
    out = torch.empty_like(st["q"])
    for i, (ids, n) in enumerate(zip(st["ids"], st["lens"])):
        out[i] = _attend_rows(st["q"][i], st["k"][ids].flatten(0, 1)[:n],
                              st["v"][ids].flatten(0, 1)[:n], st["scale"])
    return out


def _plain_selected(st):
    q, want = st["q"], st["case"]["pages"]
    hkv, d = st["case"]["n_kv"], st["case"]["head_dim"]
    out = torch.empty_like(q)
    width = min(want, max(len(t) for t in st["ids"]))
    chosen = torch.full((len(st["ids"]), hkv, width), -1, dtype=torch.int32, device=q.device)
    heads = torch.arange(hkv, device=q.device)[:, None]
    for i, (ids, n) in enumerate(zip(st["ids"], st["lens"])):
        npg = len(ids)
        if npg <= want:
            pick = torch.arange(npg, device=q.device).expand(hkv, npg)
        else:
            qq = q[i].double().view(hkv, -1, d)
            lo = st["lo"][ids[:-1]].double().permute(1, 2, 0).contiguous()
            hi = st["hi"][ids[:-1]].double().permute(1, 2, 0).contiguous()
            b = torch.matmul(qq.clamp(min=0), hi) + torch.matmul(qq.clamp(max=0), lo)
            best = torch.sort(b.amax(dim=1), dim=-1, descending=True, stable=True).indices
            pick = torch.sort(best[:, :want - 1], dim=-1).values
            pick = torch.cat([pick, torch.full_like(heads, npg - 1)], dim=1)
        chosen[i, :, :pick.shape[1]] = pick.int()
        live = (pick.shape[1] - 1) * PAGE + n - (npg - 1) * PAGE
        # (pages, page rows, D) of each head, the last page's rows last
        k = st["k"][ids[pick], :, heads].flatten(1, 2)[:, :live]
        v = st["v"][ids[pick], :, heads].flatten(1, 2)[:, :live]
        out[i] = _attend_rows(q[i], k.transpose(0, 1), v.transpose(0, 1), st["scale"])
    return {"out": out, "pages": chosen}


def run(state):
    case = state["case"]
    if not own:
        return {"rotate": _plain_rotate, "shared": _plain_shared,
                "selected": _plain_selected}[case["kind"]](state)
    bk, meta = state["bk"], state["meta"]
    if case["kind"] == "rotate":
        q, k, v = state["qkv"]
        return {"q": bk.append_kv_rotated(0, q, k, v, meta, state["table"]), **state["cache"]}
    if case["kind"] == "shared":
        return bk.attend_shared(state["q"], 0, state["scale"], meta)
    out, pages = bk.attend_selected(state["q"], 0, state["scale"], meta, case["pages"],
                                    return_pages=True)
    return {"out": out, "pages": pages}


# ------------------------------------------------------------- work, exact ---

def work(case):
    eb = 4 if case["dtype"] == "float32" else 2
    hq, hkv, d = case["n_heads"], case["n_kv"], case["head_dim"]
    lens = _lengths(case)
    if case["kind"] == "rotate":
        tokens = sum(n for _, n in lens)
        positions = len({p for h, n in lens for p in range(h, h + n)})
        total = 2 * tokens * (hq + 2 * hkv) * d * eb + positions * case["rotary_dim"] * 4
        if case["bounds"]:   # rows that earlier steps wrote to the pages now complete
            done = [(h, (h + n) // PAGE - h // PAGE) for h, n in lens]
            total += sum((h % PAGE + 2 * c) * hkv * d * eb for h, c in done if c)
        return {"bytes": total, "flops": 3 * tokens * (hq + hkv) * case["rotary_dim"]}
    qo = 2 * len(lens) * hq * d * eb
    row = 2 * hkv * d * eb
    keys = sum(h + n for h, n in lens)
    if case["kind"] == "shared":
        groups = min(case["groups"], case["n"])
        once = keys - (case["n"] - 1) * case["root"] - (case["n"] - groups) * case["branch"]
        return {"bytes": qo + once * row, "flops": 4 * d * hq * keys}
    read = bounds = 0
    for h, n in lens:
        npg = _pages(h + n)
        read += h + n if npg <= case["pages"] else h + n - (npg - case["pages"]) * PAGE
        bounds += npg - 1 if npg > case["pages"] else 0
    width = min(case["pages"], max(_pages(h + n) for h, n in lens))
    return {"bytes": qo + (read + bounds) * row + len(lens) * hkv * width * 4,
            "flops": 4 * d * hq * (read + bounds)}


def _exact_rotate(case, tables, k, v, x):
    hq, hkv, d, r = case["n_heads"], case["n_kv"], case["head_dim"], case["rotary_dim"]
    x = x.double().view(x.shape[0], hq + 2 * hkv, d)
    pos = torch.cat([torch.arange(h, h + n, device=DEV) for h, n in _lengths(case)]).double()
    # each pair as one complex number, times e^(i p f)
    turn = torch.polar(torch.ones((), dtype=torch.float64, device=DEV),
                       pos[:, None] * _frequencies(case)[None, :])[:, None, :]
    rows = x[:, :hq + hkv]
    head = rows[..., :r]
    if case["interleaved"]:
        z = torch.view_as_complex(head.reshape(*head.shape[:2], r // 2, 2).contiguous()) * turn
        head = torch.view_as_real(z).flatten(2)
    else:
        z = torch.complex(head[..., :r // 2].contiguous(), head[..., r // 2:].contiguous()) * turn
        head = torch.cat([z.real, z.imag], dim=-1)
    rows = torch.cat([head, rows[..., r:]], dim=-1)
    k, v = k.double(), v.double()
    low, high = _bounds(k) if case["bounds"] else (None, None)
    at = 0
    for (h, n), ids in zip(_lengths(case), tables):
        for j0 in range(h // PAGE, (h + n - 1) // PAGE + 1):
            a, b = max(h, j0 * PAGE), min(h + n, (j0 + 1) * PAGE)
            span = slice(a - j0 * PAGE, b - j0 * PAGE)
            k[ids[j0], span] = rows[at + a - h:at + b - h, hq:]
            v[ids[j0], span] = x[at + a - h:at + b - h, hq + hkv:]
            if case["bounds"] and b == (j0 + 1) * PAGE:
                low[ids[j0]], high[ids[j0]] = k[ids[j0]].amin(0), k[ids[j0]].amax(0)
        at += n
    out = {"q": rows[:, :hq].contiguous(), "k": k, "v": v}
    if case["bounds"]:
        out.update(lo=low, hi=high)
    return out


def _exact_attention(case, q, keys, values):
    """One token's (Hq, D) output; keys and values a (N, D) tensor a KV head."""
    groups, outs = case["n_heads"] // case["n_kv"], []
    for h in range(case["n_kv"]):
        s = q[h * groups:(h + 1) * groups].double() @ keys[h].double().t().contiguous()
        outs.append(torch.softmax(s / math.sqrt(case["head_dim"]), dim=-1) @ values[h].double())
    return torch.cat(outs)


def exact(case, seed):
    _, tables, k, v, x = _inputs(case, seed)
    if case["kind"] == "rotate":
        return _exact_rotate(case, tables, k, v, x)
    hkv, d = case["n_kv"], case["head_dim"]
    groups = case["n_heads"] // hkv
    q = x.view(-1, case["n_heads"], d)
    out = torch.empty(q.shape, dtype=torch.float64, device=DEV)
    width = min(case.get("pages", 0), max(len(t) for t in tables))
    pages = torch.full((len(tables), hkv, width), -1, dtype=torch.int32)
    for i, ((h0, n), ids) in enumerate(zip(_lengths(case), tables)):
        total, npg = h0 + n, len(ids)
        kk, vv = k[ids], v[ids]
        if case["kind"] == "shared" or npg <= case["pages"]:
            if case["kind"] == "selected":
                pages[i, :, :npg] = torch.arange(npg, dtype=torch.int32)
            kk, vv = kk.flatten(0, 1)[:total], vv.flatten(0, 1)[:total]
            out[i] = _exact_attention(case, q[i], kk.unbind(1), vv.unbind(1))
            continue
        lo, hi = _bounds(kk[:-1].double())
        keys, values = [], []
        for h in range(hkv):
            best = torch.stack([torch.maximum(qg * lo[:, h], qg * hi[:, h]).sum(-1)
                                for qg in q[i, h * groups:(h + 1) * groups].double()]).amax(0)
            rank = sorted(range(npg - 1), key=lambda p, s=best.tolist(): (-s[p], p))
            take = sorted(rank[:case["pages"] - 1]) + [npg - 1]
            pages[i, h] = torch.tensor(take, dtype=torch.int32)
            live = (len(take) - 1) * PAGE + total - (npg - 1) * PAGE
            keys.append(kk[take, :, h].flatten(0, 1)[:live])
            values.append(vv[take, :, h].flatten(0, 1)[:live])
        out[i] = _exact_attention(case, q[i], keys, values)
    return out if case["kind"] == "shared" else {"out": out, "pages": pages.to(DEV)}
