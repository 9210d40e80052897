"""
Performance cases of serving from a cache held in 4 bits, and of drafted
tokens. Three kinds of case:

* ``store``   one layer's append to the 4-bit cache: each row of a KV head is
  cut into groups (64 elements, or the whole row where head_dim is no multiple
  of 64); a group keeps 4-bit codes, a step and a zero; then the appended rows
  read back as the values that the cache holds for them.
* ``attend``  one layer's causal attention over the 4-bit cache: single tokens,
  a few drafted tokens a sequence, or prompt chunks.
* ``verify``  drafted tokens checked against the target's logits with given
  uniform numbers: how many of each sequence's drafts stand, and the token
  drawn behind them.

A group's zero is its least element rounded down to float16 (elements are
brought to +-65504 first), its step the least float16 that is not below
(largest - zero) / 15; code c = (x - zero) / step rounded to the nearest whole
number (ties to even), at most 15; the cache holds zero + c step.

A draft x at a row with target probabilities p (softmax of logits /
temperature) and draft probabilities q stands if u q(x) < p(x), u the row's
number; without draft probabilities q is 1 at x. The first that does not stand
ends the sequence's run, and its place takes a token drawn from max(p - q, 0);
behind a run that stands whole one is drawn from the last row's p. Drawn is the
first token whose running sum of weights exceeds the last row's number times
their sum. Temperature 0: a draft stands if it is the row's largest logit (the
first of equals), and that token is taken.

With ``own`` false everything is elementary torch in 32 bits (64 for codes
next to a border, and for probabilities, whose borders decide); with ``own``
true the calls of ``FourBitBackend`` and ``verify_drafts``. Lengths are fixed
by the case; page tables, cache contents, activations, logits and numbers come
from the seed.
"""

from __future__ import annotations

import math
import random

import torch

own = False

DEV = "cuda:0"
PAGE = 16
DTYPES = {"float16": torch.float16, "bfloat16": torch.bfloat16, "float32": torch.float32}

# 32 query heads over 8 KV heads at head_dim 64, the benchmark's geometry
BASE = {"n_kv": 8, "n_heads": 32, "head_dim": 64}
D128 = {"n_kv": 8, "n_heads": 32, "head_dim": 128}
VOCAB = 128256


def _paged(kind, name, dtype, *, n, lo, hi, new_lo=1, new_hi=1, law="uniform", mean=0,
           lens_seed=20260731, **geom):
    case = {"kind": kind, "dtype": dtype, **BASE, **geom, "n": n, "lo": lo, "hi": hi,
            "new_lo": new_lo, "new_hi": new_hi, "law": law, "mean": mean,
            "lens_seed": lens_seed}
    return {"name": name, **case} if name else case


def _verify(name, dtype, *, n, drafts_lo, drafts_hi, vocab=VOCAB, probs=None, temps=(1.0,), pad=0,
            lens_seed=20260731):
    case = {"kind": "verify", "dtype": dtype, "n": n, "drafts_lo": drafts_lo,
            "drafts_hi": drafts_hi, "vocab": vocab, "probs": probs or "", "temps": " ".join(map(str, temps)),
            "pad": pad, "lens_seed": lens_seed}
    return {"name": name, **case} if name else case


def listed():
    return [
        # one user alone: the new token's k, v of one layer
        _paged("store", "store_single", "float16", n=1, lo=1371, hi=1371),
        # a batch-256 decode step of a model with head_dim 128, in bf16
        _paged("store", "store_decode", "bfloat16", n=256, lo=16, hi=400, **D128),
        # chunked prefill of eight requests at once
        _paged("store", "store_chunks", "bfloat16", n=8, lo=135, hi=135, new_lo=512, new_hi=1000,
               **D128),
        # one user with a long history
        _paged("attend", "attend_single", "float16", n=1, lo=32749, hi=32749),
        # the headline decode batch
        _paged("attend", "attend_batch", "float16", n=256, lo=1, hi=2048, law="lognormal",
               mean=258),
        # long documents
        _paged("attend", "attend_long", "bfloat16", n=16, lo=20000, hi=60000, **D128),
        # a step that verifies up to five drafted tokens a sequence
        _paged("attend", "attend_drafts", "bfloat16", n=48, lo=2000, hi=8000, new_lo=2, new_hi=6,
               **D128),
        # chunked prefill over a cached prefix, the benchmark's
        _paged("attend", "attend_chunks", "float16", n=8, lo=1536, hi=1536, new_lo=512,
               new_hi=512),
        # one user, four drafts of a small model, the model's own vocabulary
        _verify("verify_single", "float16", n=1, drafts_lo=4, drafts_hi=4, probs="float32",
                temps=(0.7,)),
        # a batch with the drafting model's probabilities, greedy requests among it
        _verify("verify_batch", "bfloat16", n=64, drafts_lo=1, drafts_hi=5, probs="float32",
                temps=(0.0, 0.6, 0.8, 1.0)),
        # drafts looked up in the prompt, without probabilities; rows padded
        _verify("verify_lookup", "float16", n=128, drafts_lo=0, drafts_hi=3, vocab=32003, pad=61,
                temps=(0.8,)),
        # logits in 32 bits, long drafts
        _verify("verify_wide", "float32", n=24, drafts_lo=8, drafts_hi=8, probs="bfloat16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


GEOMS = [(8, 32, 64), (8, 32, 64), (8, 32, 128), (8, 32, 128), (2, 8, 128), (8, 8, 64), (4, 8, 64),
         (2, 32, 64), (4, 32, 128), (1, 8, 64), (3, 12, 64), (4, 24, 128)]


def draw(rng):
    kind = rng.choices(["store", "attend", "verify"], [1, 2, 1.3])[0]
    seed = rng.randrange(1 << 30)
    if kind == "verify":
        dtype = rng.choices(["float16", "bfloat16", "float32"], [2, 2, 1])[0]
        vocab, hi = _log(rng, 500, 150000), rng.randint(0, 8)
        n = min(_log(rng, 1, 160), max(1, 30_000_000 // (vocab * (hi + 1))))
        temps = rng.choice([[1.0], [0.7], [0.0], [0.0, 0.5, 1.0, 1.3]])
        return _verify(None, dtype, n=n, drafts_lo=rng.randint(0, hi), drafts_hi=hi, vocab=vocab,
                       probs=rng.choice([None, "float32", "float32", dtype]), temps=temps,
                       pad=rng.choice([0, 0, rng.randint(1, 200)]), lens_seed=seed)
    n_kv, n_heads, d = rng.choice(GEOMS)
    geom = {"n_kv": n_kv, "n_heads": n_heads, "head_dim": d, "lens_seed": seed}
    dtype = rng.choice(["float16", "bfloat16"])
    if kind == "store":
        if rng.random() < 0.5:
            n = _log(rng, 1, 1000)
            return _paged("store", None, dtype, n=n, lo=1, hi=min(4000, 200000 // n), **geom)
        n, hi = rng.randint(1, 8), _log(rng, 2, 1000)
        return _paged("store", None, dtype, n=n, lo=1, hi=1500, new_lo=max(1, hi // 2), new_hi=hi,
                      **geom)
    form = rng.choices(["tokens", "drafts", "chunks"], [3, 1, 1])[0]
    if form == "chunks":
        n, hi = rng.randint(1, 6), _log(rng, 10, 700)
        return _paged("attend", None, dtype, n=n, lo=1, hi=_log(rng, 10, 1500),
                      new_lo=max(1, hi // 3), new_hi=hi, **geom)
    n = _log(rng, 1, 250)
    hi = min(_log(rng, 20, 60000), 400000 // n)
    new = rng.randint(2, 9) if form == "drafts" else 1
    return _paged("attend", None, dtype, n=n, lo=max(1, hi // 4), hi=hi, new_lo=1, new_hi=new,
                  **geom)


# ------------------------------------------------------------------ inputs ---

def _pages(n):
    return -(-n // PAGE)


def _lengths(case):
    """(history, new tokens) of every sequence; for ``verify`` (0, 1 + drafts).
    ``lo`` to ``hi`` are the lengths before prompt chunks and with other new
    tokens."""
    rng = random.Random(case["lens_seed"])
    if case["kind"] == "verify":
        return [(0, 1 + rng.randint(case["drafts_lo"], case["drafts_hi"]))
                for _ in range(case["n"])]
    out = []
    for _ in range(case["n"]):
        if case["law"] == "lognormal":
            mu = math.log(case["mean"]) - 0.8 ** 2 / 2.0
            total = max(case["lo"], min(case["hi"], int(round(rng.lognormvariate(mu, 0.8)))))
        else:
            total = rng.randint(case["lo"], case["hi"])
        new = rng.randint(case["new_lo"], case["new_hi"])
        out.append((total, new) if case["new_hi"] > 9 else (max(0, total - new), new))
    return out


def _tables(case, seed):
    """(blocks of the pool, page ids of every sequence)."""
    own_pages = [_pages(h + n) for h, n in _lengths(case)]
    nb = sum(own_pages) + max(8, sum(own_pages) // 16)
    order = list(range(nb))
    random.Random(seed).shuffle(order)
    tables, at = [], 0
    for k in own_pages:
        tables.append(order[at:at + k])
        at += k
    return nb, tables


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _values(shape, dtype, g):
    return torch.randn(shape, generator=g, device=DEV).mul_(0.5).to(dtype)


def _inputs(case, seed):
    """(blocks, tables, the cache's rows before they are quantised or None, the
    step's q or its k and v). A few of the keys' dims lie far from zero, as in a
    model's."""
    dt, d, hkv = DTYPES[case["dtype"]], case["head_dim"], case["n_kv"]
    nb, tables = _tables(case, seed)
    g = _gen(seed)
    tokens = sum(n for _, n in _lengths(case))
    centre = torch.randn((hkv, d), generator=g, device=DEV)
    centre = torch.where(centre.abs() > 1.9, 2 * centre, 0 * centre).to(dt)
    if case["kind"] == "store":
        return nb, tables, None, (_values((tokens, hkv, d), dt, g) + centre,
                                  _values((tokens, hkv, d), dt, g))
    rows = (_values((nb * PAGE, hkv, d), dt, g).add_(centre),
            _values((nb * PAGE, hkv, d), dt, g))
    return nb, tables, rows, _values((tokens, case["n_heads"], d), dt, g)


def _drafting(case, seed):
    """Logits (a view of wider rows where the case pads them), the step's tokens,
    the rows' numbers, the drafts' probabilities (or None) and the temperatures."""
    g, v = _gen(seed), case["vocab"]
    lens = [n for _, n in _lengths(case)]
    rows = sum(lens)
    base = torch.randn((rows, v), generator=g, device=DEV).mul_(3.0)
    wide = torch.zeros((rows, v + case["pad"]), dtype=DTYPES[case["dtype"]], device=DEV)
    wide[:, :v] = base
    # the drafting model: near the target
    base.add_(torch.randn((rows, v), generator=g, device=DEV).mul_(0.7))
    first = torch.zeros(rows, dtype=torch.bool)
    first[torch.tensor([0] + lens[:-1]).cumsum(0)] = True
    before = torch.cat([first[1:], torch.ones(1, dtype=torch.bool)]).to(DEV)
    base = base[~before]      # the rows that a draft follows
    tokens = torch.randint(0, v, (rows,), generator=g, device=DEV)
    q = None
    if base.shape[0]:
        if case["probs"]:
            q = torch.softmax(base, dim=-1)
            tokens[~first.to(DEV)] = torch.multinomial(q, 1, generator=g)[:, 0]
            q = q.to(DTYPES[case["probs"]])
        else:
            tokens[~first.to(DEV)] = base.argmax(-1)
    numbers = torch.rand(rows, generator=g, device=DEV)
    rng = random.Random(seed)
    temps = [float(rng.choice(case["temps"].split())) for _ in lens]
    return wide[:, :v], tokens, numbers, q, temps


def prepare(case, seed):
    lens = _lengths(case)
    state = {"case": case}
    if case["kind"] == "verify":
        logits, tokens, numbers, q, temps = _drafting(case, seed)
        state.update(logits=logits, tokens=tokens, numbers=numbers, q=q,
                     temps=torch.tensor(temps, dtype=torch.float32, device=DEV))
        if own:
            state["meta"] = _meta(case, sum(_pages(n) for _, n in lens), None)
        else:
            ends = torch.tensor([n for _, n in lens], device=DEV).cumsum(0)
            width = max(n for _, n in lens)
            drafts = torch.tensor([n - 1 for _, n in lens], device=DEV)
            at = (ends - drafts - 1)[:, None] + torch.arange(width, device=DEV)
            state.update(drafts=drafts, at=at, last=ends - 1)
        return state
    hq, hkv, d = case["n_heads"], case["n_kv"], case["head_dim"]
    nb, tables, rows, x = _inputs(case, seed)
    state.update(x=x, scale=d ** -0.5)
    if own:
        from llm_serving_layer_amd import FourBitBackend
        bk = FourBitBackend(1, nb, PAGE, hkv, hq, d, device=DEV, dtype=DTYPES[case["dtype"]])
        if rows is not None:
            bk.append_kv(0, *rows, _whole(nb))
        state.update(bk=bk, meta=_meta(case, nb, tables))
        return state
    ids = [torch.tensor(t, device=DEV) for t in tables]
    if case["kind"] == "store":
        pos = [torch.arange(h, h + n, device=DEV) for h, n in lens]
        state["slots"] = torch.cat([t[p // PAGE] * PAGE + p % PAGE for t, p in zip(ids, pos)])
        shape, groups = (nb * PAGE, hkv, d), _groups(d)
        state["cache"] = [(torch.zeros(shape, dtype=torch.uint8, device=DEV),
                           *(torch.zeros((*shape[:2], groups), device=DEV) for _ in range(2)))
                          for _ in range(2)]
    else:
        state.update(cache=[_quantise(r) for r in rows], ids=ids)
    return state


def _meta(case, nb, tables):
    from llm_serving_layer_amd import (BlockAllocator, ScheduledSeq, SequenceBlocks,
                                       build_batch_meta)
    alloc = BlockAllocator(nb, PAGE)
    free = alloc.allocate(nb)
    seqs = []
    for i, (h, n) in enumerate(_lengths(case)):
        s = SequenceBlocks(alloc, seq_id=i)
        if tables is None:
            ids, free = free[:_pages(n)], free[_pages(n):]
        else:
            ids = tables[i]
        s.block_ids, s.num_tokens = list(ids), h + n
        seqs.append(ScheduledSeq(s, [0] * n))
    return build_batch_meta(seqs, DEV, PAGE)


def _whole(nb):
    """One sequence that owns every row of the pool, as a prompt."""
    from llm_serving_layer_amd import (BlockAllocator, ScheduledSeq, SequenceBlocks,
                                       build_batch_meta)
    alloc = BlockAllocator(nb, PAGE)
    alloc.allocate(nb)
    s = SequenceBlocks(alloc, seq_id=0)
    s.block_ids, s.num_tokens = list(range(nb)), nb * PAGE
    return build_batch_meta([ScheduledSeq(s, [0] * (nb * PAGE))], DEV, PAGE)


# --------------------------------------------------------------- plain form ---

def _groups(d):
    return d // 64 if d % 64 == 0 else 1


def _step_toward(h, up):
    """The next float16 above (below) h, for finite h."""
    bits = h.view(torch.int16).int()
    away = (bits >= 0) == up
    bits = torch.where(away, bits + 1, bits - 1)
    zero = (h == 0)
    bits = torch.where(zero, torch.full_like(bits, 1 if up else -32767), bits)
    return bits.to(torch.int16).view(torch.float16)


def _quantise(x):
    """(codes uint8, step, zero float32) of rows (N, Hkv, D)."""
    codes, steps, zeros = [], [], []
    g = _groups(x.shape[-1])
    for part in x.split(65536):
        y = part.double().clamp(-65504.0, 65504.0).unflatten(-1, (g, -1))
        lo, hi = y.amin(-1), y.amax(-1)
        z = lo.to(torch.float16)
        z = torch.where(z.double() > lo, _step_toward(z, False), z)
        need = (hi - z.double()) / 15.0
        s = need.to(torch.float16)
        s = torch.where(s.double() < need, _step_toward(s, True), s)
        zd, sd = z.double()[..., None], s.double()[..., None]
        c = torch.where(sd > 0, torch.round((y - zd) / torch.where(sd > 0, sd, 1.0 + 0 * sd)), 0 * y)
        codes.append(c.clamp(0, 15).to(torch.uint8).flatten(-2))
        steps.append(s.float())
        zeros.append(z.float())
    return torch.cat(codes), torch.cat(steps), torch.cat(zeros)


def _held(codes, step, zero):
    """The values that codes stand for, in 32 bits."""
    c = codes.float().unflatten(-1, (step.shape[-1], -1))
    return (c * step[..., None] + zero[..., None]).flatten(-2)


def _plain_store(st):
    out = []
    for x, cache in zip(st["x"], st["cache"]):
        for held, new in zip(cache, _quantise(x)):
            held[st["slots"]] = new
        out.append(_held(*(held[st["slots"]] for held in cache)).to(x.dtype))
    return {"k": out[0], "v": out[1]}


def _plain_attend(st):
    q, case = st["x"], st["case"]
    hkv, d = case["n_kv"], case["head_dim"]
    out = torch.empty_like(q)
    at = 0
    for (h, n), ids in zip(_lengths(case), st["ids"]):
        rows = (ids[:, None] * PAGE + torch.arange(PAGE, device=q.device)).flatten()[:h + n]
        k, v = (_held(*(held[rows] for held in cache)) for cache in st["cache"])
        qq = q[at:at + n].float().view(n, hkv, -1, d).permute(1, 2, 0, 3).reshape(hkv, -1, d)
        s = torch.matmul(qq, k.permute(1, 2, 0).contiguous()).view(hkv, -1, n, h + n)
        s = s * st["scale"]
        see = torch.arange(h + n, device=q.device) <= torch.arange(h, h + n, device=q.device)[:, None]
        s = torch.where(see, s, torch.full_like(s, -math.inf))
        p = torch.exp(s - s.amax(dim=-1, keepdim=True))
        p = (p / p.sum(dim=-1, keepdim=True)).view(hkv, -1, h + n)
        o = torch.matmul(p, v.permute(1, 0, 2).contiguous()).view(hkv, -1, n, d)
        out[at:at + n] = o.permute(2, 0, 1, 3).reshape(n, -1, d).to(q.dtype)
        at += n
    return out


def _plain_verify(st):
    x, tokens, numbers, q = st["logits"], st["tokens"], st["numbers"].double(), st["q"]
    drafts, at, last, temps = st["drafts"], st["at"], st["last"], st["temps"].double()
    (n, width), (rows, vocab) = at.shape, x.shape
    index = torch.arange(vocab, device=x.device)
    top = torch.where(x == x.amax(-1, keepdim=True), index, vocab).amin(-1)
    owner = torch.repeat_interleave(torch.arange(n, device=x.device), drafts + 1, output_size=rows)
    t = temps[owner]
    y = x.double() / torch.where(t > 0, t, 1.0 + 0 * t)[:, None]
    e = torch.exp(y - y.amax(-1, keepdim=True))
    p = e / e.sum(-1, keepdim=True)
    # the draft behind each row (none behind a sequence's last)
    nxt = torch.roll(tokens, -1)
    follows = torch.arange(rows, device=x.device) != last[owner]
    drow = torch.arange(rows, device=x.device) - owner      # row of q
    qx = torch.ones(rows, dtype=torch.float64, device=x.device)
    if q is not None:
        drow = drow.clamp(max=q.shape[0] - 1)
        qx = q[drow, nxt].double()
    stands = torch.where(t > 0, numbers * qx < p.gather(1, nxt[:, None])[:, 0], top == nxt)
    stands = stands & follows
    inside = torch.arange(width, device=x.device) < drafts[:, None]
    run = (stands[at.clamp(max=rows - 1)] & inside).int().cumprod(1).sum(1)
    row = at[:, 0] + run
    w = p[row]
    ended = (run < drafts)[:, None]
    if q is not None:
        rest = (w - q[drow[row]].double()).clamp(min=0)
    else:
        rest = torch.where(index == nxt[row][:, None], 0 * w, w)
    rest = torch.where(rest.sum(-1, keepdim=True) > 0, rest, w)
    w = torch.where(ended, rest, w)
    total = w.cumsum(-1)
    pick = (total <= numbers[last][:, None] * total[:, -1:]).sum(-1)
    pick = torch.minimum(pick, torch.where(w > 0, index, 0).amax(-1))
    pick = torch.where(temps > 0, pick, top[row])
    j = torch.arange(width, device=x.device)
    kept = tokens[(at + 1).clamp(max=rows - 1)]
    ids = torch.where(j < run[:, None], kept, torch.where(j == run[:, None], pick[:, None], -1))
    return {"ids": ids, "accepted": run.long()}


def run(state):
    kind = state["case"]["kind"]
    if not own:
        return {"store": _plain_store, "attend": _plain_attend, "verify": _plain_verify}[kind](state)
    if kind == "store":
        bk, meta = state["bk"], state["meta"]
        bk.append_kv(0, *state["x"], meta)
        k, v = bk.read_kv(0, meta.slot_mapping)
        return {"k": k, "v": v}
    if kind == "attend":
        return state["bk"].attend(state["x"], 0, state["scale"], state["meta"])
    from llm_serving_layer_amd.sampling import verify_drafts
    ids, accepted = verify_drafts(state["logits"], state["tokens"], state["meta"],
                                  state["numbers"], draft_probs=state["q"],
                                  temperature=state["temps"])
    return {"ids": ids, "accepted": accepted}


# ------------------------------------------------------------- work, exact ---

def work(case):
    lens = _lengths(case)
    eb = 4 if case["dtype"] == "float32" else 2
    tokens = sum(n for _, n in lens)
    if case["kind"] == "verify":
        pb = {"": 0, "float32": 4}.get(case["probs"], 2)
        # every row of logits; of the drafts' probabilities one row a sequence
        total = tokens * case["vocab"] * eb + case["n"] * case["vocab"] * pb * (tokens > case["n"])
        return {"bytes": total + tokens * 12 + case["n"] * 16, "flops": 4 * tokens * case["vocab"]}
    hq, hkv, d = case["n_heads"], case["n_kv"], case["head_dim"]
    row = 2 * hkv * (d // 2 + 4 * _groups(d))          # a token's K and V in the cache
    if case["kind"] == "store":
        return {"bytes": tokens * (4 * hkv * d * eb + row), "flops": 8 * tokens * hkv * d}
    seen = sum(n * h + n * (n + 1) // 2 for h, n in lens)
    keys = sum(h + n for h, n in lens)
    return {"bytes": 2 * tokens * hq * d * eb + keys * row, "flops": 4 * d * hq * seen}


def _half_floor(x):
    """x rounded down to a float16, in 64 bits."""
    e = torch.frexp(x).exponent.double() - 1
    ulp = torch.exp2(e.clamp(min=-14.0) - 10.0)
    return torch.floor(x / ulp) * ulp


def _exact_rows(x):
    """What the cache holds for rows x, in 64 bits."""
    out = []
    g = _groups(x.shape[-1])
    for part in x.split(65536):
        y = part.double().clamp(-65504.0, 65504.0).unflatten(-1, (g, -1))
        zero = _half_floor(y.amin(-1, keepdim=True))
        step = -_half_floor((zero - y.amax(-1, keepdim=True)) / 15)
        t = (y - zero) / step.clamp(min=2.0 ** -24)
        c = torch.floor(t)
        rest = t - c
        c += ((rest > 0.5) | ((rest == 0.5) & (c % 2 == 1))).double()
        out.append((zero + c.clamp(max=15.0) * step).flatten(-2))
    return torch.cat(out)


def _exact_verify(case, seed):
    logits, tokens, numbers, q, temps = _drafting(case, seed)
    lens = [n for _, n in _lengths(case)]
    ids = torch.full((len(lens), max(lens)), -1, dtype=torch.int64)
    counts = torch.zeros(len(lens), dtype=torch.int64)
    u, tok = numbers.double().tolist(), tokens.tolist()
    at = 0
    for i, (n, t) in enumerate(zip(lens, temps)):
        run, pick = 0, None
        while pick is None:
            row = logits[at + run].double()
            x = tok[at + run + 1] if run < n - 1 else None
            if t == 0:
                best = int((row == row.max()).nonzero()[0])
                if x == best:
                    run += 1
                else:
                    pick = best
                continue
            t32 = float(torch.tensor(t, dtype=torch.float32))
            p = torch.softmax(row / t32, dim=-1)
            if x is not None:
                qr = None if q is None else q[at - i + run].double()
                if u[at + run] * (1.0 if qr is None else float(qr[x])) < float(p[x]):
                    run += 1
                    continue
                w = p.clone() if qr is None else torch.relu(p - qr)
                if qr is None:
                    w[x] = 0.0
                p = w if float(w.sum()) > 0 else p
            cum = torch.cumsum(p, 0)
            target = (cum[-1] * u[at + n - 1]).reshape(1)
            pick = int(torch.searchsorted(cum, target, right=True))
            pick = min(pick, int(p.nonzero()[-1]))
        ids[i, :run] = torch.tensor(tok[at + 1:at + 1 + run], dtype=torch.int64)
        ids[i, run], counts[i] = pick, run
        at += n
    return {"ids": ids.to(DEV), "accepted": counts.to(DEV)}


def exact(case, seed):
    if case["kind"] == "verify":
        return _exact_verify(case, seed)
    nb, tables, rows, x = _inputs(case, seed)
    if case["kind"] == "store":
        return {"k": _exact_rows(x[0]), "v": _exact_rows(x[1])}
    hkv, d = case["n_kv"], case["head_dim"]
    out = torch.empty(x.shape, dtype=torch.float64, device=DEV)
    at = 0
    for (h, n), ids in zip(_lengths(case), tables):
        ix = torch.tensor([b * PAGE + r for b in ids for r in range(PAGE)], device=DEV)[:h + n]
        hidden = torch.ones((n, h + n), dtype=torch.bool, device=DEV).triu(h + 1)
        k, v = _exact_rows(rows[0][ix]), _exact_rows(rows[1][ix])
        for head in range(case["n_heads"]):
            of = head * hkv // case["n_heads"]
            s = x[at:at + n, head].double() @ k[:, of].t().contiguous()
            s = (s / math.sqrt(d)).masked_fill(hidden, -math.inf)
            out[at:at + n, head] = torch.softmax(s, dim=-1) @ v[:, of]
        at += n
    return out
