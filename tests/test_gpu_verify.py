"""
``verify_drafts`` on the GPU against its definition in 64 bits: whole numbers,
compared exactly. Inputs whose decisions lie closer than 1e-11 to a border (where
64-bit sums of another order may differ) do not occur: the oracle's margin says so.
"""

from __future__ import annotations

import math
import random

import pytest
import torch

from llm_serving_layer_amd import (BlockAllocator, FourBitBackend, ScheduledSeq, SequenceBlocks,
                                   build_batch_meta, build_token_tensor)
from llm_serving_layer_amd.sampling import greedy, verify_drafts

from ._util import meta_to_device
from ._verify import verify64

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


def meta_of(lens, device=DEV):
    alloc = BlockAllocator(sum(-(-n // 16) for n in lens), 16)
    seqs = []
    for i, n in enumerate(lens):
        s = SequenceBlocks(alloc, seq_id=i)
        s.append(n)
        seqs.append(ScheduledSeq(s, [0] * n))
    return build_batch_meta(seqs, device, 16)


def inputs(lens, vocab, dtype, seed=0, spread=2.0, probs=F32, near=0.7):
    """(logits, tokens, numbers, draft probabilities): drafts from a model near
    the target."""
    g = torch.Generator().manual_seed(seed)
    rows = sum(lens)
    base = torch.randn((rows, vocab), generator=g) * spread
    tokens = torch.randint(0, vocab, (rows,), generator=g)
    logits = base.to(dtype)
    q, at, out = None, 0, []
    for n in lens:
        for j in range(n - 1):
            d = torch.softmax(base[at + j] + near * torch.randn(vocab, generator=g), -1)
            tokens[at + j + 1] = (int(torch.multinomial(d, 1, generator=g)) if probs
                                  else int(d.argmax()))
            out.append(d)
        at += n
    if probs and out:
        q = torch.stack(out).to(probs)
    return logits, tokens, torch.rand(rows, generator=g), q


def check(lens, logits, tokens, numbers, q=None, temps=1.0, device_logits=None, exact=False):
    meta = meta_of(lens)
    temp = torch.tensor(temps, dtype=F32, device=DEV) if isinstance(temps, list) else temps
    ids, accepted = verify_drafts(
        logits.to(DEV) if device_logits is None else device_logits, tokens.to(DEV), meta,
        numbers.to(DEV), draft_probs=None if q is None else q.to(DEV), temperature=temp)
    t64 = ([float(torch.tensor(t, dtype=F32)) for t in temps] if isinstance(temps, list)
           else float(torch.tensor(temps, dtype=F32)))
    want, count, margin = verify64(logits, tokens, lens, numbers, q, t64)
    assert exact or margin > 1e-11, "the inputs decide nothing clearly"
    assert ids.dtype == accepted.dtype == torch.int64
    assert torch.equal(accepted.cpu(), count)
    assert torch.equal(ids.cpu(), want)
    return count


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("probs", [None, F16, BF16, F32])
@pytest.mark.parametrize("vocab", [1, 2, 37, 1000, 4099, 50021])
def test_against_the_definition(dtype, probs, vocab):
    print(f"verify {dtype} {probs} {vocab}", flush=True)
    lens = [1, 4, 2, 6, 1, 3, 5]
    x = inputs(lens, vocab, dtype, seed=vocab, probs=probs)
    check(lens, *x)
    check(lens, *x, temps=[0.7, 0.0, 1.0, 0.3, 2.0, 1.5, -1.0])


@pytest.mark.parametrize("probs", [None, F32])
@pytest.mark.parametrize("lens", [[1], [9], [1] * 40, [2] * 300, [300, 1, 280]])
def test_batch_shapes(probs, lens):
    check(lens, *inputs(lens, 700, F16, seed=len(lens), probs=probs, near=0.05))


def test_a_real_vocabulary():
    lens = [5, 3, 1, 9]
    count = check(lens, *inputs(lens, 128256, BF16, seed=3, spread=3.0))
    check(lens, *inputs(lens, 151939, F16, seed=5, spread=3.0, probs=None))
    assert count.sum() > 0


@pytest.mark.parametrize("probs", [None, F32])
def test_flat_rows(probs):
    """Every token as likely as the others, nearly: all borders close together."""
    lens = [3] * 20
    check(lens, *inputs(lens, 30011, F32, seed=8, spread=1e-3, probs=probs, near=1e-3))


@pytest.mark.parametrize("seed", range(6))
def test_acceptance_next_to_the_border(seed):
    """Numbers one step of 32 bits on either side of p / q: the sum in 32 bits
    cannot tell, the one in 64 does."""
    lens = [2] * 64
    logits, tokens, numbers, q = inputs(lens, 997, F16, seed=seed)
    for i in range(64):
        x = int(tokens[2 * i + 1])
        p = torch.softmax(logits[2 * i].double(), -1)[x] / q[i, x].double()
        u = p.to(F32)
        if float(u) < 1:
            step = torch.tensor(math.inf if seed % 2 else -math.inf)
            numbers[2 * i] = torch.nextafter(u, step) if seed % 3 else u
    check(lens, logits, tokens, numbers, q)


@pytest.mark.parametrize("u", [0.0, 1.0 - 2.0 ** -24])
@pytest.mark.parametrize("probs", [None, F32])
def test_the_least_and_the_largest_number(u, probs):
    lens = [1, 2, 4]
    logits, tokens, numbers, q = inputs(lens, 5003, F32, seed=2, probs=probs)
    logits[:, :100] = -math.inf
    logits[:, -7:] = -math.inf
    numbers[:] = u
    check(lens, logits, tokens, numbers, q)


def test_rows_without_a_distribution():
    lens = [2] * 6 + [1] * 3
    logits, tokens, numbers, q = inputs(lens, 600, F32, seed=4)
    logits[0, 77] = math.nan
    logits[2, 5] = math.inf
    logits[4] = -math.inf
    logits[6, 300:] = math.nan
    logits[8, 9] = logits[8, 8] = math.inf
    logits[12, 599] = math.nan
    logits[13] = -math.inf
    tokens[1] = 77
    tokens[3] = 5
    for temps in (1.0, [0.0] * 9):
        check(lens, logits, tokens, numbers, q, temps)
        check(lens, logits, tokens, numbers, None, temps)


def test_drafts_outside_the_vocabulary_fall():
    lens = [3, 3, 2]
    logits, tokens, numbers, q = inputs(lens, 300, F16, seed=6, near=0.01)
    tokens[1], tokens[5], tokens[7] = -1, 300, 2**40
    for t in (1.0, [0.0, 0.5, 1.0]):
        check(lens, logits, tokens, numbers, q, t)
        check(lens, logits, tokens, numbers, None, t)


def test_a_draft_that_is_all_there_is():
    """Nothing is left beside the draft, or beside q: drawn from p. (Ones and zeros
    alone, which no sum rounds.)"""
    lens = [2, 2]
    logits = torch.full((4, 50), -math.inf)
    logits[:, 7] = 1.0
    tokens = torch.tensor([0, 7, 0, 7])
    numbers = torch.tensor([1.0, 0.5, 1.0, 0.5])   # (1 is past the last: it falls)
    check(lens, logits, tokens, numbers, exact=True)
    check(lens, logits, tokens, numbers, torch.full((2, 50), 1.0), exact=True)


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("probs", [None, F32])
@pytest.mark.parametrize("t", [1e-30, 1e-3, 1e4])
def test_extreme_temperatures_and_logits(dtype, probs, t):
    lens = [3, 2, 1]
    logits, tokens, numbers, q = inputs(lens, 811, dtype, seed=11, probs=probs)
    check(lens, logits, tokens, numbers, q, t)
    check(lens, logits * 1000, tokens, numbers, q, t)
    if dtype == F32:
        check(lens, logits * 1e37, tokens, numbers, q, t)


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
def test_ties_go_to_the_first(dtype):
    lens = [2, 2, 1]
    logits = torch.zeros((5, 9000), dtype=dtype)
    for r, at in enumerate([(4000, 17), (8999, 3), (16, 15), (0, 8999), (8191, 8192)]):
        for i in at:
            logits[r, i] = 5.0
    tokens = torch.tensor([0, 17, 0, 16, 0])
    got = check(lens, logits, tokens, torch.rand(5), temps=0.0)
    assert got.tolist() == [1, 0, 0]


def test_rows_of_other_strides():
    lens = [3, 1, 4]
    logits, tokens, numbers, q = inputs(lens, 517, F16, seed=12)
    for pad, shift in ((3, 0), (64, 5), (1, 1)):
        wide = torch.full((8, 517 + pad + shift), 60000.0, dtype=F16, device=DEV)
        view = wide[:, shift:shift + 517]
        view.copy_(logits)
        check(lens, logits, tokens, numbers, q, device_logits=view)
    for view in (logits.t().contiguous().t().to(DEV), logits.to(DEV)):
        check(lens, logits, tokens, numbers, q, device_logits=view)
    one = logits[:1].expand(8, 517)
    check(lens, one, tokens, numbers, None, device_logits=logits[:1].to(DEV).expand(8, 517))


def test_without_host_arrays_and_in_a_graph():
    lens = [4, 1, 3]
    logits, tokens, numbers, q = (x.to(DEV) for x in inputs(lens, 3001, F16, seed=13))
    meta = meta_of(lens)
    bare = meta_to_device(meta_of(lens, "cpu"), DEV, mirror=False)
    want = verify_drafts(logits, tokens, meta, numbers, draft_probs=q)
    got = verify_drafts(logits, tokens, bare, numbers, draft_probs=q)
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = verify_drafts(logits, tokens, meta, numbers, draft_probs=q)
        two = verify_drafts(logits, tokens, meta, numbers, temperature=0.5)
    with pytest.raises(RuntimeError, match="captured"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            torch.zeros(1, device=DEV)
            verify_drafts(logits, tokens, bare, numbers)
    torch.cuda.synchronize()
    for i in range(5):
        new = inputs(lens, 3001, F16, seed=20 + i)
        for a, b in zip((logits, tokens, numbers, q), new):
            a.copy_(b)
        graph.replay()
        eager = verify_drafts(logits, tokens, meta, numbers, draft_probs=q)
        other = verify_drafts(logits, tokens, meta, numbers, temperature=0.5)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out + two, eager + other))


def test_lengths_that_do_not_sum_up_are_refused():
    lens = [4, 1, 3]
    logits, tokens, numbers, _ = (x.to(DEV) for x in inputs(lens, 301, F16, seed=13))
    bare = meta_to_device(meta_of(lens, "cpu"), DEV, mirror=False)
    bare.cu_query_lens[2] = 7
    with pytest.raises(ValueError, match="sums"):
        verify_drafts(logits, tokens, bare, numbers)


def test_calls_on_two_streams_at_once():
    lens = [3] * 50
    a = [x.to(DEV) for x in inputs(lens, 20011, F16, seed=30)]
    b = [x.to(DEV) for x in inputs(lens, 20011, F16, seed=31)]
    meta = meta_of(lens)
    want = [verify_drafts(*x[:2], meta, x[2], draft_probs=x[3]) for x in (a, b)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for _ in range(5):
        for x, s in zip((a, b), streams):
            with torch.cuda.stream(s):
                got.append(verify_drafts(*x[:2], meta, x[2], draft_probs=x[3]))
    torch.cuda.synchronize()
    for i, g in enumerate(got):
        assert all(torch.equal(p, q) for p, q in zip(g, want[i % 2]))


def test_drafts_are_distributed_as_the_target():
    """Over many numbers the first token's frequencies are the target's, whatever
    the drafting distribution: 20 000 draws, 5 standard deviations."""
    vocab, n = 12, 20000
    g = torch.Generator().manual_seed(1)
    row, drow = torch.randn(vocab, generator=g), torch.randn(vocab, generator=g)
    q = torch.softmax(drow, -1)
    tokens = torch.zeros(2 * n, dtype=torch.int64)
    tokens[1::2] = torch.multinomial(q, n, replacement=True, generator=g)
    ids, _ = verify_drafts(row.expand(2 * n, vocab).to(DEV), tokens.to(DEV), meta_of([2] * n),
                           torch.rand(2 * n, generator=g).to(DEV),
                           draft_probs=q.expand(n, vocab).to(DEV))
    p = torch.softmax(row.double(), -1)
    seen = torch.bincount(ids[:, 0].cpu(), minlength=vocab).double() / n
    assert ((seen - p).abs() <= 5 * (p * (1 - p) / n).sqrt()).all()


def test_a_speculative_loop_over_the_4_bit_cache():
    """Drafts appended, attended and verified; the rows of those that fell are
    overwritten by the next step. The tokens are those of single greedy steps
    over the same kind of cache."""
    g = torch.Generator().manual_seed(2)
    vocab, n_kv, hq, d, ps = 61, 2, 8, 64, 16
    emb = torch.randn((vocab, (hq + 2 * n_kv) * d), generator=g).half().to(DEV)
    head = torch.randn((hq * d, vocab), generator=g).half().to(DEV)

    class Model:
        def __init__(self):
            self.bk = FourBitBackend(1, 64, ps, n_kv, hq, d, device=DEV)

        def __call__(self, tokens, meta):
            q, k, v = (t.view(len(tokens), h, d) for t, h in
                       zip(emb[tokens].split([hq * d, n_kv * d, n_kv * d], 1), (hq, n_kv, n_kv)))
            self.bk.append_kv(0, k, v, meta)
            o = self.bk.attend(q, 0, d ** -0.5, meta)
            return (o.reshape(len(tokens), -1).float() @ head.float())

    def step(model, seqs, new):
        scheds = [ScheduledSeq(s, list(t)) for s, t in zip(seqs, new)]
        meta = build_batch_meta(scheds, DEV, ps)
        tokens = build_token_tensor(scheds, DEV)
        return tokens, meta, model(tokens, meta)

    prompts = [[3, 1, 4, 1, 5], [9, 2, 6], [5] * 20]
    rng = random.Random(0)

    def begin(model):
        alloc = BlockAllocator(64, ps)
        seqs = [SequenceBlocks(alloc, seq_id=i) for i in range(3)]
        for s, p in zip(seqs, prompts):
            s.append(len(p))
        _, meta, logits = step(model, seqs, prompts)
        return seqs, [[t] for t in greedy(logits[meta.last_token_ix.long()]).tolist()]

    plain, spec = Model(), Model()
    seqs, out = begin(plain)
    for _ in range(24):
        for s in seqs:
            s.append(1)
        _, _, logits = step(plain, seqs, [o[-1:] for o in out])
        for o, t in zip(out, greedy(logits).tolist()):
            o.append(t)
    seqs, got = begin(spec)
    steps = 0
    while min(map(len, got)) < 20:
        new = []
        for o, want in zip(got, out):
            true = want[len(o):len(o) + rng.randint(0, 4)]
            drafts = [t if rng.random() < 0.8 else rng.randrange(vocab) for t in true]
            new.append([o[-1], *drafts])
        old = [s.num_tokens for s in seqs]
        for s, t in zip(seqs, new):
            need = s.num_tokens + len(t)
            if need > s.capacity:
                s.append(len(t))
            else:
                s.num_tokens = need
        tokens, meta, logits = step(spec, seqs, new)
        ids, accepted = verify_drafts(logits, tokens, meta, torch.rand(len(tokens), device=DEV),
                                      temperature=0.0)
        for i, (o, row, a) in enumerate(zip(got, ids.tolist(), accepted.tolist())):
            o.extend(row[:a + 1])
            seqs[i].num_tokens = old[i] + 1 + a
            keep = -(-seqs[i].num_tokens // ps)
            if len(seqs[i].block_ids) > keep:
                seqs[i]._alloc.free(seqs[i].block_ids[keep:])
                seqs[i].block_ids = seqs[i].block_ids[:keep]
        steps += 1
    assert [o[:20] for o in got] == [o[:20] for o in out]
    assert steps < 20
    spec.bk.check_device_errors()
