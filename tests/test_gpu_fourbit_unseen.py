"""
Attention over the 4-bit cache where keys differ in scale, or hold what is not
finite: a token's output depends on the keys that it sees alone, and is NaN where
one of them is.
"""

from __future__ import annotations

import math

import pytest
import torch

from ._fourbit import attend64
from ._ops64 import assert_within
from ._util import make_meta
from .test_gpu_fourbit import BF16, DEV, F16, Cache, rows

pytestmark = pytest.mark.gpu


def fill(c, k, v):
    """The rows of sequence 0, all at once."""
    n = k.shape[0]
    if not c.seqs[0].num_tokens:
        c.seqs[0].append(n)
    c.k, c.v = [k], [v]
    c.bk.append_kv(0, k.to(DEV), v.to(DEV), make_meta(c.seqs, [n], c.ps, device=DEV))


def attend_last(c, new, scale, q=None):
    """(queries, outputs) of the last ``new`` tokens."""
    q = c.q([new]) if q is None else q
    out = c.bk.attend(q.to(DEV), 0, scale, make_meta(c.seqs, [new], c.ps, device=DEV))
    return q, out.cpu()


# (query heads of 2 KV heads, new tokens, compute units): rows in four, two and one
# classes, wide rows twice, tall ones
FORMS = [(4, 2, None), (8, 2, None), (8, 4, None), (8, 6, None), (16, 8, None), (8, 40, 1)]


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("hq,new,units", FORMS)
@pytest.mark.parametrize("history", [0, 100, 300])
@pytest.mark.parametrize("bad", [math.nan, math.inf, 60000.0])
@pytest.mark.parametrize("spread", [0.5, 0.02])
def test_a_later_value_leaves_earlier_tokens_as_they_are(d, hq, new, units, history, bad, spread):
    """The last token's V is not finite, or a thousand times the others: the tokens
    before it stay within the bound of a call without it."""
    print(f"later {d} {hq} {new} {history} {bad} {spread}", flush=True)
    n = history + new
    c = Cache([0], F16, 2, hq, d, room=400, compute_units=units)
    k, v = rows((n, 2, d), F16, 1), rows((n, 2, d), F16, 2).mul(spread)
    v[-1, :, 3] = bad                # (of the first group)
    fill(c, k, v)
    q, out = attend_last(c, new, d ** -0.5)
    want, bound = attend64(q[:-1], k[:-1], v[:-1], d ** -0.5, F16)
    assert_within(out[:-1], want, bound, "earlier tokens")
    if math.isfinite(bad):
        want, bound = attend64(q[-1:], k, v, d ** -0.5, F16)
        assert_within(out[-1:], want, bound, "the token itself")
        return
    assert out[-1, :, :64].isnan().all()
    if d == 128:                     # the other group is finite
        v[-1, :, :64] = 0
        want, bound = attend64(q[-1:], k, v, d ** -0.5, F16)
        assert_within(out[-1:, :, 64:], want[..., 64:], bound[..., 64:], "the other group")


@pytest.mark.parametrize("hq,new", [f[:2] for f in FORMS])
def test_small_steps_behind_tiles_without_one(hq, new):
    """V of the first tiles is nothing; the first steps that come are the least
    there are. (One piece: its first wave takes tiles 0 and 4.)"""
    n = 256 + 8
    c = Cache([0], BF16, 2, hq, 64, room=400, compute_units=1)
    k = rows((n, 2, 64), BF16, 1)
    v = torch.zeros((n, 2, 64), dtype=BF16)
    g = torch.Generator().manual_seed(3)
    v[256:] = (torch.randint(0, 16, (8, 2, 64), generator=g).float() * 2.0 ** -24).to(BF16)
    v[256:, :, 0], v[256:, :, 1] = 0.0, 15 * 2.0 ** -24
    fill(c, k, v)
    q, out = attend_last(c, new, 0.125)
    want, bound = attend64(q, k, v, 0.125, BF16)
    assert_within(out, want, bound)


@pytest.mark.parametrize("d", [64, 128, 80])
@pytest.mark.parametrize("n", [20, 300])
@pytest.mark.parametrize("hq,new,units", FORMS)
def test_a_seen_nan_of_hardly_any_weight(d, n, hq, new, units):
    """A weight of e^-300 is not nothing: a token that sees the key gets NaN."""
    n += new
    c = Cache([0], F16, 2, hq, d, room=400, compute_units=units)
    k, v = rows((n, 2, d), F16, 1, centre=0.0), rows((n, 2, d), F16, 2)
    q = torch.full((new, hq, d), 4.0, dtype=F16)
    k[3] = -300.0 / (4 * d * 0.125)
    v[3] = math.nan
    fill(c, k, v)
    _, out = attend_last(c, new, 0.125, q)
    assert out.isnan().all()


@pytest.mark.parametrize("d,hq", [(64, 4), (64, 8), (128, 4)])
@pytest.mark.parametrize("units", [2, 4, 8])
def test_pieces_whose_scores_are_all_nan(d, hq, units):
    """K of all of one piece of a cut sequence is NaN: it has no finite score, and the
    output is NaN."""
    n = 3000
    c = Cache([0], F16, 2, hq, d, room=3100, compute_units=units)
    k, v = rows((n, 2, d), F16, 1), rows((n, 2, d), F16, 2)
    fill(c, k, v)
    _, out = attend_last(c, 1, d ** -0.5)
    assert torch.isfinite(out).all()
    pieces = c.bk._planned.buffers[5].view(-1, 28)[:, 6:8].tolist()
    assert len(pieces) == units and sum(tiles for _, tiles in pieces) == 47
    for first, tiles in pieces:
        spoilt = k.clone()
        spoilt[64 * first:64 * (first + tiles)] = math.nan
        fill(c, spoilt, v)
        _, out = attend_last(c, 1, d ** -0.5)
        assert out.isnan().all(), (first, tiles)


def test_owners_that_the_lengths_contradict():
    """A token said to be a sequence's, but behind its end: it sees the keys that the
    sequence has."""
    c = Cache([40, 9], F16, 2, 4, 80)
    counts = [2, 5]
    meta = c.append(counts)
    q = c.q(counts)
    meta.batch_indices[:] = 0
    out = c.bk.attend(q.to(DEV), 0, 0.1, meta).cpu()
    for t in range(7):
        n = min(41 + t, 42)
        want, bound = attend64(q[t:t + 1], c.k[0][:n], c.v[0][:n], 0.1, F16)
        assert_within(out[t:t + 1], want, bound, f"token {t}")


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("hq,new,units", FORMS)
@pytest.mark.parametrize("power", [16, 20, 23])
def test_scores_next_to_the_largest(d, hq, new, units, power):
    """Scores to 2^25.7, so far apart that the largest takes all the weight: that key's V
    comes out."""
    n = 70 + new
    c = Cache([0], BF16, 2, hq, d, room=400, compute_units=units)
    k, v = rows((n, 2, d), BF16, 1), rows((n, 2, d), BF16, 2)
    k *= 0.25
    k[33] = 8.0                      # (a constant row is held exactly)
    fill(c, k, v)
    q = torch.full((new, hq, d), 2.0 ** (power - 4), dtype=BF16)
    q[..., 0] = 2.0 ** power
    _, out = attend_last(c, new, d ** -0.5, q)
    want, _ = attend64(q, k, v, d ** -0.5, BF16)
    _, bound = attend64(q * 0, k[33:34].expand(new, 2, d), v[33:34].expand(new, 2, d), 1.0, BF16)
    assert_within(out, want, bound)
