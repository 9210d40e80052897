"""``verify_drafts`` at the ends of its ranges, against its definition in 64 bits."""

from __future__ import annotations

import math

import pytest
import torch

from .test_gpu_verify import BF16, F16, F32, check, inputs

pytestmark = pytest.mark.gpu
MOST = torch.finfo(F32).max


def below(temps):
    """Temperatures as the definition has them: past the largest float, that."""
    return [min(t, MOST) for t in temps]


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("vocab", [37, 4099, 16384, 50021])
@pytest.mark.parametrize("probs", [None, F32])
def test_a_temperature_without_end(dtype, vocab, probs, monkeypatch):
    """Every token as likely as the others, but for those at -inf."""
    from . import test_gpu_verify as t
    lens = [3, 2, 1, 4]
    logits, tokens, numbers, q = inputs(lens, vocab, dtype, seed=vocab, probs=probs, near=0.05)
    logits[:, 5:9] = -math.inf
    logits[:, -2:] = -math.inf
    tokens[1] = 6                    # (a draft that cannot be)
    oracle = t.verify64
    monkeypatch.setattr(t, "verify64",
                        lambda *a: oracle(*a[:5], below(a[5]) if isinstance(a[5], list) else min(a[5], MOST)))
    check(lens, logits, tokens, numbers, q, temps=[math.inf, 1.0, math.inf, math.inf])
    check(lens, logits, tokens, numbers, q, temps=[0.5, math.inf, 0.0, MOST])
    check(lens, logits, tokens, numbers, q, temps=MOST)
    check(lens, logits, tokens, numbers, q, temps=1e39)


@pytest.mark.parametrize("probs", [None, F32])
def test_temperatures_next_to_the_floats_ends(probs):
    """Logits so close together, or so far apart, that log2(e) / temperature, or the
    difference itself, leaves 32 bits."""
    lens = [2] * 24
    logits, tokens, numbers, q = inputs(lens, 700, F32, seed=3, probs=probs)
    g = torch.Generator().manual_seed(9)
    for scale, temp in ((2.0 ** -102, 1e-38), (2.0 ** -120, 2.0 ** -120), (1.4e38, 1e38),
                        (8e37, 2.0 ** 126)):
        near = (torch.randn((48, 700), generator=g).clamp(-2.3, 2.3) * scale).float()
        assert torch.isfinite(near).all()
        check(lens, near, tokens, numbers, q, temp)


def test_a_row_of_nothing_but_minus_infinity_at_temperature_zero():
    """It has no distribution: no draft stands, not that of its greedy id either."""
    lens = [3, 2]
    logits, tokens, numbers, q = inputs(lens, 600, F32, seed=4)
    logits[0] = -math.inf
    logits[3] = -math.inf
    tokens[1] = tokens[4] = 0
    for probs in (q, None):
        count = check(lens, logits, tokens, numbers, probs, [0.0, 0.0])
        assert count.tolist() == [0, 0]
        check(lens, logits, tokens, numbers, probs, [1.0, 0.0])


# Past 262144 tokens a thread takes several cells of eight, past 16777216 more than a
# wave's lanes can share out one each.
@pytest.mark.parametrize("vocab", [262144, 262145, 262152, 524289, 786433])
@pytest.mark.parametrize("probs", [None, F32])
def test_vocabularies_of_several_cells_a_thread(vocab, probs):
    print(f"cells {vocab} {probs}", flush=True)
    lens = [3, 1, 2]
    for dtype, seed in ((BF16, vocab), (F32, vocab + 1)):
        logits, tokens, numbers, q = inputs(lens, vocab, dtype, seed=seed, spread=3.0, probs=probs)
        check(lens, logits, tokens, numbers, q)
        for u in (0.0, 0.5, 1.0 - 2.0 ** -24):
            numbers[:] = u           # (at 0 the first weight of all: no sum decides)
            check(lens, logits, tokens, numbers, q, [0.8, 1.0, 1.3], exact=u == 0.0)


@pytest.mark.parametrize("vocab", [262145, 600000])
@pytest.mark.parametrize("where", ["first", "last of a unit", "second cell", "last"])
def test_weight_in_one_cell_alone(vocab, where):
    """All the weight lies in a few tokens: of a unit's last cell, of the row's last,
    of a thread's second."""
    per = -(-vocab // (64 * 4096))
    at = {"first": 0, "last of a unit": 3 * 4096 * per - 8, "second cell": 8,
          "last": vocab - 3}[where]
    lens = [2, 1]
    g = torch.Generator().manual_seed(at + vocab)
    logits = torch.full((3, vocab), -math.inf)
    n = min(8, vocab - at)
    logits[:, at:at + n] = torch.randn((3, n), generator=g)
    tokens = torch.tensor([0, at + 1, 0])
    q = torch.zeros((1, vocab))
    q[0, at + 1] = 1.0
    for u in (0.0, 0.2, 0.6, 1.0 - 2.0 ** -24):
        for falls in (0.0, 1.0 - 2.0 ** -24):
            numbers = torch.tensor([falls, u, u])
            check(lens, logits, tokens, numbers, q, exact=u == 0.0)
            check(lens, logits, tokens, numbers, None, exact=u == 0.0)


@pytest.mark.parametrize("seed", range(3))
def test_a_vocabulary_whose_threads_hold_more_cells_than_a_wave_has_lanes(seed):
    vocab = 64 * 4096 * 65 + 11      # (66 cells a thread)
    g = torch.Generator().manual_seed(seed)
    logits = (torch.randn((2, vocab), generator=g) * 4.0).to(F16)
    tokens = torch.tensor([0, int(torch.randint(0, vocab, (1,), generator=g))])
    q = torch.softmax(logits[:1].float() + 0.3 * torch.randn((1, vocab), generator=g), -1)
    numbers = torch.rand(2, generator=g)
    check([2], logits, tokens, numbers, q)
    check([1, 1], logits, tokens, numbers)
    numbers[0] = 1.0 - 2.0 ** -24
    check([2], logits, tokens, numbers, None, 0.9)
