"""Random batches over the 4-bit cache whose values differ in scale: each token within
the bound of a call with the keys that it sees and no others."""

from __future__ import annotations

import random

import pytest
import torch

from ._fourbit import attend64
from ._util import make_meta
from .test_gpu_fourbit import BF16, DEV, F16, Cache

pytestmark = pytest.mark.gpu
GEOMS = [(2, 8, 64), (2, 8, 128), (1, 4, 64), (1, 8, 128), (1, 16, 64), (1, 32, 128), (3, 3, 64),
         (1, 6, 64), (2, 48, 64)]


def scaled(v, how, tot, g, rng):
    """V of (T, n_kv, d), its rows by powers of two."""
    n = v.shape[0]
    if how == "any":
        return v * torch.exp2(torch.rand((n, 1, 1), generator=g) * 16 - 8)
    if how == "rare":
        return v * (torch.rand((n, 1, 1), generator=g) < 0.05)
    if how == "rising":
        return v * torch.exp2(torch.linspace(-10, 6, n))[:, None, None]
    at, v = 0, v.clone()
    for t in tot:                    # the last tokens alone
        v[at + t - rng.randint(1, min(t, 4)):at + t] *= 2.0 ** rng.randint(4, 14)
        at += t
    return v


@pytest.mark.parametrize("how", ["any", "rare", "rising", "late"])
@pytest.mark.parametrize("seed", range(12))
def test_random_batches(how, seed):
    rng, g = random.Random(seed), torch.Generator().manual_seed(seed)
    n_kv, hq, d = rng.choice(GEOMS)
    dtype, units, ps = rng.choice([F16, BF16]), rng.choice([None, None, 1, 4, 16]), rng.choice([16, 64])
    counts = [rng.choice([1, 2, 3, 5, 8, 17, 40]) for _ in range(rng.randint(1, 3))]
    tot = [n + rng.choice([0, 10, 63, 64, 300, 1000]) for n in counts]
    print(f"random {how} {n_kv} {hq} {d} {dtype} {units} {ps} {counts} {tot}", flush=True)
    c = Cache([0] * len(tot), dtype, n_kv, hq, d, ps, room=1100, compute_units=units)
    for s, n in zip(c.seqs, tot):
        s.append(n)
    k = (torch.randn((sum(tot), n_kv, d), generator=g) * 0.5).to(dtype)
    v = scaled(torch.randn((sum(tot), n_kv, d), generator=g) * 0.5, how, tot, g, rng)
    v = v.clamp(-60000, 60000).to(dtype)
    c.bk.append_kv(0, k.to(DEV), v.to(DEV), make_meta(c.seqs, tot, ps, device=DEV))
    q = (torch.randn((sum(counts), hq, d), generator=g) * rng.choice([0.3, 1, 4])).to(dtype)
    out = c.bk.attend(q.to(DEV), 0, d ** -0.5, make_meta(c.seqs, counts, ps, device=DEV)).cpu()
    at = row = 0
    for n, new in zip(tot, counts):
        for j in range(new):
            sees = slice(at, at + n - new + j + 1)
            want, bound = attend64(q[row:row + 1], k[sees], v[sees], d ** -0.5, dtype)
            off = (out[row:row + 1].double() - want).abs() - bound
            assert float(off.max()) <= 0, f"token {j} of {new}: {float(off.max())}"
            row += 1
        at += n
