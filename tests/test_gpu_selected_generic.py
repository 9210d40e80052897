"""
attend_selected where no matrix-core kernel applies: its products run in 32
bits, so only the output is rounded to the pool's type.
"""

from __future__ import annotations

import pytest
import torch

from ._ops64 import assert_within, attend64, chosen64
from .test_gpu_selection import DEV, Cache

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n_heads, n_kv, d, dtype, ps", [
    (9, 3, 80, torch.float16, 16), (4, 2, 7, torch.bfloat16, 16), (8, 2, 64, torch.float16, 8),
    (12, 4, 64, torch.bfloat16, 16), (4, 4, 256, torch.bfloat16, 32)])
@pytest.mark.parametrize("pages", [1, 5, 40])
def test_only_the_output_is_rounded(n_heads, n_kv, d, dtype, ps, pages):
    """The bound: that of the 32-bit arithmetic (each probability's rounding to 32
    bits among it), and half a step of the pool's type of what it gives."""
    print(f"generic {n_heads}/{n_kv}/{d} {dtype} ps={ps} pages={pages}", flush=True)
    c = Cache([1, ps, ps + 1, 23 * ps + 5, 700], n_heads, n_kv, d, dtype, ps=ps)
    q = c.q()
    out, chosen = c.bk.attend_selected(q, 0, 0.125, c.meta, pages, return_pages=True)
    kp, vp = c.bk.k_pool[0], c.bk.v_pool[0]
    info = torch.finfo(dtype)
    for i, s in enumerate(c.seqs):
        ids = torch.tensor(s.block_ids, device=DEV)
        want = chosen64(q[i], kp.amin(1)[ids], kp.amax(1)[ids], len(ids), pages)
        assert [[p for p in w if p >= 0] for w in chosen[i].tolist()] == want
        live = s.num_tokens - (len(ids) - 1) * ps
        keys, values = ([p[ids[w], :, h].flatten(0, 1)[:(len(w) - 1) * ps + live]
                         for h, w in enumerate(want)] for p in (kp, vp))
        o, b = attend64(q[i], keys, values, 0.125, torch.float32)
        assert_within(out[i], o, b + info.eps / 2 * (o.abs() + b) + info.tiny * info.eps / 2,
                      label=f"seq {i}")
