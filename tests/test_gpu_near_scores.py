"""
The choice of pages whose scores run in 32 bits first: every kernel it is made
of (query heads a KV head, lists of each size the choice is compiled for): the
chosen pages are those of the 64-bit scores.
"""

from __future__ import annotations

import pytest
import torch

from .test_gpu_selection import DEV, Cache

pytestmark = pytest.mark.gpu

NEAR_LEAST = 16 << 20      # elements (sequences x KV heads x longest list x head_dim)
SELECT_MAX = 16384         # pages of the longest list


def near_cache(n_heads, n_kv, d, dtype, max_pages, budget=30):
    """A few long lists, the longest of max_pages, and as many short ones as it
    takes for the 32-bit pass, whose rule is on the longest list and the count."""
    n = -(-NEAR_LEAST // (n_kv * max_pages * d))
    lens = [max_pages * 16 - 3, max_pages * 11, max_pages * 7 + 5]
    lens += [1 + 29 * i % (budget * 16 + 40) for i in range(n - 3)]
    c = Cache(lens, n_heads, n_kv, d, dtype)
    longest = max(s.num_blocks for s in c.seqs)
    assert longest == max_pages <= SELECT_MAX
    assert len(lens) * n_kv * longest * d >= NEAR_LEAST and d in (64, 128)
    return c


@pytest.mark.parametrize("n_heads, n_kv, d", [
    (64, 4, 64), (64, 4, 128), (32, 4, 64), (16, 2, 128), (16, 4, 64), (8, 4, 128), (8, 8, 128)])
@pytest.mark.parametrize("max_pages", [500, 1024, 1025, 4096, 4097])
@pytest.mark.parametrize("dtype, close", [
    (torch.float16, False), (torch.bfloat16, False), (torch.bfloat16, True)])
def test_every_kernel_of_the_choice(n_heads, n_kv, d, max_pages, dtype, close):
    """Random pages, and pages that only 64 bits tell apart."""
    print(f"near {n_heads}/{n_kv}/{d} {max_pages} {dtype} close={close}", flush=True)
    c = near_cache(n_heads, n_kv, d, dtype, max_pages)
    q = c.q()
    if close:
        kp = c.bk.k_pool[0]
        page = c.rand((16, n_kv, d)).abs() + 1
        page[..., 5] = 2.0 ** -9
        step = torch.randperm(kp.shape[0], generator=c.g, device=DEV) % 50
        kp.copy_(page)
        kp[..., 5] *= (1 + step * torch.finfo(dtype).eps)[:, None, None].to(dtype)
        c.bk.refresh_page_bounds()
        q = q.abs()
    out, chosen = c.bk.attend_selected(q, 0, 0.125, c.meta, 30, return_pages=True)
    c.bk.check_device_errors()
    c.check(q, 30, out, chosen)
