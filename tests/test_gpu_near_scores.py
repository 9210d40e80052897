"""
The choice of pages whose scores run in 32 bits first: every kernel it is made
of (query heads a KV head, lists of each size the choice is compiled for), and
values that 32-bit sums lose: the chosen pages are those of the 64-bit scores.
"""

from __future__ import annotations

import pytest
import torch

from ._ops64 import chosen64
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


def assert_chosen(c, q, chosen, budget):
    lo, hi = c.bk.key_bounds[0]
    for i, s in enumerate(c.seqs[:3]):
        ids = torch.tensor(s.block_ids, device=DEV)
        want = chosen64(q[i], lo[ids], hi[ids], len(ids), budget)
        assert [w[:budget] for w in chosen[i].tolist()] == want, f"seq {i}"


@pytest.mark.parametrize("n_heads, n_kv, d", [(64, 4, 64), (16, 4, 128), (4, 4, 64)])
@pytest.mark.parametrize("first", [1, -1])
@pytest.mark.parametrize("lanes", [1, 2])
@pytest.mark.parametrize("size", [2e18, 4e18])
def test_sums_that_overflow_on_the_way(n_heads, n_kv, d, first, lanes, size):
    """bf16 products of 2e38 and 5e38 (the largest float is 3.4e38) of both signs:
    a few pages whose 32-bit sum overflows on its way to a score that does not,
    the lowest or the highest of all, in one lane's elements and from one lane's
    to another's; a second query head's scores are small. (The attention's own
    scores overflow with them: its output is not looked at.)"""
    print(f"near overflow {n_heads}/{n_kv}/{d} {first} {lanes} {size}", flush=True)
    c = near_cache(n_heads, n_kv, d, torch.bfloat16, 600)
    kp, groups = c.bk.k_pool[0], n_heads // n_kv
    a, b = [0, 1], [2, 3] if lanes == 1 else [8, 9]
    q = torch.zeros((len(c.seqs), n_heads, d), dtype=torch.bfloat16, device=DEV)
    q[..., a], q[..., b] = first * 1e20, -first * 1e20
    if groups > 1:
        q[:, 1::groups] = c.q()[:, 1::groups]
    kp.zero_()
    rand = torch.rand((kp.shape[0], 1, n_kv), generator=c.g, device=DEV)
    for j in (*a, *b):
        kp[..., j] = (1e17 * rand.roll(j, 0)).to(kp.dtype)
    for s in c.seqs[:3]:
        some = torch.tensor(s.block_ids[3:400:40], device=DEV)
        big = size * (1 + torch.rand((len(some), 1, 1), generator=c.g, device=DEV) / 4)
        for j in a:
            kp[some, ..., j] = big.to(kp.dtype)
        for j in b:        # the score: 2e20 first (big - this)
            kp[some, ..., j] = (big * 1.2).to(kp.dtype)
    c.bk.refresh_page_bounds()
    _, chosen = c.bk.attend_selected(q, 0, 1e-30, c.meta, 30, return_pages=True)
    c.bk.check_device_errors()
    assert_chosen(c, q, chosen, 30)


@pytest.mark.parametrize("n_heads, n_kv, d", [(64, 4, 64), (16, 4, 128), (4, 4, 64)])
def test_queries_below_the_smallest_normal(n_heads, n_kv, d):
    """bf16: one query element of 1e-36, the others subnormal, keys of up to 1e30:
    what the subnormal elements add decides, far above the sums' roundings."""
    print(f"near subnormal {n_heads}/{n_kv}/{d}", flush=True)
    c = near_cache(n_heads, n_kv, d, torch.bfloat16, 600)
    kp = c.bk.k_pool[0]
    kp.copy_((kp.float() * 1e30).to(kp.dtype))
    q = (torch.rand((len(c.seqs), n_heads, d), generator=c.g, device=DEV) * 1e-38).bfloat16()
    q[..., 0] = 1e-36
    c.bk.refresh_page_bounds()
    _, chosen = c.bk.attend_selected(q, 0, 0.125, c.meta, 30, return_pages=True)
    c.bk.check_device_errors()
    assert_chosen(c, q, chosen, 30)
