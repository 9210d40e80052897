"""
Attention in 64 bits over lists of keys and values, with a bound on what the
kernels' arithmetic may be off by, for the tests of the decode operators.
"""

from __future__ import annotations

import torch


def attend64(q, k, v, scale, dtype):
    """
    One token's attention: q (Hq, D), k and v (N, Hkv, D) or per-head lists of
    (N, D). Returns (out, bound), (Hq, D) in 64 bits.

    The bound, with u = eps / 2 of the pool dtype (one rounding to it), per
    output element, A = sum_j p_j |v_j| with the p's sum 1:
      u |out|                         the output's rounding
      u A                             each probability's rounding
      (2 delta + 2 (N + 64) 2^-24) A  fp32: delta bounds a score's error (D
                                      products and their sum, the scale and
                                      log2 e), which moves a probability and the
                                      sum by its factor; sums of N terms over
                                      p and p v, plus the merge of up to 64 parts
      N 2^-25 max|v|                  fp16 only: probabilities below 2^-14 round
                                      by 2^-25; the row's largest is at least 1
    """
    heads = [k[:, h] for h in range(k.shape[1])] if torch.is_tensor(k) else k
    vals = [v[:, h] for h in range(v.shape[1])] if torch.is_tensor(v) else v
    groups = q.shape[0] // len(heads)
    outs, bounds = [], []
    u = torch.finfo(dtype).eps / 2
    for h, (kk, vv) in enumerate(zip(heads, vals)):
        qq, kk, vv = q[h * groups:(h + 1) * groups].double(), kk.double(), vv.double()
        n, d = kk.shape
        p = torch.softmax(qq @ kk.t().contiguous() * scale, dim=-1)
        o, a = p @ vv, p @ vv.abs()
        delta = (d + 4) * 2.0 ** -24 * scale * (qq.abs() @ kk.abs().t().contiguous()).amax(1)
        b = u * o.abs() + (u + 2 * delta[:, None] + 2 * (n + 64) * 2.0 ** -24) * a
        if dtype == torch.float16:
            b = b + n * 2.0 ** -25 * vv.abs().amax(0)
        outs.append(o)
        bounds.append(b * 1.001 + torch.finfo(dtype).tiny)
    return torch.cat(outs), torch.cat(bounds)


def assert_within(got, want, bound, label=""):
    assert torch.isfinite(got).all(), f"{label}: non-finite output"
    over = (got.double() - want).abs() - bound
    assert float(over.max()) <= 0, (
        f"{label}: off by {float(over.max()):.3g} past a bound of "
        f"{float(bound.reshape(-1)[over.argmax()]):.3g}")


def chosen64(q, lo, hi, n_pages, pages):
    """The choice by its definition: per KV head the ascending page indices. q
    (Hq, D); lo, hi (n_pages, Hkv, D) bounds of the sequence's pages."""
    hkv = lo.shape[1]
    groups = q.shape[0] // hkv
    if n_pages <= pages:
        return [list(range(n_pages))] * hkv
    out = []
    for h in range(hkv):
        qq = q[h * groups:(h + 1) * groups, None, :].double()
        b = torch.where(qq < 0, lo[None, :-1, h].double(), hi[None, :-1, h].double())
        s = (qq * b).sum(-1)
        s = torch.where(s.isnan().any(0), float("nan"), s.amax(0)).tolist()
        rank = sorted(range(n_pages - 1),
                      key=lambda p: (0 if s[p] != s[p] else 1, -s[p] if s[p] == s[p] else 0, p))
        out.append(sorted(rank[:pages - 1]) + [n_pages - 1])
    return out
