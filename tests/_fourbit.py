"""
The 4-bit cache by its definition, in 64 bits on the CPU, and a bound on what
the attention's arithmetic over it may be off by.
"""

from __future__ import annotations

import math

import torch

MAX = 65504.0


def groups_of(d):
    return d // 64 if d % 64 == 0 else 1


def f16_down(x):
    """The largest float16 not above each x (64 bits, |x| <= 65504)."""
    m, e = torch.frexp(x)
    ulp = torch.ldexp(torch.ones_like(x), torch.clamp(e - 1, min=-14) - 10)
    return torch.floor(x / ulp) * ulp


def quantise64(x):
    """(codes, step, zero) in 64 bits of rows (..., D): codes (..., G, D / G)."""
    y = x.detach().cpu().double()
    y = y.reshape(*y.shape[:-1], groups_of(y.shape[-1]), -1)
    odd = ~torch.isfinite(y).all(-1)
    y = torch.nan_to_num(y, nan=0.0, posinf=MAX, neginf=-MAX).clamp(-MAX, MAX)
    zero = f16_down(y.amin(-1))
    step = -f16_down(-(y.amax(-1) - zero) / 15.0)
    t = (y - zero[..., None]) / torch.where(step > 0, step, torch.ones_like(step))[..., None]
    codes = torch.round(t).clamp(0, 15)     # (torch.round: ties to even)
    codes = torch.where((step > 0)[..., None], codes, torch.zeros_like(codes))
    nan = torch.full_like(zero, math.nan)
    return codes, torch.where(odd, nan, step), torch.where(odd, nan, zero)


def held64(x):
    """The values that the cache holds for rows x, in 64 bits."""
    codes, step, zero = quantise64(x)
    return (zero[..., None] + codes * step[..., None]).flatten(-2)


def attend64(q, k, v, scale, dtype):
    """
    Causal attention of the last n of N tokens: q (n, Hq, D); k, v (N, Hkv, D)
    rows before they are quantised. Returns (out, bound), (n, Hq, D) in 64 bits.

    The kernels compute sum_t r_t c_t + sum_t p_t (zero_t + 7.5 step_t) - 7.5
    sum_t r_t, p the softmax's weights and r_t = p_t step_t rounded to float16,
    so that r_t's error enters times c_t - 7.5 (the plain ones sum_t p_t (zero_t +
    step_t c_t)). With u = eps / 2 of the output's type, v16 = 2^-11, B = sum_t
    p_t (step_t c_t + |zero_t + 7.5 step_t| + 7.5 step_t), per output element:
      u |out|                          the output's rounding
      v16 sum_t p_t step_t |c_t - 7.5| each product's rounding
      (2 delta + 2 (N + 64) 2^-24) B   32 bits: delta bounds a score's error
                                       (terms of magnitude |q| (step c + |zero|):
                                       D + 8 roundings of the sum, the factors
                                       and the exponent), which moves a weight
                                       and the sum by its factor; sums of N
                                       terms and the merge of parts
      N 2^-25 15 S                     p step below 2^-14 rounds by 2^-25 of a
                                       unit in which the largest step S of the
                                       sequence is below 2 and the row's largest
                                       p at least 1 / 2: up to 4 units a code,
                                       hence 4 times that
    """
    n, hq, d = q.shape
    total, hkv = k.shape[0], k.shape[1]
    gr = hq // hkv
    (kc, ks, kz), (vc, vs, vz) = quantise64(k), quantise64(v)
    kk, kb = ((kz[..., None] + kc * ks[..., None]).flatten(-2),
              (kz.abs()[..., None] + kc * ks[..., None]).flatten(-2))
    vv, vb = ((vz[..., None] + vc * vs[..., None]).flatten(-2),
              ((vz + 7.5 * vs).abs()[..., None] + (vc + 7.5) * vs[..., None]).flatten(-2))
    vr = ((vc - 7.5).abs() * vs[..., None]).flatten(-2)
    u = torch.finfo(dtype).eps / 2
    qq = q.detach().cpu().double()
    see = torch.arange(total) <= torch.arange(total - n, total)[:, None]
    out, bound = torch.empty_like(qq), torch.empty_like(qq)
    for h in range(hq):
        of = h // gr
        s = qq[:, h] @ kk[:, of].t() * scale
        p = torch.softmax(s.masked_fill(~see, -math.inf), dim=-1)
        delta = ((d + 8) * 2.0 ** -24 * abs(scale)
                 * (qq[:, h].abs() @ kb[:, of].t()).masked_fill(~see, 0).amax(1, keepdim=True))
        out[:, h] = p @ vv[:, of]
        bound[:, h] = (u * out[:, h].abs() + 2.0 ** -11 * (p @ vr[:, of])
                       + (2 * delta + 2 * (total + 64) * 2.0 ** -24) * (p @ vb[:, of])
                       + total * 2.0 ** -23 * 15 * vs[:, of].max())
    return out, bound * 1.001 + torch.finfo(dtype).tiny
