"""Verification of drafted tokens by its definition, in 64 bits, row by row."""

from __future__ import annotations

import math

import torch


def greedy_id(row):
    """torch's argmax order: the first NaN, else the first of the largest."""
    nan = row.isnan().nonzero()
    return int(nan[0]) if len(nan) else int((row == row.max()).nonzero()[0])


def verify64(logits, tokens, lens, numbers, probs=None, temps=1.0):
    """(ids, accepted, margin) of CPU tensors; margin: how close the nearest
    decision was to its border (relative to the sum)."""
    temps = [temps] * len(lens) if not isinstance(temps, list) else temps
    vocab = logits.shape[1]
    ids, counts, margin = [], [], math.inf
    at = 0
    for i, (n, t) in enumerate(zip(lens, temps)):
        run, pick = 0, None
        while pick is None:
            r = at + run
            row = logits[r].double()
            x = int(tokens[r + 1]) if run < n - 1 else None
            best = greedy_id(row)
            broken = bool(row.isnan().any()) or float(row.max()) in (math.inf, -math.inf)
            if not t > 0 or broken:
                if x == best and not broken:
                    run += 1
                else:
                    pick = best
                continue
            p = torch.softmax(row / t, dim=-1)
            w = p
            if x is not None:
                ok = 0 <= x < vocab
                q = probs[r - i].double() if probs is not None else None
                if ok:
                    need = float(numbers[r]) * (1.0 if q is None else float(q[x]))
                    if need != 0 or float(p[x]) != 0:      # (both exactly 0: no rounding)
                        margin = min(margin, abs(need - float(p[x])) / max(float(p[x]), 1e-300))
                    if need < float(p[x]):
                        run += 1
                        continue
                if q is not None:
                    w = torch.relu(p - q)
                elif ok:
                    w = p.clone()
                    w[x] = 0
                if not float(w.sum()) > 0:
                    w = p
            cum = torch.cumsum(w, 0)
            target = float(numbers[at + n - 1]) * float(cum[-1])
            margin = min(margin, float(((cum - target).abs() / cum[-1])[w > 0].min()))
            past = (cum > target).nonzero()
            pick = int(past[0]) if len(past) else int(w.nonzero()[-1])
        ids.append(([int(z) for z in tokens[at + 1:at + 1 + run]] + [pick]
                    + [-1] * (max(lens) - run - 1)))
        counts.append(run)
        at += n
    return torch.tensor(ids), torch.tensor(counts), margin
