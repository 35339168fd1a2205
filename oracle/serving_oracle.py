"""Oracle of a serving step over a paged cache: rotary positions, attention of a step's rows, verification of drafts, in 64 bits on the CPU, from the definitions.

TEST INFRASTRUCTURE ONLY.  Nothing in the product package may import this module.  Loops over sequences, rows and heads; masks and pages as they are written
down, no tiles, no running statistics.
"""
from __future__ import annotations

import math

import torch


def rotary(x, cos, sin, positions, interleaved=False, back=False):
    """x [B,T,H,D], positions [B,T] (a negative one: the row as it is) -> (y, magnitude of what is added up), both fp64."""
    x, cos, sin = x.double().cpu(), cos.double().cpu(), sin.double().cpu()
    half = cos.shape[1]
    y, size = x.clone(), x.abs().clone()
    for b in range(x.shape[0]):
        for t in range(x.shape[1]):
            pos = int(positions[b, t])
            if pos < 0:
                continue
            for j in range(half):
                i1, i2 = (2 * j, 2 * j + 1) if interleaved else (j, j + half)
                c, s = (cos[pos, j], -sin[pos, j] if back else sin[pos, j]) if pos < cos.shape[0] else (math.nan, math.nan)
                y[b, t, :, i1], y[b, t, :, i2] = x[b, t, :, i1] * c - x[b, t, :, i2] * s, x[b, t, :, i1] * s + x[b, t, :, i2] * c
                size[b, t, :, i1] = (x[b, t, :, i1] * c).abs() + (x[b, t, :, i2] * s).abs()
                size[b, t, :, i2] = (x[b, t, :, i1] * s).abs() + (x[b, t, :, i2] * c).abs()
    return y, size


def slot_of(table, n, slot, pages, page_size):
    """(page, place in it) or None."""
    if slot < 0 or slot >= table.shape[1] * page_size:
        return None
    page = int(table[n, slot // page_size])
    return (page, slot % page_size) if 0 <= page < pages else None


def paged_attn(q, k_cache, v_cache, table, context, rows, sees, scale):
    """q [rows of all sequences, HQ, D]; rows: [(first, last)] of each sequence; sees(n, i, j) -> whether row i sees row j of its sequence.

    Returns (o, sum_j p_j |v_j|, largest sum_d |q_d k_d scale| over the keys seen, largest |score - maximum|), fp64."""
    q, k_cache, v_cache = q.double().cpu(), k_cache.double().cpu(), v_cache.double().cpu()
    pages, page_size, HK, D = k_cache.shape
    HQ = q.shape[1]
    o, size = torch.zeros_like(q), torch.zeros_like(q)
    dots, spread = torch.zeros(q.shape[:2], dtype=torch.float64), torch.zeros(q.shape[:2], dtype=torch.float64)
    for n, (first, last) in enumerate(rows):
        at = [slot_of(table, n, j, pages, page_size) for j in range(int(context[n]) + last - first)]
        for i in range(last - first):
            seen = [a for j, a in enumerate(at) if a is not None and (j < int(context[n]) or sees(n, i, j - int(context[n])))]
            if not seen:
                continue
            page, place = (torch.tensor(x) for x in zip(*seen))
            for h in range(HQ):
                k, v, x = k_cache[page, place, h * HK // HQ], v_cache[page, place, h * HK // HQ], q[first + i, h]
                s = (k * x).sum(1) * scale
                w = torch.exp(s - s.max())
                w = w / w.sum()
                o[first + i, h] = (w[:, None] * v).sum(0)
                size[first + i, h] = (w[:, None] * v.abs()).sum(0)
                dots[first + i, h] = (k * x).abs().sum(1).max() * abs(scale)
                spread[first + i, h] = (s.max() - s).max()
    return o, size, dots, spread


def verify_drafts(p, tokens, u, parents=None, q=None, lengths=None):
    """p, q [N,R,V], tokens, u [N,R], parents [R] or [N,R], lengths [N] -> (next_token, accepted, rows)."""
    N, R, V = p.shape
    clean = lambda x: torch.nan_to_num(x.double().cpu(), nan=0.0, posinf=math.inf).clamp(min=0)
    p, q = clean(p), None if q is None else clean(q)
    token, accepted, rows = torch.zeros(N, dtype=torch.int64), torch.zeros(N, dtype=torch.int32), torch.full((N, R), -1, dtype=torch.int32)
    for n in range(N):
        count = R if lengths is None else min(max(int(lengths[n]), 1), R)
        path, left = [0], p[n, 0].clone()
        for r in range(1, count):
            parent = r - 1 if parents is None else int(parents[r] if parents.dim() == 1 else parents[n, r])
            word = int(tokens[n, r])
            # (a word outside the vocabulary was drawn from nothing: there is nothing of it to take from p)
            if parent != path[-1] or parent >= r or not 0 <= word < V:
                continue
            chance = 1.0 if q is None else float(q[n, parent, word])
            if float(u[n, r]) * chance < float(left[word]):
                path.append(r)
                left = p[n, r].clone()
                continue
            rest = left.clone()
            if q is not None:
                rest = (rest - q[n, parent]).clamp(min=0)
            else:
                rest[word] = 0
            if float(rest.sum()) > 0:
                left = rest / rest.sum()
        upto = left.cumsum(0)
        total = float(upto[-1])
        if not 0 < total < math.inf:
            token[n] = -1
        else:
            passed = (upto > float(u[n, 0]) * total).nonzero()
            token[n] = int(passed[0]) if len(passed) else int((left > 0).nonzero()[-1])
        accepted[n] = len(path)
        rows[n, :len(path)] = torch.tensor(path, dtype=torch.int32)
    return token, accepted, rows
