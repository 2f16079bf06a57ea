"""Plain 64-bit references of the paged cache's operators (include/lcpp_b200_model.h), written from their definitions:
rotary positions, attention over pages, eviction."""
from __future__ import annotations

import numpy as np
import torch

HALF, INTERLEAVED = 0, 1


def turn(x, positions, frequencies, layout, scale=1.0, inverse=False):
    """x [tokens, heads, dim] float64; (turned, sum of the magnitudes that went into each value)."""
    angle = np.asarray(positions, np.longdouble)[:, None] * np.asarray(frequencies, np.longdouble)
    angle = np.fmod(angle, 2 * np.longdouble("3.14159265358979323846264338327950288"))
    cos, sin = np.cos(angle).astype(np.float64) * scale, np.sin(angle).astype(np.float64) * scale
    if inverse:
        sin = -sin
    out, size = np.array(x, np.float64), np.abs(np.array(x, np.float64))
    half = len(frequencies)
    for i in range(half):
        a, b = (i, i + half) if layout == HALF else (2 * i, 2 * i + 1)
        c, s = cos[:, i, None], sin[:, i, None]
        out[:, :, a] = x[:, :, a] * c - x[:, :, b] * s
        out[:, :, b] = x[:, :, b] * c + x[:, :, a] * s
        size[:, :, a] = size[:, :, b] = (np.abs(x[:, :, a]) + np.abs(x[:, :, b])) * scale
    return out, size


def attend(q, k, v, table, lens, scale, window=0, softcap=0.0, scores=None, decay=1.0):
    """Float64 torch tensors: q [r, h, d], caches [pages, block, kv, d]; lists otherwise.
    (out, sum p |v|, lse, scores after the step or None)."""
    r, h, d = q.shape
    pages, block, kv, _ = k.shape
    out, size = torch.zeros_like(q), torch.zeros_like(q)
    lse = torch.full((r, h), -float("inf"), dtype=torch.float64, device=q.device)
    after = None if scores is None else scores.clone()
    for i in range(r):
        n = max(0, min(int(lens[i]), table.shape[1] * block))
        token = torch.arange(n, device=q.device)
        page = table[i].to(q.device).long()[token // block]
        seen = (page >= 0) & (page < pages)
        slot = (page * block + token % block)[seen]
        if after is not None:
            after[slot] = decay * scores[slot]
        if window:
            seen &= token >= n - window
        slot = (page * block + token % block)[seen]
        if not len(slot):
            continue
        kk, vv = k[slot // block, slot % block], v[slot // block, slot % block]
        x = torch.einsum("kgd,tkd->kgt", q[i].view(kv, h // kv, d), kk) * scale
        if softcap:
            x = softcap * torch.tanh(x / softcap)
        top = x.max(-1, keepdim=True).values
        live = ~torch.isneginf(top)
        e = torch.exp(x - torch.where(live, top, torch.zeros_like(top)))
        total = e.sum(-1, keepdim=True)
        p = torch.where(live, e / total, torch.zeros_like(e))
        lse[i] = torch.where(live, top + total.log(), top).flatten()
        out[i] = torch.einsum("kgt,tkd->kgd", p, vv).reshape(h, d)
        size[i] = torch.einsum("kgt,tkd->kgd", p, vv.abs()).reshape(h, d)
        if after is not None:
            after[slot] += p.sum((0, 1))
    return out, size, lse, after


def evict(lens, table, scores, positions, evicted, budget, trigger, first, recent, block, pages, room):
    """(lengths, evicted, moves of each request as [(from, to)], freed pages in order)."""
    new, gone, moves, freed = [], [], [], []
    for r, n in enumerate(lens):
        n = max(0, min(int(n), table.shape[1] * block))
        page = table[r, np.arange(n) // block].astype(np.int64)
        slot = page * block + np.arange(n) % block
        pairs = None
        if n > trigger and ((page >= 0) & (page < pages)).all():
            position = np.arange(n) if positions is None else positions[slot].astype(np.int64)
            safe = (position < first) | (position >= n + int(evicted[r]) - recent)
            s = scores[slot].astype(np.float64)
            # protected, then NaN, then by score; equal ones by place
            kind = np.where(safe, 2, np.where(np.isnan(s), 1, 0))
            s = np.where(kind > 0, 0.0, s)
            order = np.lexsort((np.arange(n), -s, -kind))
            kept = np.zeros(n, bool)
            kept[order[:budget]] = True
            holes = [i for i in range(budget) if not kept[i]]
            fillers = [i for i in range(budget, n) if kept[i]]
            if len(fillers) <= room:
                pairs = [(int(slot[f]), int(slot[h])) for f, h in zip(fillers, holes)]
        if pairs is None:
            new.append(n)
            gone.append(int(evicted[r]))
            moves.append([])
        else:
            new.append(budget)
            gone.append(int(evicted[r]) + n - budget)
            moves.append(pairs)
            freed += list(table[r, -(-budget // block):-(-n // block)])
    return new, gone, moves, freed
