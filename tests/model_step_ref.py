"""Plain 64-bit references of the model-step operators (include/lcpp_b200_model.h), written from their
definitions with numpy and Python loops."""
from __future__ import annotations

import numpy as np

SOFTMAX, SIGMOID = 0, 1


def extend(context, new, table, width, free, used, tokens, block):
    """Block table, slots, positions, token requests, starts, sequence lengths, used."""
    table = table.copy()
    slots, positions = np.full(tokens, -1, np.int64), np.zeros(tokens, np.int32)
    requests = np.full(tokens, -1, np.int32)
    starts, seq_lens = [0], []
    at = taken = 0
    used_after = used
    for r in range(len(context)):
        c, n = max(int(context[r]), 0), 1 if new is None else max(int(new[r]), 0)
        held, total = -(-c // block), -(-(c + n) // block)
        in_row = total <= width and c + n < 2 ** 31
        need = total - held if in_row else 0
        fits = in_row and at + n <= tokens and (need == 0 or used + taken + need <= len(free))
        if fits:
            table[r, held:total] = free[used + taken:used + taken + need]
            used_after = max(used_after, used + taken + need) if need else used_after
            for i in range(n):
                p = c + i
                page = int(table[r, p // block])
                slots[at + i] = -1 if page < 0 else page * block + p % block
                positions[at + i], requests[at + i] = p, r
        seq_lens.append(c + n if fits else c)
        at += n
        taken += need
        starts.append(min(at, 2 ** 31 - 1))
    return table, slots, positions, requests, np.array(starts), np.array(seq_lens, np.int64), used_after


def _scores(x, score):
    """(log scores, shares) of float64 rows; rows without a finite logit give NaN."""
    with np.errstate(all="ignore"):
        if score == SOFTMAX:
            log_s = x - x.max(1, keepdims=True)
            log_s = log_s - np.log(np.exp(log_s).sum(1, keepdims=True))
        else:
            log_s = np.where(x < 0, x, 0.0) - np.log1p(np.exp(-np.abs(x)))
        share = np.exp(log_s - log_s.max(1, keepdims=True))
        return log_s, share / share.sum(1, keepdims=True)


def choose(logits32, bias32, k):
    """Experts by (logit + bias in 32 bits, lower index first), -1 where none is left."""
    key = logits32 if bias32 is None else (logits32 + bias32).astype(np.float32)
    key = np.where(np.isneginf(logits32), np.float32(-np.inf), key)
    order = np.where(np.isnan(key), np.float64(np.inf), key.astype(np.float64))
    rank = np.lexsort((np.broadcast_to(np.arange(key.shape[1]), key.shape), -order, ~np.isnan(key)), axis=1)[:, :k]
    return np.where(np.isneginf(np.take_along_axis(key, rank, 1)), -1, rank)


def route(logits32, k, score, renormalize, scale, coef, bias32=None, mask=None):
    t, e = logits32.shape
    experts = choose(logits32, bias32, k)
    if mask is not None:
        experts = np.where((mask < 0)[:, None], -1, experts)
    x = logits32.astype(np.float64)
    log_s, share = _scores(x, score)
    live, has = experts[:, 0] >= 0, experts >= 0
    with np.errstate(all="ignore"):
        picked = np.where(has, np.take_along_axis(log_s, np.maximum(experts, 0), 1), -np.inf)
        if renormalize:
            top = picked.max(1, keepdims=True)
            w = np.exp(picked - top)
            w = w / w.sum(1, keepdims=True)
        else:
            w = np.exp(picked)
    weights = np.where(has, scale * w, 0.0)
    counts = np.bincount(experts[has], minlength=e)
    routed = int(live.sum())
    loss = 0.0
    if routed:
        loss = coef * e * (share[live].sum(0) / routed * counts / (k * routed)).sum()
    return weights, experts, counts, routed, loss


def route_objective(x, experts, counts, routed, g, dloss, score, renormalize, scale, coef):
    """sum(weights * g) + loss * dloss with the choice and the counts held, in 64 bits."""
    k, e = experts.shape[1], x.shape[1]
    log_s, share = _scores(x, score)
    has, live = experts >= 0, experts[:, 0] >= 0
    with np.errstate(all="ignore"):
        w = np.where(has, np.exp(np.take_along_axis(log_s, np.maximum(experts, 0), 1)), 0.0)
        if renormalize:
            w = w / w.sum(1, keepdims=True)
    total = scale * (w * g)[live].sum()
    if routed:
        total += dloss * coef * e * (share[live].sum(0) / routed * counts / (k * routed)).sum()
    return total


def route_grad(x, experts, counts, routed, g, dloss, score, renormalize, scale, coef):
    """Gradient of route_objective, by its formula."""
    t, e = x.shape
    k = experts.shape[1]
    log_s, share = _scores(x, score)
    out = np.zeros((t, e))
    pull = dloss * coef * e * counts / (k * float(max(routed, 1)) ** 2)
    for i in range(t):
        if experts[i, 0] < 0:
            continue
        s = np.exp(log_s[i])
        slope = np.ones(e) if score == SOFTMAX else 1.0 - s
        d = share[i] * (pull - (share[i] * pull).sum())
        chosen = experts[i][experts[i] >= 0]
        gi = g[i][experts[i] >= 0]
        part = np.exp(log_s[i][chosen] - log_s[i][chosen].max())
        part = part / part.sum()
        if renormalize:
            d[chosen] += scale * part * (gi - (gi * part).sum())
        else:
            d[chosen] += scale * s[chosen] * gi
            if score == SOFTMAX:
                d -= s * (scale * (gi * s[chosen]).sum())
        out[i] = slope * d
    return out


def plan(experts, num_experts, align, max_rows):
    """(starts, row_of, pair_of) of the stable grouping."""
    flat = experts.reshape(-1)
    starts, row_of, pair_of = [0], np.full(flat.size, -1), np.full(max_rows, -1)
    for e in range(num_experts):
        pairs = np.nonzero(flat == e)[0]
        rows = starts[-1] + np.arange(pairs.size)
        keep = rows < max_rows
        row_of[pairs[keep]] = rows[keep]
        pair_of[rows[keep]] = pairs[keep]
        starts.append(starts[-1] + -(-pairs.size // align) * align)
    return np.array(starts), row_of.reshape(experts.shape), pair_of


def gather(x, pair_of, k, end):
    """Rows below `end`: the token's row, or zeros."""
    rows = np.zeros((min(end, pair_of.size), x.shape[1]), x.dtype)
    for r in range(rows.shape[0]):
        if pair_of[r] >= 0:
            rows[r] = x[pair_of[r] // k]
    return rows


def combine(rows, row_of, weights):
    out = np.zeros((row_of.shape[0], rows.shape[1]))
    for t, j in zip(*np.nonzero(row_of >= 0)):
        out[t] += (1.0 if weights is None else weights[t, j]) * rows[row_of[t, j]]
    return out


def combine_grad(grad_out, rows, row_of, pair_of, weights, end):
    k = row_of.shape[1]
    grad_rows, grad_weights = np.zeros((min(end, rows.shape[0]), rows.shape[1])), np.zeros(row_of.shape)
    for r in range(grad_rows.shape[0]):
        if pair_of[r] >= 0:
            t, j = divmod(int(pair_of[r]), k)
            grad_rows[r] = weights[t, j] * grad_out[t]
            grad_weights[t, j] = grad_out[t] @ rows[r]
    return grad_rows, grad_weights
