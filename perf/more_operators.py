"""The operators of a paged key-value cache as they are measured: rotary positions with the write into the cache,
attention of one new token over the pages, and eviction by accumulated attention weight, each in a plain form of
elementary torch operations and as the library's own calls.

``own`` chooses the side: false runs the plain form in 32 bits, true the calls of ``lcpp_b200``.
"""
from __future__ import annotations

import math
import sys
from pathlib import Path

import torch

own = False

_DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_BYTES = {"f32": 4, "bf16": 2, "f16": 2}
_BASE = 500000.0
_library = None


def _lib():
    global _library
    if _library is None:
        package = str(Path(__file__).resolve().parent.parent / "luisacompute-parallelprimitive_b200")
        if package not in sys.path:
            sys.path.insert(0, package)
        import lcpp_b200
        _library = lcpp_b200
    return _library


# ---------------------------------------------------------------------------
# Cases
# ---------------------------------------------------------------------------
def listed():
    return [
        # one decode step of a small server: queries and keys turned, keys and values written to their pages
        {"name": "append_decode", "op": "append", "tokens": 64, "heads": 32, "kv_heads": 8, "dim": 128, "rotary": 128,
         "layout": "half", "dtype": "bf16", "block": 16, "order": "tokens", "far": 8192, "padded": False},
        # a long prompt chunk far into its context: part of the head turned, adjacent pairs, a page size that is no
        # power of two, heads before tokens in a page, arrays padded to a captured graph's capacity
        {"name": "append_prompt", "op": "append", "tokens": 8191, "heads": 24, "kv_heads": 4, "dim": 192, "rotary": 64,
         "layout": "interleaved", "dtype": "f16", "block": 24, "order": "heads", "far": 1_000_000, "padded": True},
        # a training batch
        {"name": "rotary_train", "op": "rotary", "tokens": 32768, "heads": 32, "kv_heads": 8, "dim": 128,
         "rotary": 128, "layout": "half", "dtype": "bf16", "far": 32768},
        # the gradient for a ragged batch in 32 bits, part of the head turned
        {"name": "rotary_grad_odd", "op": "rotary_grad", "tokens": 5003, "heads": 12, "kv_heads": 3, "dim": 80,
         "rotary": 40, "layout": "interleaved", "dtype": "f32", "far": 4096},
        # one request early in its answer: latency
        {"name": "attend_one", "op": "attend", "requests": 1, "context": 700, "heads": 32, "kv_heads": 8, "dim": 128,
         "dtype": "bf16", "block": 16, "order": "tokens", "window": 0, "scored": False},
        # a server's batch of long and short requests
        {"name": "attend_batch", "op": "attend", "requests": 64, "context": 16384, "heads": 32, "kv_heads": 8,
         "dim": 128, "dtype": "bf16", "block": 16, "order": "tokens", "window": 0, "scored": False},
        # two requests of a very long context: the work of a request is split over the whole GPU
        {"name": "attend_long", "op": "attend", "requests": 2, "context": 131072, "heads": 16, "kv_heads": 2,
         "dim": 256, "dtype": "f16", "block": 64, "order": "heads", "window": 0, "scored": False},
        # many short requests in 32 bits with a sliding window, odd head and page sizes, a head for each query
        {"name": "attend_window", "op": "attend", "requests": 301, "context": 1500, "heads": 7, "kv_heads": 7,
         "dim": 80, "dtype": "f32", "block": 24, "order": "tokens", "window": 1000, "scored": False},
        # a batch whose attention weights are gathered for eviction
        {"name": "attend_scored", "op": "attend", "requests": 48, "context": 4096, "heads": 40, "kv_heads": 8,
         "dim": 128, "dtype": "bf16", "block": 32, "order": "tokens", "window": 0, "scored": True},
        # requests that passed their budget by a page in the course of their answers
        {"name": "evict_page", "op": "evict", "requests": 64, "context": 2100, "budget": 2048, "trigger": 2063,
         "first": 4, "recent": 256, "block": 16},
        # prompts cut down to their heaviest tokens
        {"name": "evict_prompts", "op": "evict", "requests": 16, "context": 131072, "budget": 8192, "trigger": 8192,
         "first": 16, "recent": 1024, "block": 64},
        # the moves of those prompts in one layer's cache
        {"name": "move_prompts", "op": "move", "requests": 16, "context": 131072, "budget": 8192, "trigger": 8192,
         "first": 16, "recent": 1024, "block": 64, "kv_heads": 8, "dim": 128, "dtype": "bf16", "order": "tokens"},
    ]


def _log_int(rng, low, high):
    return max(low, min(high, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng):
    op = rng.choice(["append", "rotary", "rotary_grad", "attend", "attend", "attend", "evict", "move"])
    dtype = rng.choice(["f32", "bf16", "bf16", "f16"])
    kv_heads = rng.choice([1, 2, 3, 4, 8, 8])
    heads = kv_heads * rng.choice([1, 2, 3, 4, 4, 5, 7, 8, 12, 16])
    dim = rng.choice([64, 64, 80, 96, 128, 128, 128, 192, 256])
    block = rng.choice([1, 8, 16, 16, 24, 32, 64, 128])
    order = rng.choice(["tokens", "heads"])
    row = dim * _BYTES[dtype]
    if op in ("append", "rotary", "rotary_grad"):
        rotary = rng.choice([dim, dim, dim // 2, 2 * rng.randint(1, dim // 2)])
        budget = 32768 * 40 * 256 // (row * (heads + 2 * kv_heads))
        case = {"op": op, "tokens": _log_int(rng, 1, min(65536, budget)), "heads": heads, "kv_heads": kv_heads,
                "dim": dim, "rotary": rotary, "layout": rng.choice(["half", "interleaved"]), "dtype": dtype,
                "far": _log_int(rng, 1, 1_000_000)}
        return case | ({"block": block, "order": order, "padded": rng.random() < 0.5} if op == "append" else {})
    if op == "attend":
        requests = _log_int(rng, 1, 512)
        tokens = min(940_000_000 // (row * kv_heads), 2_400_000_000 // (heads * dim))
        context = _log_int(rng, 1, max(1, min(131072, tokens // requests)))
        return {"op": op, "requests": requests, "context": context, "heads": heads, "kv_heads": kv_heads, "dim": dim,
                "dtype": dtype, "block": block, "order": order,
                "window": rng.choice([0, 0, _log_int(rng, 1, context)]), "scored": rng.random() < 0.3}
    requests = _log_int(rng, 1, 512)
    context = _log_int(rng, 2, min(131072, 16 * 131072 // requests))
    budget = rng.randint(1, context)
    first, recent = rng.randint(0, budget // 4), rng.randint(0, budget // 2)
    case = {"op": op, "requests": requests, "context": context, "budget": budget,
            "trigger": budget + rng.choice([0, rng.randint(0, block)]), "first": first, "recent": recent, "block": block}
    if op == "evict":
        return case
    fit = 5_500_000_000 // (2 * row * kv_heads * requests)  # moves of no more bytes than the largest listed reads
    case["context"] = max(2, min(context, fit))
    case["budget"] = budget = min(budget, case["context"])
    case["trigger"], case["first"], case["recent"] = budget, min(first, budget // 4), min(recent, budget // 2)
    return case | {"kv_heads": kv_heads, "dim": dim, "dtype": dtype, "order": order}


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------
def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed * 6271 + 29)


def _rand(g, *shape):
    return torch.rand(*shape, device="cuda", generator=g)


def _randn(g, dtype, *shape):
    return torch.randn(*shape, device="cuda", generator=g, dtype=dtype)


def _cache(g, case, pages):
    """Keys or values of `pages` pages, [page, token, head, column] in either memory order."""
    block, heads, dim, dtype = case["block"], case["kv_heads"], case["dim"], _DTYPES[case["dtype"]]
    if case["order"] == "tokens":
        return _randn(g, dtype, pages, block, heads, dim)
    return _randn(g, dtype, pages, heads, block, dim).transpose(1, 2)


def _table(g, lens, width, block):
    """Page ids of every request, no page twice, the pages in no order; (table, pages of the pool)."""
    r = lens.numel()
    held = (lens.to(torch.int64) + block - 1) // block
    pages = int(held.sum()) + 2
    order = torch.randperm(pages - 2, device="cuda", generator=g)
    column = torch.arange(width, device="cuda")
    index = (torch.cumsum(held, 0) - held)[:, None] + column
    page = order[index.clamp(max=max(0, pages - 3))] if pages > 2 else torch.zeros_like(index)
    return torch.where(column < held[:, None], page, -1).to(torch.int32).view(r, width).contiguous(), pages


def _prepare_rotary(case, g):
    t, h, kv, d, dtype = case["tokens"], case["heads"], case["kv_heads"], case["dim"], _DTYPES[case["dtype"]]
    # one projection gives queries, keys and values side by side
    rows = _randn(g, dtype, t, (h + 2 * kv) * d)
    q, k, v = (x.unflatten(1, (-1, d)) for x in rows.split((h * d, kv * d, kv * d), 1))
    index = torch.arange(case["rotary"] // 2, device="cuda", dtype=torch.float64)
    state = {"q": q, "k": k, "v": v, "frequencies": _BASE ** (-2 * index / case["rotary"])}
    if case["op"] != "append":
        state["positions"] = (_rand(g, t) * case["far"]).to(torch.int32)
        return state | {"q_out": torch.zeros(t, h, d, dtype=dtype, device="cuda"),
                        "k_out": torch.zeros(t, kv, d, dtype=dtype, device="cuda")}
    live = t - t // 9 if case["padded"] else t
    slot_count = (t + case["block"] - 1) // case["block"] * case["block"]
    pages = slot_count // case["block"] + 2
    page = torch.randperm(pages - 1, device="cuda", generator=g)
    token = torch.arange(t, device="cuda")
    slots = page[token // case["block"]] * case["block"] + token % case["block"]
    start = int(_rand(g, 1) * case["far"])
    inside = token < live
    state |= {"slots": torch.where(inside, slots, -1), "positions": torch.where(inside, start + token, 0).to(torch.int32),
              "requests": torch.where(inside, 0, -1).to(torch.int32)}
    # the cache's last page belongs to nobody
    return state | {"q_out": torch.zeros(t, h, d, dtype=dtype, device="cuda"), "k_cache": _cache(g, case, pages),
                    "v_cache": _cache(g, case, pages)}


def _prepare_attend(case, g):
    r, h, d, dtype = case["requests"], case["heads"], case["dim"], _DTYPES[case["dtype"]]
    # lengths from a quarter of the longest on, in the seed's order; one request in twenty idle
    rank = torch.randperm(r, device="cuda", generator=g)
    lens = (case["context"] * (1 - 0.75 * rank / r)).to(torch.int32).clamp(min=1)
    lens[rank % 20 == 13] = 0
    width = (case["context"] + case["block"] - 1) // case["block"] + 1
    table, pages = _table(g, lens, width, case["block"])
    f32 = {"dtype": torch.float32, "device": "cuda"}
    # some heads look closely, others far around
    q = _randn(g, dtype, r, h, d) * (0.5 + 2 * _rand(g, h, 1)).to(dtype)
    state = {"lens": lens, "table": table, "q": q, "k": _cache(g, case, pages), "v": _cache(g, case, pages),
             "out": torch.zeros(r, h, d, dtype=dtype, device="cuda"), "lse": torch.zeros(r, h, **f32), "pages": pages}
    if case["scored"]:
        slots = pages * case["block"]
        state |= {"scores": _rand(g, slots) * 4, "scores_out": torch.zeros(slots, **f32)}
    return state


def _evict_width(case):
    return (case["context"] + case["block"] - 1) // case["block"]


def _evict_moves(case):
    return max(1, min(case["budget"], case["context"] - case["budget"]))


def _prepare_evict(case, g):
    r, context, block = case["requests"], case["context"], case["block"]
    rank = torch.randperm(r, device="cuda", generator=g)
    lens = (context - (context - case["budget"]) * 1.2 * (rank / r) ** 2).to(torch.int32).clamp(min=1)
    table, pages = _table(g, lens, _evict_width(case), block)
    # a few heavy tokens, many light ones; weights of tokens that nothing looked at are equal
    scores = (_rand(g, pages * block) * 12 - 6).exp()
    scores[_rand(g, pages * block) < 0.05] = 0
    i32 = {"dtype": torch.int32, "device": "cuda"}
    # tokens in the order in which earlier evictions left them: filled holes in the front part
    evicted = (_rand(g, r) * context).to(torch.int32)
    total = (lens + evicted).to(torch.int64)
    index = torch.arange(_evict_width(case) * block, device="cuda")
    shuffle = torch.where(index % 5 == 3, index * 2 % 7, 0)
    position = ((index + evicted[:, None] - shuffle) % total.clamp(min=1)[:, None]).to(torch.int32)
    slot = table.to(torch.int64).repeat_interleave(block, 1) * block + index % block
    held = index < lens[:, None]
    positions = torch.zeros(pages * block, **i32)
    positions[slot[held]] = position[held]
    free = torch.arange(pages, pages + pages + 11, **i32)
    state = {"lens": lens, "table": table, "scores": scores, "positions": positions, "evicted": evicted, "pages": pages,
             "free": free, "used": torch.full((1,), pages + 7, **i32), "used_out": torch.zeros(1, **i32),
             "lens_out": torch.zeros(r, **i32), "evicted_out": torch.zeros(r, **i32), "counts": torch.zeros(r, **i32),
             "moves": torch.full((r, _evict_moves(case), 2), -1, dtype=torch.int64, device="cuda")}
    if case["op"] == "evict":
        return state
    plan = _plain_evict(case, state)
    keep = {k: state[k] for k in ("scores", "positions", "pages")}
    return keep | {"moves": plan["moves"], "counts": plan["counts"], "k": _cache(g, case, pages),
                   "v": _cache(g, case, pages)}


def prepare(case, seed):
    g = _generator(seed)
    if case["op"] in ("append", "rotary", "rotary_grad"):
        state = _prepare_rotary(case, g)
    elif case["op"] == "attend":
        state = _prepare_attend(case, g)
    else:
        state = _prepare_evict(case, g)
    return {"case": case, **state}


# ---------------------------------------------------------------------------
# Plain forms
# ---------------------------------------------------------------------------
def _plain_turn(case, x, cos, sin):
    """The first `rotary` columns of every head turned, the others as they are."""
    rotary = case["rotary"]
    x = x.float()
    turned, rest = x[..., :rotary], x[..., rotary:]
    if case["layout"] == "half":
        a, b = turned[..., :rotary // 2], turned[..., rotary // 2:]
        return torch.cat([a * cos - b * sin, b * cos + a * sin, rest], -1)
    a, b = turned[..., 0::2], turned[..., 1::2]
    return torch.cat([torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2), rest], -1)


def _plain_angles(s):
    """Angles in 64 bits: far positions lose their fractions in 32."""
    angle = s["positions"].double()[:, None] * s["frequencies"]
    return angle.cos().float()[:, None], angle.sin().float()[:, None]


def _plain_rotary(case, s):
    cos, sin = _plain_angles(s)
    if case["op"] == "rotary_grad":
        sin = -sin
    return {"q": _plain_turn(case, s["q"], cos, sin).to(s["q"].dtype),
            "k": _plain_turn(case, s["k"], cos, sin).to(s["k"].dtype)}


def _plain_append(case, s):
    cos, sin = _plain_angles(s)
    live, block = s["slots"] >= 0, case["block"]
    q = torch.where(live[:, None, None], _plain_turn(case, s["q"], cos, sin).to(s["q"].dtype), s["q_out"])
    # the marked tokens go to the page that belongs to nobody
    slot = torch.where(live, s["slots"], s["k_cache"].shape[0] * block - 1)
    s["k_cache"][slot // block, slot % block] = _plain_turn(case, s["k"], cos, sin).to(s["k"].dtype)
    s["v_cache"][slot // block, slot % block] = s["v"]
    return {"q": q, "k_cache": s["k_cache"][:-1], "v_cache": s["v_cache"][:-1]}


def _plain_slots(case, s, count):
    """Slots of every request's tokens 0..count-1, and which of them the request holds."""
    index = torch.arange(count, device="cuda")
    page = s["table"][:, index // case["block"]].to(torch.int64)
    held = index < s["lens"][:, None]
    return torch.where(held, page * case["block"] + index % case["block"], 0), held


def _plain_attend(case, s):
    r, h, kv, d, block = case["requests"], case["heads"], case["kv_heads"], case["dim"], case["block"]
    slots, held = _plain_slots(case, s, case["context"])
    seen = held
    if case["window"]:
        seen = held & (torch.arange(case["context"], device="cuda") >= s["lens"][:, None] - case["window"])
    k = s["k"][slots // block, slots % block].float().permute(0, 2, 3, 1)  # [r, kv, d, tokens]
    q = s["q"].float().view(r, kv, h // kv, d)
    logits = torch.matmul(q, k) / math.sqrt(d)
    logits = logits.masked_fill_(~seen[:, None, None], -math.inf)
    top = logits.max(-1, keepdim=True).values
    weight = torch.exp(logits - top.clamp(min=-1e30))
    total = weight.sum(-1, keepdim=True)
    weight = weight / total.clamp(min=1e-30)
    v = s["v"][slots // block, slots % block].float().permute(0, 2, 1, 3)  # [r, kv, tokens, d]
    result = {"out": torch.matmul(weight, v).view(r, h, d).to(s["q"].dtype), "lse": (top + total.log()).view(r, h)}
    if case["scored"]:
        slot = torch.where(held, slots, s["scores"].numel() - 1)  # the last slot belongs to nobody
        result["scores"] = s["scores_out"].clone()
        result["scores"][slot] = s["scores"][slot] + weight.sum((1, 2))
        result["scores"] = result["scores"][:-1]
    return result


def _plain_evict(case, s):
    r, block, budget, count = case["requests"], case["block"], case["budget"], case["context"]
    slots, held = _plain_slots(case, s, count)
    lens = s["lens"].to(torch.int64)
    total = (lens + s["evicted"])[:, None]
    position = s["positions"][slots]
    safe = (position < case["first"]) | (position >= total - case["recent"])
    key = torch.where(held, torch.where(safe, math.inf, s["scores"][slots]), -math.inf)
    order = torch.sort(key, dim=1, descending=True, stable=True).indices[:, :budget]
    kept = torch.zeros(r, count, dtype=torch.bool, device="cuda").scatter_(1, order, True)
    over = lens > case["trigger"]
    index = torch.arange(count, device="cuda")
    hole = ~kept & (index < budget) & over[:, None]
    filler = kept & (index >= budget) & over[:, None]
    room = s["moves"].shape[1]
    moves = torch.cat([s["moves"], s["moves"][:, :1]], 1)
    moves[:, :, 0].scatter_(1, torch.where(filler, filler.cumsum(1) - 1, room), slots)
    moves[:, :, 1].scatter_(1, torch.where(hole, hole.cumsum(1) - 1, room), slots)
    new = torch.where(over, budget, lens)
    # pages behind the shortened requests go back to the free list, in the order of the requests
    before, after = (lens + block - 1) // block, (new + block - 1) // block
    freed = before - after
    end = torch.cumsum(freed, 0)
    used = s["used"].to(torch.int64) - end[-1]
    column = torch.arange(s["table"].shape[1], device="cuda")
    gone = (column >= after[:, None]) & (column < before[:, None])
    at = used + (end - freed)[:, None] + column - after[:, None]
    free = torch.cat([s["free"], s["free"][:1]])
    free[torch.where(gone, at, s["free"].numel())] = s["table"]
    return {"lens": new.to(torch.int32), "evicted": (s["evicted"] + lens - new).to(torch.int32),
            "counts": filler.sum(1).to(torch.int32), "moves": moves[:, :room], "free": free[:-1],
            "used": used.to(torch.int32)}


def _plain_move(case, s):
    block = case["block"]
    # entries that hold no move copy the last slot, which belongs to nobody, onto itself
    src, dst = torch.where(s["moves"] < 0, s["pages"] * block - 1, s["moves"]).view(-1, 2).unbind(1)
    s["k"][dst // block, dst % block] = s["k"][src // block, src % block]
    s["v"][dst // block, dst % block] = s["v"][src // block, src % block]
    s["scores"][dst] = s["scores"][src]
    s["positions"][dst] = s["positions"][src]
    return {"k": s["k"], "v": s["v"], "scores": s["scores"], "positions": s["positions"]}


_PLAIN = {"append": _plain_append, "rotary": _plain_rotary, "rotary_grad": _plain_rotary, "attend": _plain_attend,
          "evict": _plain_evict, "move": _plain_move}


# ---------------------------------------------------------------------------
# The library's calls
# ---------------------------------------------------------------------------
def _layout(L, case):
    return L.ROTARY_HALF if case["layout"] == "half" else L.ROTARY_INTERLEAVED


def _own_rotary(case, s):
    L = _lib()
    call = L.DeviceRotary().Forward if case["op"] == "rotary" else L.DeviceRotary().Backward
    call(s["q"], s["k"], s["q_out"], s["k_out"], s["positions"], s["frequencies"], case["tokens"],
         layout=_layout(L, case))
    return {"q": s["q_out"], "k": s["k_out"]}


def _own_append(case, s):
    L = _lib()
    L.DeviceRotary().Append(s["q"], s["k"], s["v"], s["q_out"], s["k_cache"], s["v_cache"], s["slots"], s["positions"],
                            s["frequencies"], case["tokens"], layout=_layout(L, case))
    return {"q": s["q_out"], "k_cache": s["k_cache"][:-1], "v_cache": s["v_cache"][:-1]}


def _own_attend(case, s):
    L = _lib()
    slots = s["pages"] * case["block"] if case["scored"] else 0
    if "temp" not in s:
        s["temp"] = L.alloc_temp(L.DevicePagedAttention.GetTempStorageBytes(case["requests"], case["heads"],
                                                                           case["kv_heads"], case["dim"], slots))
    L.DevicePagedAttention().Decode(s["temp"], s["q"], s["k"], s["v"], s["table"], s["lens"], s["out"],
                                    case["requests"], window=case["window"], d_lse_out=s["lse"],
                                    d_scores=s.get("scores"), d_scores_out=s.get("scores_out"))
    result = {"out": s["out"], "lse": s["lse"]}
    if case["scored"]:
        result["scores"] = s["scores_out"][:-1]
    return result


def _own_evict(case, s):
    L = _lib()
    L.DeviceCacheEviction().Plan(s["lens"], s["table"], s["scores"], s["lens_out"], s["counts"], s["moves"],
                                 case["requests"], case["block"], case["budget"], trigger=case["trigger"],
                                 keep_first=case["first"], keep_recent=case["recent"], d_positions=s["positions"],
                                 d_evicted=s["evicted"], d_evicted_out=s["evicted_out"], d_free_blocks=s["free"],
                                 d_free_used=s["used"], d_free_used_out=s["used_out"])
    return {"lens": s["lens_out"], "evicted": s["evicted_out"], "counts": s["counts"], "moves": s["moves"],
            "free": s["free"], "used": s["used_out"]}


def _own_move(case, s):
    L = _lib()
    L.DeviceCacheEviction().Move(s["moves"], s["counts"], s["k"], s["v"], case["requests"], d_scores=s["scores"],
                                 d_positions=s["positions"])
    return {"k": s["k"], "v": s["v"], "scores": s["scores"], "positions": s["positions"]}


_OWN = {"append": _own_append, "rotary": _own_rotary, "rotary_grad": _own_rotary, "attend": _own_attend,
        "evict": _own_evict, "move": _own_move}


def run(state):
    case = state["case"]
    return (_OWN if own else _PLAIN)[case["op"]](case, state)


# ---------------------------------------------------------------------------
# Work and exact results
# ---------------------------------------------------------------------------
def work(case):
    """Bytes that have to be read and written once and operations that have to be done, in one pass (the number of
    moves by its mean)."""
    if case["op"] in ("append", "rotary", "rotary_grad"):
        t, turned = case["tokens"], case["heads"] + case["kv_heads"]
        rows = turned + (case["kv_heads"] if case["op"] == "append" else 0)
        return {"bytes": 2 * t * rows * case["dim"] * _BYTES[case["dtype"]] + 12 * t,
                "flops": 3 * t * turned * case["rotary"]}
    if case["op"] == "attend":
        ranks = [k for k in range(case["requests"]) if k % 20 != 13]
        tokens = case["context"] * sum(1 - 0.75 * k / case["requests"] for k in ranks)
        if case["window"]:
            tokens = min(tokens, case["window"] * case["requests"])
        rows = 2 * case["requests"] * case["heads"] * case["dim"]
        return {"bytes": int((2 * tokens * case["kv_heads"] * case["dim"] + rows) * _BYTES[case["dtype"]]
                             + 8 * tokens * case["scored"]),
                "flops": int(4 * tokens * case["heads"] * case["dim"])}
    tokens = case["requests"] * max(1, case["context"] - 0.4 * (case["context"] - case["budget"]))
    if case["op"] == "evict":
        moves = case["requests"] * _evict_moves(case) // 2
        return {"bytes": int(8 * tokens + 16 * moves + 8 * tokens / case["block"]), "flops": int(8 * tokens)}
    moves = case["requests"] * case["budget"] * (1 - min(1.0, case["budget"] * case["requests"] / tokens))
    return {"bytes": int(moves * (4 * case["kv_heads"] * case["dim"] * _BYTES[case["dtype"]] + 32)), "flops": 0}


def _exact_turned(case, s, x):
    """Pairs as complex numbers, multiplied by exp(i angle); the gradient by its conjugate."""
    rotary = case["rotary"]
    angle = s["positions"].double()[:, None] * s["frequencies"]
    factor = torch.polar(torch.ones_like(angle), angle if case["op"] != "rotary_grad" else -angle)[:, None]
    x = x.double().clone()
    part = x[..., :rotary].unflatten(-1, (2, -1) if case["layout"] == "half" else (-1, 2))
    if case["layout"] == "half":
        part = part.transpose(-1, -2)
    turned = torch.view_as_real(torch.view_as_complex(part.contiguous()) * factor)
    if case["layout"] == "half":
        turned = turned.transpose(-1, -2)
    x[..., :rotary] = turned.flatten(-2)
    return x


def _exact_append(case, s):
    live, block = (s["slots"] >= 0).nonzero()[:, 0], case["block"]
    q, k, v = s["q_out"].double(), s["k_cache"].double(), s["v_cache"].double()
    q[live] = _exact_turned(case, s, s["q"])[live]
    slot = s["slots"][live]
    k[slot // block, slot % block] = _exact_turned(case, s, s["k"])[live]
    v[slot // block, slot % block] = s["v"][live].double()
    return {"q": q, "k_cache": k[:-1], "v_cache": v[:-1]}


def _exact_attend(case, s):
    r, h, kv, d, block = case["requests"], case["heads"], case["kv_heads"], case["dim"], case["block"]
    out = torch.zeros(r, h, d, dtype=torch.float64, device="cuda")
    lse = torch.full((r, h), -math.inf, dtype=torch.float64, device="cuda")
    scores = s["scores_out"].double() if case["scored"] else None
    for i, n in enumerate(s["lens"].tolist()):
        if not n:
            continue
        pages = s["table"][i, :-(-n // block)].long()
        k, v = (s[x][pages].flatten(0, 1)[:n].double() for x in ("k", "v"))
        first = max(0, n - case["window"]) if case["window"] else 0
        q = s["q"][i].double().view(kv, h // kv, d)
        logits = torch.einsum("kgd,tkd->kgt", q, k[first:]) * d ** -0.5
        lse[i] = torch.logsumexp(logits, -1).flatten()
        share = torch.softmax(logits, -1)
        out[i] = torch.einsum("kgt,tkd->kgd", share, v[first:]).reshape(h, d)
        if case["scored"]:
            slot = (pages[:, None] * block + torch.arange(block, device="cuda")).flatten()[:n]
            scores[slot] = s["scores"][slot].double()
            scores[slot[first:]] += share.sum((0, 1))
    return {"out": out, "lse": lse} | ({"scores": scores[:-1]} if case["scored"] else {})


def _exact_move(case, s):
    block = case["block"]
    k, v, scores = s["k"].double(), s["v"].double(), s["scores"].double()
    for i, n in enumerate(s["counts"].tolist()):
        src, dst = s["moves"][i, :n].unbind(1)
        k[dst // block, dst % block] = s["k"][src // block, src % block].double()
        v[dst // block, dst % block] = s["v"][src // block, src % block].double()
        scores[dst] = s["scores"][src].double()
    return {"k": k, "v": v, "scores": scores, "positions": None}


def exact(case, seed):
    """The results from the definitions in 64 bits; None where all outputs are whole numbers."""
    if case["op"] == "evict":
        return None
    s = prepare(case, seed)
    if case["op"] == "attend":
        return _exact_attend(case, s)
    if case["op"] == "append":
        return _exact_append(case, s)
    if case["op"] == "move":
        return _exact_move(case, s)
    return {"q": _exact_turned(case, s, s["q"]), "k": _exact_turned(case, s, s["k"])}
