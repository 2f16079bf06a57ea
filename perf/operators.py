"""The model-step operators as they are measured: paged block tables, expert routing with its balance loss,
and expert dispatch, each in a plain form of elementary torch operations and as the library's own calls.

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


def _lib():
    package = str(Path(__file__).resolve().parent.parent / "luisacompute-parallelprimitive_b200")
    if package not in sys.path:
        sys.path.insert(0, package)
    import lcpp_b200
    return lcpp_b200


# ---------------------------------------------------------------------------
# Cases
# ---------------------------------------------------------------------------
def listed():
    return [
        # one decode step of a small server: one new token for each of 64 requests
        {"name": "table_decode", "op": "table", "requests": 64, "tokens": 64, "decode": True, "block": 16,
         "context": 8192, "capacity": 64, "short": False},
        # a mixed step: prompts beside decodes and idle requests, a page size that is no power of two, and
        # arrays padded to a captured graph's capacity
        {"name": "table_mixed", "op": "table", "requests": 301, "tokens": 7001, "decode": False, "block": 24,
         "context": 5000, "capacity": 8192, "short": False},
        # a whole cache laid out again after a restart: millions of tokens at once
        {"name": "table_refill", "op": "table", "requests": 6001, "tokens": 4_000_003, "decode": False, "block": 64,
         "context": 1, "capacity": 4_194_304, "short": False},
        # routing of one decode step
        {"name": "route_decode", "op": "route", "tokens": 16, "experts": 128, "top_k": 8, "dtype": "bf16",
         "score": "softmax", "renormalize": True, "bias": False, "masked": False},
        # a prompt chunk, sigmoid scores with a selection bias, an expert count that is no power of two,
        # padding tokens left out
        {"name": "route_bias", "op": "route", "tokens": 4099, "experts": 160, "top_k": 6, "dtype": "f32",
         "score": "sigmoid", "renormalize": True, "bias": True, "masked": True},
        # a training batch
        {"name": "route_train", "op": "route", "tokens": 131072, "experts": 256, "top_k": 8, "dtype": "bf16",
         "score": "softmax", "renormalize": True, "bias": False, "masked": False},
        # the router's gradient for a short ragged batch
        {"name": "route_grad_odd", "op": "route_grad", "tokens": 3001, "experts": 60, "top_k": 4, "dtype": "f16",
         "score": "softmax", "renormalize": False, "bias": False, "masked": True},
        # the router's gradient for a training batch
        {"name": "route_grad_train", "op": "route_grad", "tokens": 131072, "experts": 256, "top_k": 8,
         "dtype": "bf16", "score": "sigmoid", "renormalize": True, "bias": True, "masked": False},
        # grouping and moving the rows of one decode step
        {"name": "dispatch_decode", "op": "dispatch", "tokens": 16, "experts": 128, "top_k": 8, "hidden": 4096,
         "dtype": "bf16", "align": 16, "masked": False},
        # grouping and moving the rows of a training batch, segments aligned to a product's row tile
        {"name": "dispatch_train", "op": "dispatch", "tokens": 16384, "experts": 256, "top_k": 8, "hidden": 4096,
         "dtype": "bf16", "align": 128, "masked": False},
        # the experts' rows summed back for a prompt chunk
        {"name": "combine_prompt", "op": "combine", "tokens": 8191, "experts": 64, "top_k": 6, "hidden": 2880,
         "dtype": "bf16", "align": 64, "masked": True},
        # the gradient of that sum for a training batch
        {"name": "combine_grad_train", "op": "combine_grad", "tokens": 16384, "experts": 256, "top_k": 8,
         "hidden": 4096, "dtype": "bf16", "align": 128, "masked": False},
    ]


def _log_int(rng, low, high):
    return max(low, min(high, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng):
    op = rng.choice(["table", "route", "route_grad", "dispatch", "combine", "combine_grad"])
    if op == "table":
        decode = rng.random() < 0.3
        requests = _log_int(rng, 1, 8000)
        tokens = requests if decode else _log_int(rng, max(8, requests // 2), 4_000_000)
        capacity = tokens + rng.choice([0, 0, rng.randint(1, 1 + tokens // 8)])
        block = rng.choice([1, 8, 16, 24, 32, 64, 128])
        context = _log_int(rng, 1, max(1, min(32768, 4_000_000 * block // requests)))
        return {"op": op, "requests": requests, "tokens": tokens, "decode": decode, "block": block,
                "context": context, "capacity": capacity, "short": rng.random() < 0.2}
    experts = _log_int(rng, 2, 512) if rng.random() < 0.5 else 2 ** rng.randint(3, 9)
    top_k = min(experts, rng.choice([1, 2, 4, 6, 8, 8, 10]))
    dtype = rng.choice(["f32", "bf16", "bf16", "f16"])
    masked = rng.random() < 0.5
    if op in ("route", "route_grad"):
        tokens = _log_int(rng, 1, min(400_000, 131072 * 512 // (experts * _BYTES[dtype])))
        score = rng.choice(["softmax", "sigmoid"])
        return {"op": op, "tokens": tokens, "experts": experts, "top_k": top_k, "dtype": dtype, "score": score,
                "renormalize": rng.random() < 0.7, "bias": rng.random() < 0.5, "masked": masked}
    hidden = _log_int(rng, 64, 8192)
    if rng.random() < 0.67:
        hidden = max(64, hidden // 8 * 8)
    align = rng.choice([1, 16, 64, 128])
    budget = 16384 * 8 * 4096 * 2 // (top_k * hidden * _BYTES[dtype])
    tokens = _log_int(rng, 1, max(1, min(65536, budget - experts * align // top_k)))
    return {"op": op, "tokens": tokens, "experts": experts, "top_k": top_k, "hidden": hidden, "dtype": dtype,
            "align": align, "masked": masked}


def _max_rows(case):
    pairs = case["tokens"] * case["top_k"]
    return pairs + min(case["experts"], pairs) * (case["align"] - 1)


def _table_width(case):
    """Columns of the block table: every request may grow to its context and a share of the new tokens."""
    longest = case["context"] + (1 if case["decode"] else 4 * case["tokens"] // case["requests"] + 64)
    return -(-longest // case["block"]) + 1


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------
def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed * 7919 + 17)


def _rand(g, *shape):
    return torch.rand(*shape, device="cuda", generator=g)


def _randn(g, *shape):
    return torch.randn(*shape, device="cuda", generator=g)


def _logits(g, case):
    """Router logits: unit noise on top of experts that differ in popularity."""
    popular = _randn(g, case["experts"]) * 0.7
    x = _randn(g, case["tokens"], case["experts"]) * 1.5 + popular
    return x.to(_DTYPES[case["dtype"]])


def _token_mask(g, case):
    """Request of each token; about one token in ten is padding where the case has a mask."""
    request = torch.arange(case["tokens"], device="cuda", dtype=torch.int32) // 7
    if not case["masked"]:
        return None
    return torch.where(_rand(g, case["tokens"]) < 0.1, torch.full_like(request, -1), request)


def _choices(g, case):
    """k different experts for each token (popular ones more often), -1 for padding tokens."""
    key = _rand(g, case["tokens"], case["experts"]).log().neg().log().neg() + _randn(g, case["experts"]) * 0.7
    experts = torch.topk(key, case["top_k"], dim=1).indices.to(torch.int32)
    mask = _token_mask(g, case)
    if mask is not None:
        experts = torch.where((mask < 0)[:, None], torch.full_like(experts, -1), experts)
    return experts.contiguous()


def _prepare_table(case, g):
    r, block, width = case["requests"], case["block"], _table_width(case)
    context = (_rand(g, r) ** 2 * case["context"]).to(torch.int32)
    if case["decode"]:
        new, total = None, torch.ones(r, device="cuda", dtype=torch.int64)
    else:
        # a third one token each, some idle, the rest prompts that share the tokens
        kind, share = _rand(g, r), _rand(g, r) ** 2
        share = torch.where(kind < 0.4, torch.zeros_like(share), share + 1e-6)
        budget = max(0, case["tokens"] - r)
        prompt = (share.double() / share.double().sum().clamp_min(1e-6) * budget).to(torch.int32)
        new = torch.where(kind < 0.07, torch.zeros_like(prompt), prompt + 1)
        total = new.to(torch.int64)
    context64 = context.to(torch.int64)
    need = (context64 + total + block - 1) // block - (context64 + block - 1) // block
    pages = int(need.sum())
    free = pages * 3 // 4 if case["short"] else pages + 5
    held = r * width
    order = torch.randperm(held + free + 8, device="cuda", generator=g).to(torch.int32)
    table = order[:held].view(r, width).contiguous()
    used = torch.full((1,), 3, dtype=torch.int32, device="cuda")
    i32 = {"dtype": torch.int32, "device": "cuda"}
    return {"context": context, "new": new, "table": table, "free": order[held:held + free + 3].contiguous(),
            "used": used, "used_out": torch.zeros(1, **i32), "seq_lens": torch.zeros(r, **i32),
            "starts": torch.zeros(r + 1, **i32),
            "slots": torch.zeros(case["capacity"], dtype=torch.int64, device="cuda"),
            "positions": torch.zeros(case["capacity"], **i32), "requests": torch.zeros(case["capacity"], **i32)}


def _prepare_route(case, g):
    t, e, k = case["tokens"], case["experts"], case["top_k"]
    i32, f32 = {"dtype": torch.int32, "device": "cuda"}, {"dtype": torch.float32, "device": "cuda"}
    state = {"logits": _logits(g, case), "mask": _token_mask(g, case),
             "bias": _randn(g, e) * 0.3 if case["bias"] else None}
    if case["op"] == "route":
        return state | {"weights": torch.zeros(t, k, **f32), "experts": torch.zeros(t, k, **i32),
                        "counts": torch.zeros(e, **i32), "routed": torch.zeros(1, **i32), "loss": torch.zeros(1, **f32)}
    chosen = _plain_route(case, state)
    return state | {"experts": chosen["experts"], "counts": chosen["counts"], "routed": chosen["routed"],
                    "grad_weights": _randn(g, t, k) * 0.02, "grad_loss": torch.full((1,), 1.5, **f32),
                    "grad_logits": torch.zeros_like(state["logits"])}


def _prepare_rows(case, g):
    t, k, h, dt = case["tokens"], case["top_k"], case["hidden"], _DTYPES[case["dtype"]]
    rows = _max_rows(case)
    i32 = {"dtype": torch.int32, "device": "cuda"}
    state = {"experts": _choices(g, case)}
    if case["op"] == "dispatch":
        return state | {"x": _randn(g, t, h).to(dt), "expert_starts": torch.zeros(case["experts"] + 1, **i32),
                        "row_of": torch.zeros(t, k, **i32), "pair_of": torch.zeros(rows, **i32),
                        "rows": torch.zeros(rows, h, dtype=dt, device="cuda")}
    state |= _plain_plan(case, state["experts"])
    weights = _rand(g, t, k) + 0.05
    state["weights"] = weights / weights.sum(1, keepdim=True)
    # what the experts gave; rows that belong to no pair hold zeros
    y = _randn(g, rows, h).to(dt)
    state["rows"] = y.masked_fill_((state["pair_of"] < 0)[:, None], 0)
    if case["op"] == "combine":
        return state | {"out": torch.zeros(t, h, dtype=dt, device="cuda")}
    return state | {"grad_out": _randn(g, t, h).to(dt), "grad_rows": torch.zeros(rows, h, dtype=dt, device="cuda"),
                    "grad_weights": torch.zeros(t, k, dtype=torch.float32, device="cuda")}


def prepare(case, seed):
    g = _generator(seed)
    if case["op"] == "table":
        state = _prepare_table(case, g)
    elif case["op"] in ("route", "route_grad"):
        state = _prepare_route(case, g)
    else:
        state = _prepare_rows(case, g)
    return {"case": case, **state}


# ---------------------------------------------------------------------------
# Plain forms
# ---------------------------------------------------------------------------
def _plain_table(case, s):
    r, block, width, capacity = case["requests"], case["block"], s["table"].shape[1], case["capacity"]
    context = s["context"].to(torch.int64)
    new = torch.ones_like(context) if s["new"] is None else s["new"].to(torch.int64)
    held, total = (context + block - 1) // block, (context + new + block - 1) // block
    in_row = total <= width
    need = torch.where(in_row, total - held, 0)
    token_end, page_end = torch.cumsum(new, 0), torch.cumsum(need, 0)
    token_start, page_start = token_end - new, page_end - need
    used = s["used"].to(torch.int64)
    fits = in_row & (token_end <= capacity) & ((need == 0) | (used + page_end <= s["free"].numel()))
    used_out = used + torch.where(fits & (need > 0), page_end, 0).max()
    # each token's request, position and page
    token = torch.arange(capacity, device="cuda")
    request = torch.searchsorted(token_end, token, right=True)
    inside = request < r
    request = request.clamp(max=r - 1)
    inside &= fits[request]
    position = context[request] + token - token_start[request]
    page = position // block
    taken = (used + page_start[request] + page - held[request]).clamp(0, s["free"].numel() - 1)
    page_id = torch.where(page >= held[request], s["free"][taken], s["table"][request, page.clamp(0, width - 1)])
    slot = page_id.to(torch.int64) * block + position % block
    # the table with its new pages
    column = torch.arange(width, device="cuda")
    fresh = fits[:, None] & (column >= held[:, None]) & (column < total[:, None])
    index = (used + page_start[:, None] + column - held[:, None]).clamp(0, s["free"].numel() - 1)
    return {"table": torch.where(fresh, s["free"][index], s["table"]), "slots": torch.where(inside, slot, -1),
            "positions": torch.where(inside, position, 0).to(torch.int32),
            "requests": torch.where(inside, request, -1).to(torch.int32),
            "starts": torch.cat([torch.zeros_like(token_end[:1]), token_end]).to(torch.int32),
            "seq_lens": torch.where(fits, context + new, context).to(torch.int32), "used": used_out.to(torch.int32)}


_LOSS_COEF, _WEIGHT_SCALE = 0.01, 2.5


def _plain_scores(case, x):
    """Scores, the scores as shares of their row's sum, and the slope factor of either form."""
    if case["score"] == "softmax":
        shifted = torch.exp(x - x.max(1, keepdim=True).values)
        share = shifted / shifted.sum(1, keepdim=True)
        return share, share, torch.ones_like(share)
    score = 1 / (1 + torch.exp(-x))
    return score, score / score.sum(1, keepdim=True), 1 - score


def _plain_route(case, s):
    x, k, e = s["logits"].float(), case["top_k"], case["experts"]
    score, share, _ = _plain_scores(case, x)
    key = x if s["bias"] is None else x + s["bias"]
    chosen = torch.sort(key, dim=1, descending=True, stable=True).indices[:, :k]
    weights = torch.gather(score, 1, chosen)
    if case["renormalize"]:
        weights = weights / weights.sum(1, keepdim=True)
    weights = weights * _WEIGHT_SCALE
    live = torch.ones(x.shape[0], dtype=torch.bool, device="cuda") if s["mask"] is None else s["mask"] >= 0
    routed = live.sum()
    counts = torch.zeros(e, dtype=torch.int64, device="cuda")
    counts.scatter_add_(0, chosen.reshape(-1), live[:, None].expand(-1, k).reshape(-1).to(torch.int64))
    tokens = routed.clamp(min=1).float()
    balance = ((share * live[:, None]).sum(0) / tokens * (counts.float() / (k * tokens))).sum()
    return {"weights": torch.where(live[:, None], weights, 0), "experts": torch.where(live[:, None], chosen, -1).to(torch.int32),
            "counts": counts.to(torch.int32), "routed": routed.reshape(1).to(torch.int32),
            "loss": (_LOSS_COEF * e * balance).reshape(1)}


def _plain_route_grad(case, s):
    x, k, e = s["logits"].float(), case["top_k"], case["experts"]
    score, share, slope = _plain_scores(case, x)
    live = s["experts"][:, :1] >= 0
    chosen = s["experts"].clamp(min=0).to(torch.int64)
    tokens = s["routed"].clamp(min=1).float()
    pull = s["grad_loss"] * (_LOSS_COEF * e) * s["counts"].float() / (k * tokens * tokens)
    grad = share * (pull - (share * pull).sum(1, keepdim=True))
    picked, g = torch.gather(score, 1, chosen), s["grad_weights"]
    if case["renormalize"]:
        part = picked / picked.sum(1, keepdim=True)
        grad.scatter_add_(1, chosen, _WEIGHT_SCALE * part * (g - (g * part).sum(1, keepdim=True)))
    else:
        grad.scatter_add_(1, chosen, _WEIGHT_SCALE * picked * g)
        if case["score"] == "softmax":
            grad = grad - score * (_WEIGHT_SCALE * (g * picked).sum(1, keepdim=True))
    return {"grad_logits": torch.where(live, grad * slope, 0).to(s["logits"].dtype)}


def _plain_plan(case, experts):
    e, align, rows = case["experts"], case["align"], _max_rows(case)
    key = experts.reshape(-1).to(torch.int64)
    key = torch.where(key < 0, e, key)
    order = torch.sort(key, stable=True).indices
    counts = torch.zeros(e + 1, dtype=torch.int64, device="cuda").scatter_add_(0, key, torch.ones_like(key))
    padded = (counts[:e] + align - 1) // align * align
    starts = torch.cat([torch.zeros_like(padded[:1]), torch.cumsum(padded, 0)])
    sorted_key = key[order]
    rank = torch.arange(key.numel(), device="cuda") - (torch.cumsum(counts, 0) - counts)[sorted_key]
    row = torch.where(sorted_key < e, starts[sorted_key] + rank, rows)
    row_of = torch.empty_like(key).scatter_(0, order, torch.where(row < rows, row, -1))
    pair_of = torch.full((rows + 1,), -1, dtype=torch.int64, device="cuda").scatter_(0, row, order)[:rows]
    return {"expert_starts": starts.to(torch.int32), "row_of": row_of.view(experts.shape).to(torch.int32),
            "pair_of": pair_of.to(torch.int32)}


def _plain_dispatch(case, s):
    plan = _plain_plan(case, s["experts"])
    token = plan["pair_of"].clamp(min=0).to(torch.int64) // case["top_k"]
    rows = s["x"][token].masked_fill_((plan["pair_of"] < 0)[:, None], 0)
    return {**plan, "rows": rows}


def _plain_combine(case, s):
    index, live = s["row_of"].clamp(min=0).to(torch.int64), s["row_of"] >= 0
    rows = s["rows"][index].float().masked_fill_(~live[:, :, None], 0)
    return {"out": (rows * s["weights"][:, :, None]).sum(1).to(s["rows"].dtype)}


def _plain_combine_grad(case, s):
    index, live = s["row_of"].clamp(min=0).to(torch.int64), s["row_of"] >= 0
    grad_weights = (s["rows"][index].float() * s["grad_out"].float()[:, None, :]).sum(2).masked_fill_(~live, 0)
    pair, filled = s["pair_of"].clamp(min=0).to(torch.int64), s["pair_of"] >= 0
    grad_rows = s["grad_out"][pair // case["top_k"]].float() * s["weights"].reshape(-1)[pair][:, None]
    return {"grad_rows": grad_rows.masked_fill_(~filled[:, None], 0).to(s["rows"].dtype), "grad_weights": grad_weights}


_PLAIN = {"table": _plain_table, "route": _plain_route, "route_grad": _plain_route_grad, "dispatch": _plain_dispatch,
          "combine": _plain_combine, "combine_grad": _plain_combine_grad}


# ---------------------------------------------------------------------------
# The library's calls
# ---------------------------------------------------------------------------
def _own_table(case, s):
    L = _lib()
    if "temp" not in s:
        s["temp"] = L.alloc_temp(L.DeviceBlockTable.GetTempStorageBytes(case["requests"], case["capacity"]))
    L.DeviceBlockTable().Extend(s["temp"], s["context"], s["new"], s["table"], s["free"], s["used"], s["used_out"],
                                s["seq_lens"], s["starts"], s["slots"], s["positions"], s["requests"],
                                case["requests"], case["block"])
    return {"table": s["table"], "slots": s["slots"], "positions": s["positions"], "requests": s["requests"],
            "starts": s["starts"], "seq_lens": s["seq_lens"], "used": s["used_out"]}


def _options(L, case):
    return {"score": L.SCORE_SOFTMAX if case["score"] == "softmax" else L.SCORE_SIGMOID,
            "renormalize": case["renormalize"], "weight_scale": _WEIGHT_SCALE, "loss_coef": _LOSS_COEF}


def _own_route(case, s):
    L = _lib()
    if "temp" not in s:
        s["temp"] = L.alloc_temp(L.DeviceRouter.GetTempStorageBytes(case["tokens"], case["experts"]))
    L.DeviceRouter().Forward(s["temp"], s["logits"], s["weights"], s["experts"], s["counts"], s["routed"], s["loss"],
                             case["tokens"], case["experts"], case["top_k"], d_bias=s["bias"],
                             d_token_request=s["mask"], **_options(L, case))
    return {"weights": s["weights"], "experts": s["experts"], "counts": s["counts"], "routed": s["routed"],
            "loss": s["loss"]}


def _own_route_grad(case, s):
    L = _lib()
    L.DeviceRouter().Backward(s["logits"], s["experts"], s["counts"], s["routed"], s["grad_weights"], s["grad_loss"],
                              s["grad_logits"], case["tokens"], case["experts"], case["top_k"], **_options(L, case))
    return {"grad_logits": s["grad_logits"]}


def _own_dispatch(case, s):
    L = _lib()
    t, k, e = case["tokens"], case["top_k"], case["experts"]
    if "temp" not in s:
        s["temp"] = L.alloc_temp(L.DeviceDispatch.GetTempStorageBytes(t, k, e))
    d = L.DeviceDispatch()
    d.Plan(s["temp"], s["experts"], s["expert_starts"], s["row_of"], s["pair_of"], t, k, e, case["align"])
    d.Gather(s["x"], s["row_of"], s["pair_of"], s["expert_starts"], s["rows"], t, k, e)
    return {"expert_starts": s["expert_starts"], "row_of": s["row_of"], "pair_of": s["pair_of"], "rows": s["rows"]}


def _own_combine(case, s):
    L = _lib()
    L.DeviceDispatch().Combine(s["rows"], s["row_of"], s["weights"], s["out"], case["tokens"], case["top_k"])
    return {"out": s["out"]}


def _own_combine_grad(case, s):
    L = _lib()
    L.DeviceDispatch().CombineBackward(s["grad_out"], s["rows"], s["row_of"], s["pair_of"], s["expert_starts"],
                                       s["weights"], s["grad_rows"], s["grad_weights"], case["tokens"],
                                       case["top_k"], case["experts"])
    return {"grad_rows": s["grad_rows"], "grad_weights": s["grad_weights"]}


_OWN = {"table": _own_table, "route": _own_route, "route_grad": _own_route_grad, "dispatch": _own_dispatch,
        "combine": _own_combine, "combine_grad": _own_combine_grad}


def run(state):
    case = state["case"]
    return (_OWN if own else _PLAIN)[case["op"]](case, state)


# ---------------------------------------------------------------------------
# Work and exact results
# ---------------------------------------------------------------------------
def work(case):
    """Bytes that have to be read and written once and operations that have to be done, in one pass."""
    if case["op"] == "table":
        r, pages = case["requests"], case["tokens"] // case["block"] + case["requests"] // 2
        return {"bytes": 16 * r + 16 * case["capacity"] + 8 * pages, "flops": 8 * case["capacity"]}
    t, e, k = case["tokens"], case["experts"], case["top_k"]
    size, pairs = _BYTES[case["dtype"]], t * k
    if case["op"] == "route":
        return {"bytes": t * e * size + 8 * pairs + 8 * e + 4 * t * case["masked"], "flops": 6 * t * e}
    if case["op"] == "route_grad":
        return {"bytes": 2 * t * e * size + 8 * pairs + 4 * e, "flops": 8 * t * e}
    h = case["hidden"]
    if case["op"] == "dispatch":
        return {"bytes": (t + pairs) * h * size + 12 * pairs + 4 * e, "flops": pairs}
    if case["op"] == "combine":
        return {"bytes": (t + pairs) * h * size + 8 * pairs, "flops": 2 * pairs * h}
    return {"bytes": (t + 2 * pairs) * h * size + 12 * pairs, "flops": 3 * pairs * h}


def _exact_choice(key, k):
    """The k largest of each row by (value, lower index first), through unique 64-bit integers."""
    bits = (key + 0.0).contiguous().view(torch.int32).to(torch.int64)  # + 0.0: both zeros alike
    ordered = torch.where(bits < 0, -(bits & 0x7FFFFFFF), bits)
    index = torch.arange(key.shape[1] - 1, -1, -1, device=key.device)
    top = torch.topk(ordered * 4096 + index, k, dim=1).values
    return key.shape[1] - 1 - (top & 4095)


def _exact_log_scores(case, x):
    if case["score"] == "softmax":
        return torch.log_softmax(x, 1)
    return torch.nn.functional.logsigmoid(x)


def _exact_route(case, s):
    e, k = case["experts"], case["top_k"]
    x32 = s["logits"].float()
    chosen = _exact_choice(x32 if s["bias"] is None else x32 + s["bias"], k)
    log_score = _exact_log_scores(case, x32.double())
    picked = torch.gather(log_score, 1, chosen)
    weights = _WEIGHT_SCALE * (torch.softmax(picked, 1) if case["renormalize"] else picked.exp())
    live = torch.ones(case["tokens"], device="cuda").double() if s["mask"] is None else (s["mask"] >= 0).double()
    n = max(1.0, float(live.sum()))
    share = (torch.softmax(log_score, 1) * live[:, None]).sum(0) / n
    one_hot = torch.zeros(e, dtype=torch.float64, device="cuda")
    for j in range(k):
        one_hot.index_add_(0, chosen[:, j], live)
    loss = _LOSS_COEF * e * (share * one_hot / (k * n)).sum()
    return {"weights": weights * live[:, None], "experts": None, "counts": None, "routed": None, "loss": loss.reshape(1)}


def _exact_route_grad(case, s):
    e, k = case["experts"], case["top_k"]
    x = s["logits"].double().requires_grad_(True)
    live = (s["experts"][:, 0] >= 0).double()[:, None]
    chosen = s["experts"].clamp(min=0).long()
    n = max(1.0, float(s["routed"]))
    log_score = _exact_log_scores(case, x)
    picked = torch.gather(log_score, 1, chosen)
    weights = _WEIGHT_SCALE * (torch.softmax(picked, 1) if case["renormalize"] else picked.exp())
    share = (torch.softmax(log_score, 1) * live).sum(0) / n
    loss = _LOSS_COEF * e * (share * s["counts"].double() / (k * n)).sum()
    total = (weights * live * s["grad_weights"].double()).sum() + loss * s["grad_loss"].double()[0]
    return {"grad_logits": torch.autograd.grad(total, x)[0]}


def _exact_dispatch(case, s):
    rows = torch.zeros(s["rows"].shape, dtype=torch.float64, device="cuda")
    start = 0
    for expert in range(case["experts"]):
        token = (s["experts"] == expert).nonzero()[:, 0]  # in the order of the pairs
        rows[start:start + token.numel()] = s["x"][token].double()
        start += -(-token.numel() // case["align"]) * case["align"]
    return {"expert_starts": None, "row_of": None, "pair_of": None, "rows": rows}


def _exact_combine(case, s):
    out = torch.zeros(case["tokens"], case["hidden"], dtype=torch.float64, device="cuda")
    for j in range(case["top_k"]):
        row = s["row_of"][:, j].long()
        live = (row >= 0).nonzero()[:, 0]
        out[live] += s["weights"][live, j].double()[:, None] * s["rows"][row[live]].double()
    return {"out": out}


def _exact_combine_grad(case, s):
    grad_rows = torch.zeros(s["rows"].shape, dtype=torch.float64, device="cuda")
    grad_weights = torch.zeros(case["tokens"], case["top_k"], dtype=torch.float64, device="cuda")
    for j in range(case["top_k"]):
        row = s["row_of"][:, j].long()
        live = (row >= 0).nonzero()[:, 0]
        dy = s["grad_out"][live].double()
        grad_rows[row[live]] = s["weights"][live, j].double()[:, None] * dy
        grad_weights[live, j] = torch.einsum("th,th->t", dy, s["rows"][row[live]].double())
    return {"grad_rows": grad_rows, "grad_weights": grad_weights}


_EXACT = {"route": _exact_route, "route_grad": _exact_route_grad, "dispatch": _exact_dispatch,
          "combine": _exact_combine, "combine_grad": _exact_combine_grad}


def exact(case, seed):
    """The results from the definitions in 64 bits; None where all outputs are whole numbers."""
    if case["op"] not in _EXACT:
        return None
    return _EXACT[case["op"]](case, prepare(case, seed))
