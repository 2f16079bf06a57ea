"""DeviceBlockTable, DeviceRouter and DeviceDispatch against 64-bit references (tests/model_step_ref.py).

Tolerances.  Whole numbers and moved rows are exact.  A weight is a quotient of sums of at most 1024
exponentials; each exponential is off by at most about 2^-22 plus 2^-24 |argument|, with |argument| < 40
where it counts, so 1e-5 relative holds with room (tiny ones: 1e-9 absolute, far below any other).  The
loss adds values of one sign: 1e-5 too.  A gradient of a row adds terms as large as the row's largest
entry: 2e-5 of that entry, plus half a unit in the last place of the logits' type (2^-8 of the value covers
bfloat16, 2^-10 half with its 2^-24 steps near zero).  A combined row adds top_k products: 1e-5 of the sum
of their magnitudes plus the same rounding."""
from __future__ import annotations

import numpy as np
import pytest

import model_step_ref as ref

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
ROUND = {"f32": (0.0, 0.0), "f16": (2.0 ** -10, 2.0 ** -24), "bf16": (2.0 ** -8, 0.0)}


def cuda(a, dtype=None):
    t = torch.from_numpy(np.ascontiguousarray(a)).cuda()
    return t if dtype is None else t.to(dtype)


def i32(*shape, fill=-77):
    return torch.full(shape, fill, dtype=torch.int32, device="cuda")


def host(t):
    return t.detach().cpu().numpy()


def host64(t):
    return t.detach().double().cpu().numpy()


# ---------------------------------------------------------------------------
# DeviceBlockTable
# ---------------------------------------------------------------------------
def run_extend(L, context, new, table, width, free, used, tokens, block, optional=True):
    n = len(context)
    d_table = cuda(table)
    out = {"used": i32(1), "seq": i32(max(n, 1)), "starts": i32(n + 1),
           "slots": torch.full((tokens,), -9, dtype=torch.int64, device="cuda")}
    positions, requests = (i32(tokens), i32(tokens)) if optional else (None, None)
    temp = L.alloc_temp(L.DeviceBlockTable.GetTempStorageBytes(n, tokens))
    L.DeviceBlockTable().Extend(temp, cuda(context), None if new is None else cuda(new), d_table[:, :width],
                                cuda(free), None if used is None else cuda(np.array([used], np.int32)), out["used"],
                                out["seq"], out["starts"], out["slots"], positions, requests, n, block)
    assert L.device_status(temp) == L.OK
    return d_table, out, positions, requests


def check_extend(L, context, new, table, width, free, used, tokens, block, optional=True):
    d_table, out, positions, requests = run_extend(L, context, new, table, width, free, used, tokens, block, optional)
    et, es, ep, er, estarts, eseq, eused = ref.extend(context, new, table, width, free, used or 0, tokens, block)
    np.testing.assert_array_equal(host(d_table), et)
    np.testing.assert_array_equal(host(out["slots"]), es)
    np.testing.assert_array_equal(host(out["starts"]), estarts)
    np.testing.assert_array_equal(host(out["seq"])[:len(context)], eseq)
    assert int(out["used"]) == eused
    if optional:
        np.testing.assert_array_equal(host(positions), ep)
        np.testing.assert_array_equal(host(requests), er)


def lengths(rng, n, most_context, most_new):
    context = rng.integers(0, most_context + 1, n).astype(np.int32)
    new = np.where(rng.random(n) < 0.3, 1, rng.integers(0, most_new + 1, n)).astype(np.int32)
    new[rng.random(n) < 0.15] = 0
    return context, new


# around one thread per request (512), two (1024) and the largest single launch (4096)
@pytest.mark.parametrize("n", [1, 2, 33, 511, 512, 513, 1024, 1025, 4095, 4096, 4097, 9001])
@pytest.mark.parametrize("block", [1, 16, 24])
def test_extend_mixed(lcpp, n, block):
    rng = np.random.default_rng(n * 100 + block)
    context, new = lengths(rng, n, 40, 9 if n > 100 else 300)
    width = 700 // block + 2
    table = rng.permutation(n * width).astype(np.int32).reshape(n, width)
    free = (n * width + rng.permutation(n * 320)).astype(np.int32)
    tokens = int(new.sum()) + int(rng.integers(0, 70))
    check_extend(lcpp, context, new, table, width, free, 5, tokens, block)


@pytest.mark.parametrize("n", [1, 64, 5000])
def test_extend_one_token_each(lcpp, n):
    """The decode step: no array of new lengths, optional outputs left out, no counter of used pages."""
    rng = np.random.default_rng(n)
    context = rng.integers(0, 100, n).astype(np.int32)
    table = rng.permutation(n * 8).astype(np.int32).reshape(n, 8)
    free = (n * 8 + rng.permutation(n)).astype(np.int32)
    check_extend(lcpp, context, None, table, 8, free, None, n, 16, optional=False)


@pytest.mark.parametrize("n,block", [(3, 2), (3, 4), (3, 24), (700, 24), (4000, 64), (5000, 24)])
@pytest.mark.parametrize("offset", [0, 1])
def test_extend_many_tokens(lcpp, n, block, offset):
    """Enough tokens for four to a thread, in arrays that start on a vector boundary or off it: long prompts,
    single tokens and idle requests side by side."""
    rng = np.random.default_rng(n)
    context, new = rng.integers(0, 50, n).astype(np.int32), np.ones(n, np.int32)
    new[rng.random(n) < 0.2] = 0
    long = rng.choice(n, 3, replace=False)
    new[long] = rng.integers(100_000, 130_000, 3)
    width, held = 130_100 // block + 1, 50 // block + 1
    table = rng.permutation(n * held).astype(np.int32).reshape(n, held)
    table = np.concatenate([table, np.full((n, width - held), -1, np.int32)], 1)
    free = (n * held + rng.permutation(400_000 // block + n)).astype(np.int32)
    tokens = int(new.sum()) + 13
    expect = ref.extend(context, new, table, width, free, 0, tokens, block)
    slots = torch.full((tokens + offset,), -9, dtype=torch.int64, device="cuda")[offset:]
    positions, requests = i32(tokens + offset)[offset:], i32(tokens + offset)[offset:]
    d_table, starts, seq, used = cuda(table), i32(n + 1), i32(n), i32(1)
    temp = lcpp.alloc_temp(lcpp.DeviceBlockTable.GetTempStorageBytes(n, tokens))
    lcpp.DeviceBlockTable().Extend(temp, cuda(context), cuda(new), d_table, cuda(free), None, used, seq, starts, slots,
                                   positions, requests, n, block)
    for got, want in zip((d_table, slots, positions, requests, starts, seq, used), expect):
        np.testing.assert_array_equal(host(got), want)


@pytest.mark.parametrize("n,seed", [(40, 0), (40, 1), (700, 2), (6000, 3)])
def test_extend_refuses(lcpp, n, seed):
    """Free pages that end early, rows that are too narrow, arrays that are too short: what does not fit
    takes nothing and is marked, later requests without need of a page are served."""
    rng = np.random.default_rng(seed)
    context, new = lengths(rng, n, 60, 60)
    context[rng.random(n) < 0.1] = 500  # past the row
    width, block = 8, 16
    table = rng.permutation(n * width).astype(np.int32).reshape(n, width)
    need = int(np.maximum(-(-(context + new) // block) - -(-context // block), 0).sum())
    free = (n * width + rng.permutation(max(need // 2, 1))).astype(np.int32)
    check_extend(lcpp, context, new, table, width, free, 2, int(new.sum() * 3 // 4), block)
    check_extend(lcpp, context, new, table, width, free[:0], 0, int(new.sum()), block)


def test_extend_strided_negative_and_large_ids(lcpp):
    """A table that is a part of wider rows, negative lengths (zero), a negative page id (slot -1), page ids
    whose slots pass 32 bits, and a used counter past the free list."""
    rng = np.random.default_rng(11)
    context = np.array([-5, 30, 17, 0, 64], np.int32)
    new = np.array([3, -2, 20, 1, 5], np.int32)
    table = rng.permutation(5 * 20).astype(np.int32).reshape(5, 20) + 2_000_000_000
    table[2, 1] = -1
    free = np.arange(2_100_000_000, 2_100_000_010, dtype=np.int32)
    check_extend(lcpp, context, new, table, 9, free, 1, 40, 16)
    check_extend(lcpp, context, new, table, 9, free, 1000, 40, 16)


def test_extend_longest_sequences(lcpp):
    """Lengths around 2^31 - 1: sums that pass 32 bits, sequences that are too long."""
    top = 2 ** 31 - 1
    context = np.array([top - 3, top - 3, top, 5], np.int32)
    new = np.array([3, 4, 0, 2], np.int32)
    block = 1 << 30
    table = np.arange(12, dtype=np.int32).reshape(4, 3)
    check_extend(lcpp, context, new, table, 3, np.arange(100, 104, dtype=np.int32), 0, 16, block)
    context = np.zeros(6, np.int32)
    new = np.array([4, top, top, top, 0, 1], np.int32)
    check_extend(lcpp, context, new, np.zeros((6, 2), np.int32), 2, np.arange(9, dtype=np.int32), 0, 16, 64)


@pytest.mark.parametrize("n", [7, 5000])
def test_extend_step_after_step(lcpp, n):
    """A captured decode step on another stream, replayed: the lengths and the used counter of one step are the
    next one's inputs, no page is given twice, and every position of a request keeps its slot."""
    rng = np.random.default_rng(n)
    block, width, steps = 4, 40, 20
    context = rng.integers(0, 60, n).astype(np.int32)
    held = -(-context // block)
    pages = rng.permutation(n * width + 3).astype(np.int32)
    table = np.full((n, width), -1, np.int32)
    given = 0
    for r in range(n):
        table[r, :held[r]] = pages[given:given + held[r]]
        given += held[r]
    free = pages[given:]
    d_table, lens, d_free = cuda(table), [cuda(context), i32(n)], cuda(free)
    used, starts = [i32(1, fill=0), i32(1)], i32(n + 1)
    slots = torch.full((n + 5,), -9, dtype=torch.int64, device="cuda")
    temp = lcpp.alloc_temp(lcpp.DeviceBlockTable.GetTempStorageBytes(n, n + 5))
    t = lcpp.DeviceBlockTable()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=torch.cuda.Stream()):
        for i in range(2):
            t.Extend(temp, lens[i], None, d_table, d_free, used[i], used[1 - i], lens[1 - i], starts, slots, None,
                     None, n, block)
    for _ in range(steps // 2):
        graph.replay()
    torch.cuda.synchronize()
    np.testing.assert_array_equal(host(lens[0]), context + steps)
    total = -(-(context + steps) // block)
    assert int(used[0]) == (total - held).sum()
    got = host(d_table)
    filled = got[np.arange(width) < total[:, None]]
    assert len(np.unique(filled)) == filled.size and set(filled) <= set(pages)
    position = context + steps - 1
    expect = got[np.arange(n), position // block].astype(np.int64) * block + position % block
    np.testing.assert_array_equal(host(slots)[:n], expect)
    assert (host(slots)[n:] == -1).all()


def test_extend_nothing(lcpp):
    empty = np.zeros(0, np.int32)
    check_extend(lcpp, empty, empty, np.zeros((0, 4), np.int32), 4, np.arange(3, dtype=np.int32), 2, 10, 16)
    # requests, but no tokens
    check_extend(lcpp, np.array([3, 0], np.int32), np.array([0, 0], np.int32), np.zeros((2, 4), np.int32), 4,
                 empty, 0, 0, 16)


# ---------------------------------------------------------------------------
# DeviceRouter
# ---------------------------------------------------------------------------
SCALE, COEF = 1.5, 0.25


def padded(x, dtype, pad, offset=0):
    """x as a view with `pad` spare columns per row, starting `offset` elements into its buffer."""
    t, e = x.shape
    buffer = torch.full((offset + t * (e + pad),), float("nan"), dtype=dtype, device="cuda")
    view = buffer[offset:].view(t, e + pad)[:, :e]
    view.copy_(cuda(x).to(dtype))
    return view


def run_route(L, logits, k, score, renormalize, bias=None, mask=None):
    t, e = logits.shape
    f32 = {"dtype": torch.float32, "device": "cuda"}
    weights, loss = torch.full((t, k), -7.0, **f32), torch.full((1,), -7.0, **f32)
    experts, counts, routed = i32(t, k), i32(e), i32(1)
    temp = L.alloc_temp(L.DeviceRouter.GetTempStorageBytes(t, e))
    L.DeviceRouter().Forward(temp, logits, weights, experts, counts, routed, loss, t, e, k, score, renormalize, SCALE,
                             COEF, None if bias is None else cuda(bias), None if mask is None else cuda(mask))
    assert L.device_status(temp) == L.OK
    return weights, experts, counts, routed, loss


def check_route(L, logits, k, score, renormalize, bias=None, mask=None):
    got = run_route(L, logits, k, score, renormalize, bias, mask)
    x32 = host(logits.float())
    weights, experts, counts, routed, loss = ref.route(x32, k, score, renormalize, SCALE, COEF, bias, mask)
    np.testing.assert_array_equal(host(got[1]), experts)
    np.testing.assert_array_equal(host(got[2]), counts)
    assert int(got[3]) == routed
    np.testing.assert_allclose(host64(got[0]), weights, rtol=1e-5, atol=1e-9)
    np.testing.assert_allclose(host64(got[4])[0], loss, rtol=1e-5, atol=1e-12)
    return got


def check_route_grad(L, logits, kind, k, score, renormalize, chosen, rng, in_place=False):
    _, experts, counts, routed, _ = chosen
    t, e = logits.shape
    g = rng.standard_normal((t, k)).astype(np.float32)
    dloss = np.array([3.0], np.float32)
    x = host64(logits)
    want = ref.route_grad(x, host(experts), host(counts), int(routed), g.astype(np.float64), 3.0, score, renormalize,
                          SCALE, COEF)
    out = logits if in_place else torch.full((t, e + 3), -7.0, dtype=logits.dtype, device="cuda")[:, :e]
    L.DeviceRouter().Backward(logits, experts, counts, routed, cuda(g), cuda(dloss), out, t, e, k, score, renormalize,
                              SCALE, COEF)
    rel, step = ROUND[kind]
    bound = 2e-5 * np.abs(want).max(1, keepdims=True) + rel * np.abs(want) + step
    # a row with an infinite logit has no gradient: NaN on both sides
    fine = ~np.isnan(want)
    np.testing.assert_array_equal(np.isnan(host(out.float())), ~fine)
    assert (np.abs(host64(out) - want) <= bound + 1e-12)[fine].all()


SHAPES = [(1, 1, 1), (1, 8, 2), (5, 2, 1), (33, 7, 3), (100, 8, 8), (300, 8, 1), (40, 9, 9), (70, 16, 4),
          (37, 13, 13), (17, 32, 4), (11, 17, 17), (29, 32, 32), (50, 33, 6), (90, 64, 6), (31, 64, 32), (301, 60, 4),
          (64, 128, 8), (257, 129, 32), (77, 160, 6), (1000, 256, 8), (41, 257, 10), (9, 512, 8), (30, 513, 2),
          (21, 1000, 32), (3, 1024, 32)]


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("score", [ref.SOFTMAX, ref.SIGMOID])
@pytest.mark.parametrize("renormalize", [True, False])
def test_route_and_gradient(lcpp, kind, score, renormalize):
    for t, e, k in SHAPES:
        rng = np.random.default_rng(t * e + k)
        x = rng.standard_normal((t, e)).astype(np.float32) * 2
        for variant in range(3):
            # contiguous; padded rows and a bias; rows off every vector boundary, a mask and a bias
            logits = padded(x, TYPES[kind], *[(0, 0), (8, 8), (3, 1)][variant])
            bias = rng.standard_normal(e).astype(np.float32) if variant else None
            mask = np.where(rng.random(t) < 0.3, -1, 2).astype(np.int32) if variant == 2 else None
            chosen = check_route(lcpp, logits, k, score, renormalize, bias, mask)
            check_route_grad(lcpp, logits, kind, k, score, renormalize, chosen, rng, in_place=variant == 1)


@pytest.mark.parametrize("e,k", [(8, 2), (60, 6), (256, 8), (1024, 4)])
@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_route_many_tokens(lcpp, e, k, kind):
    """Several blocks: counts and loss from all of them, the same bits twice."""
    rng = np.random.default_rng(e)
    t = 40_001 if e < 1024 else 9_001
    logits = cuda(rng.standard_normal((t, e)).astype(np.float32) + rng.standard_normal(e)).to(TYPES[kind])
    mask = np.where(rng.random(t) < 0.1, -1, 0).astype(np.int32)
    a = check_route(lcpp, logits, k, ref.SOFTMAX, True, None, mask)
    b = run_route(lcpp, logits, k, ref.SOFTMAX, True, None, mask)
    for x, y in zip(a, b):
        assert torch.equal(x, y)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_route_ties_go_to_the_lower_expert(lcpp, kind):
    """All equal, few different values, both zeros, and logits that differ in their last bits only."""
    rng = np.random.default_rng(3)
    for e in (8, 100, 256, 1024):
        x = np.full((40, e), 0.1, np.float32)
        x[10:20] = rng.integers(-2, 3, (10, e))
        x[20:30] = np.where(rng.random((10, e)) < 0.5, 0.0, -0.0)
        x[30:] = 1.0 + rng.integers(0, 6, (10, e)) * np.float32(2.0 ** -23)
        bias = (rng.integers(-2, 3, e) * 2.0 ** -22).astype(np.float32)
        for b in (None, bias):
            check_route(lcpp, cuda(x).to(TYPES[kind]), min(e, 9), ref.SOFTMAX, True, b)


@pytest.mark.parametrize("e,k", [(39, 23), (213, 16), (256, 8), (256, 1)])
def test_route_crowded_logits(lcpp, e, k):
    """Logits far from zero that lie close together, so that many words agree in what they keep of them, also
    past the last choice and on a lane that has handed out all it had found."""
    rng = np.random.default_rng(e * k)
    x = (rng.standard_normal((20_000, e)) * 0.01 + rng.choice([-30.0, 50.0], (20_000, 1))).astype(np.float32)
    check_route(lcpp, cuda(x), k, ref.SIGMOID, True)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("renormalize", [True, False])
def test_route_saturated_sigmoids(lcpp, kind, renormalize):
    """Sigmoids so near 1 that 1 - s has to be computed by itself."""
    rng = np.random.default_rng(17)
    x = (rng.standard_normal((200, 30)) * 6 + 22).astype(np.float32)
    logits = cuda(x).to(TYPES[kind])
    chosen = check_route(lcpp, logits, 3, ref.SIGMOID, renormalize)
    check_route_grad(lcpp, logits, kind, 3, ref.SIGMOID, renormalize, chosen, rng)


def test_route_grad_of_small_upstream(lcpp):
    """A small upstream gradient beside a large one whose weight is saturated keeps its digits."""
    x = np.tile(np.array([30.0, 0.0, -3.0, -4.0], np.float32), (40, 1))
    g = np.tile(np.array([1.0, 1e-6], np.float32), (40, 1))
    logits = cuda(x)
    _, experts, counts, routed, _ = check_route(lcpp, logits, 2, ref.SIGMOID, False)
    want = ref.route_grad(host64(logits), host(experts), host(counts), 40, g.astype(np.float64), 0.0, ref.SIGMOID, False,
                          SCALE, COEF)
    out = torch.empty_like(logits)
    lcpp.DeviceRouter().Backward(logits, experts, counts, routed, cuda(g), None, out, 40, 4, 2, ref.SIGMOID, False, SCALE,
                                 COEF)
    assert (np.abs(host64(out) - want) <= 2e-5 * np.abs(want).max(1, keepdims=True)).all()


@pytest.mark.parametrize("score", [ref.SOFTMAX, ref.SIGMOID])
def test_route_grad_of_equal_counts(lcpp, score):
    """Two experts with the same count share nearly all of a row: what its gradient is made of comes from the
    others' small shares, and is far below the slope that the two have in common."""
    x = np.full((200, 8), -42.0, np.float32)
    x[:180, :2] = -30.5
    x[:90, 0] = x[90:180, 1] = x[180:, 2] = -30.0
    logits = cuda(x)
    chosen = check_route(lcpp, logits, 1, score, True)
    check_route_grad(lcpp, logits, "f32", 1, score, True, chosen, np.random.default_rng(3))


@pytest.mark.parametrize("e,k", [(8, 8), (60, 6), (256, 8), (512, 32), (1024, 31)])
def test_route_near_ties(lcpp, e, k):
    """32-bit logits in clusters that agree in all but their last bits: of two, of a few, of more than are
    followed past the last choice, and across it."""
    rng = np.random.default_rng(e)
    t = 300
    x = rng.standard_normal((t, e)).astype(np.float32)
    for size, rows in ((2, slice(0, 100)), (4, slice(100, 180)), (30, slice(180, 240))):
        near = np.repeat(x[rows, : -(-e // size)], size, axis=1)[:, :e]
        bits = near.view(np.int32) ^ rng.integers(0, 4, near.shape).astype(np.int32)
        x[rows] = np.take_along_axis(bits.view(np.float32), np.argsort(rng.random(near.shape), axis=1), 1)
    x[240:] = (np.float32(0.1).view(np.int32) + rng.integers(0, 40, (60, e))).astype(np.int32).view(np.float32)
    bias = (rng.integers(-3, 4, e) * 2.0 ** -24).astype(np.float32)
    for b in (None, bias):
        check_route(lcpp, cuda(x), k, ref.SOFTMAX, True, b)


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("score", [ref.SOFTMAX, ref.SIGMOID])
@pytest.mark.parametrize("renormalize", [True, False])
def test_route_masked_experts(lcpp, kind, score, renormalize):
    """Experts switched off by -inf, rows with fewer than top_k experts or none, the type's lowest value, and
    logits far below zero."""
    rng = np.random.default_rng(9)
    x = rng.standard_normal((48, 20)).astype(np.float32)
    x[:, rng.random(20) < 0.4] = -np.inf
    x[5] = -np.inf
    x[6, 1:] = -np.inf
    x[7, :18] = -np.inf
    x[8] = torch.finfo(TYPES[kind]).min
    x[9, :10] = torch.finfo(TYPES[kind]).min
    x[10:14] = -70 - np.abs(rng.standard_normal((4, 20)) * 10)
    x[14:18] = 40 + rng.standard_normal((4, 20))
    logits = cuda(x).to(TYPES[kind])
    bias = rng.standard_normal(20).astype(np.float32)
    bias[3] = -np.inf
    for b in (None, bias):
        chosen = check_route(lcpp, logits, 4, score, renormalize, b)
        assert (host(chosen[1])[5] == -1).all()
        check_route_grad(lcpp, logits, kind, 4, score, renormalize, chosen, rng)


@pytest.mark.parametrize("renormalize", [True, False])
def test_route_large_logits(lcpp, renormalize):
    """Softmax only sees differences: rows far from zero, whose exponents alone would overflow, and rows that
    span the type (some of the last become infinite)."""
    rng = np.random.default_rng(21)
    for size in (300.0, 7e4, 3e6, 5e9, 1e30, 3e38):
        x = np.sign(rng.standard_normal((30, 1))) * np.float32(size) * (1 + rng.integers(0, 3, (30, 24)) * 2.0 ** -22)
        with np.errstate(over="ignore"):
            x = np.concatenate([x, rng.standard_normal((10, 24)) * size]).astype(np.float32)
        chosen = check_route(lcpp, cuda(x), 3, ref.SOFTMAX, renormalize)
        check_route_grad(lcpp, cuda(x), "f32", 3, ref.SOFTMAX, renormalize, chosen, rng)


def test_route_nothing_routed(lcpp):
    """No tokens, all tokens masked, all logits -inf: zero counts, loss and gradient, no NaN."""
    x = torch.full((6, 12), float("nan"), device="cuda")
    mask = np.full(6, -1, np.int32)
    for logits, m in ((x[:0], None), (x, mask), (torch.full_like(x, -float("inf")), None)):
        t = logits.shape[0]
        weights, experts, counts, routed, loss = run_route(lcpp, logits, 3, ref.SOFTMAX, True, None, m)
        assert int(routed) == 0 and float(loss) == 0.0 and not host(counts).any()
        assert (host(experts) == -1).all() and not host(weights).any()
        grad = torch.full_like(logits, 5.0)
        lcpp.DeviceRouter().Backward(logits, experts, counts, routed, torch.ones(t, 3, device="cuda"),
                                     torch.ones(1, device="cuda"), grad, t, 12, 3)
        assert not host(grad).any()


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("t", [9, 5000])
def test_route_nan_and_infinity(lcpp, t, kind):
    """A NaN or, under softmax, a +inf makes its own token's weights and the loss NaN, and nothing else."""
    rng = np.random.default_rng(2)
    x = rng.standard_normal((t, 16)).astype(np.float32)
    x[3, 5], x[4, 2] = -np.nan, np.inf
    logits = cuda(x).to(TYPES[kind])
    weights, experts, counts, routed, loss = run_route(lcpp, logits, 2, ref.SOFTMAX, True)
    assert int(host(experts)[3, 0]) == 5 and int(host(experts)[4, 0]) == 2
    bad = np.isnan(host(weights)).any(1)
    assert bad[3] and bad[4] and bad.sum() == 2
    assert np.isnan(float(loss)) and int(routed) == t and host(counts).sum() == 2 * t
    # a masked token's NaN reaches nothing
    mask = np.zeros(t, np.int32)
    mask[3:5] = -1
    finite = torch.nan_to_num(logits, 0.0, 0.0)
    check_route(lcpp, finite, 2, ref.SOFTMAX, True, None, mask)
    clean = run_route(lcpp, finite, 2, ref.SOFTMAX, True, None, mask)
    dirty = run_route(lcpp, logits, 2, ref.SOFTMAX, True, None, mask)
    for a, b in zip(clean, dirty):
        assert torch.equal(a, b)
    grads = []
    for values in (finite, logits):
        out = torch.empty_like(values)
        lcpp.DeviceRouter().Backward(values, *clean[1:4], torch.ones(t, 2, device="cuda"),
                                     torch.ones(1, device="cuda"), out, t, 16, 2)
        grads.append(out)
    assert torch.equal(*grads) and not host(grads[1].float())[3:5].any()


@pytest.mark.parametrize("score", [ref.SOFTMAX, ref.SIGMOID])
@pytest.mark.parametrize("renormalize", [True, False])
def test_route_gradient_against_differences(lcpp, score, renormalize):
    """Central differences of the 64-bit objective with step 1e-5: their own error is about 1e-9 (rounding,
    1e-15 / 1e-5, and 1e-10 of the third derivative), the kernel's 2e-5 of the row's largest entry."""
    rng = np.random.default_rng(4)
    t, e, k = 6, 11, 3
    x = rng.standard_normal((t, e)).astype(np.float32)
    logits = cuda(x)
    _, experts, counts, routed, _ = run_route(lcpp, logits, k, score, renormalize)
    g = rng.standard_normal((t, k)).astype(np.float32)
    out = torch.empty_like(logits)
    lcpp.DeviceRouter().Backward(logits, experts, counts, routed, cuda(g), torch.full((1,), 2.0, device="cuda"), out,
                                 t, e, k, score, renormalize, SCALE, COEF)
    args = (host(experts), host(counts), int(routed), g.astype(np.float64), 2.0, score, renormalize, SCALE, COEF)
    want = np.zeros((t, e))
    for i in range(t):
        for j in range(e):
            up, down = x.astype(np.float64), x.astype(np.float64)
            up[i, j] += 1e-5
            down[i, j] -= 1e-5
            want[i, j] = (ref.route_objective(up, *args) - ref.route_objective(down, *args)) / 2e-5
    assert (np.abs(host64(out) - want) <= 2e-5 * np.abs(want).max(1, keepdims=True) + 1e-8).all()


def test_route_gradient_without_a_part(lcpp):
    """Either upstream gradient may be missing; the parts add up."""
    rng = np.random.default_rng(6)
    t, e, k = 40, 24, 4
    logits = cuda(rng.standard_normal((t, e)).astype(np.float32))
    _, experts, counts, routed, _ = run_route(lcpp, logits, k, ref.SOFTMAX, True)
    g, dl = cuda(rng.standard_normal((t, k)).astype(np.float32)), torch.ones(1, device="cuda")

    def grad(gw, gl):
        out = torch.empty_like(logits)
        lcpp.DeviceRouter().Backward(logits, experts, counts, routed, gw, gl, out, t, e, k, ref.SOFTMAX, True, SCALE,
                                     COEF)
        return host64(out)

    both, weights, loss = grad(g, dl), grad(g, None), grad(None, dl)
    assert not grad(None, None).any()
    np.testing.assert_allclose(weights + loss, both, atol=1e-6)


# ---------------------------------------------------------------------------
# DeviceDispatch
# ---------------------------------------------------------------------------
def run_plan(L, experts, e, align, max_rows):
    t, k = experts.shape
    starts, row_of, pair_of = i32(e + 1), i32(t, k), i32(max_rows)
    temp = L.alloc_temp(L.DeviceDispatch.GetTempStorageBytes(t, k, e))
    L.DeviceDispatch().Plan(temp, cuda(experts), starts, row_of, pair_of, t, k, e, align)
    assert L.device_status(temp) == L.OK
    return starts, row_of, pair_of


def check_plan(L, experts, e, align, max_rows=None):
    t, k = experts.shape
    if max_rows is None:
        max_rows = L.DeviceDispatch.MaxRows(t, k, e, align)
    got = run_plan(L, experts, e, align, max_rows)
    for a, b in zip(got, ref.plan(experts, e, align, max_rows)):
        np.testing.assert_array_equal(host(a), b)
    return got


def choices(rng, t, k, e, missing=0.1):
    experts = np.argsort(rng.random((t, e)) - 0.3 * rng.random(e), axis=1)[:, :k].astype(np.int32)
    experts[rng.random(t) < missing] = -1
    return experts


# one block up to 2048 pairs, up to one per SM beyond (the borders: tests/test_model_step_edges_gpu.py)
@pytest.mark.parametrize("t,k,e,align", [(1, 1, 1, 1), (1, 8, 128, 16), (3, 2, 5, 7), (16, 8, 128, 128), (300, 4, 60, 8),
                                         (2048, 8, 256, 128), (2049, 8, 256, 64), (5000, 6, 1000, 1),
                                         (40_000, 2, 16, 128), (3000, 32, 33, 4), (90_001, 8, 257, 16), (500, 1, 1024, 3)])
def test_plan(lcpp, t, k, e, align):
    check_plan(lcpp, choices(np.random.default_rng(t + e), t, k, e), e, align)


def test_plan_one_expert_takes_all(lcpp):
    for t in (100, 70_000):
        experts = np.full((t, 1), 3, np.int32)
        check_plan(lcpp, experts, 8, 128)
        check_plan(lcpp, np.full((t, 1), -1, np.int32), 8, 128)


@pytest.mark.parametrize("t", [200, 9000])
def test_plan_too_few_rows_and_unknown_experts(lcpp, t):
    rng = np.random.default_rng(t)
    experts = rng.integers(-3, 12, (t, 3)).astype(np.int32)  # 8 and above name no expert
    experts[0, 0] = 2 ** 31 - 1
    for rows in (0, 1, t, 3 * t):
        check_plan(lcpp, experts, 8, 16, rows)


def test_plan_nothing(lcpp):
    starts, _, pair_of = run_plan(lcpp, np.zeros((0, 4), np.int32), 6, 16, 40)
    assert not host(starts).any() and (host(pair_of) == -1).all()


ROWS = [(1, 1, 1, 8, 1), (1, 8, 128, 4096, 16), (7, 3, 5, 1, 4), (33, 2, 8, 64, 16), (40, 6, 16, 129, 8),
        (64, 9, 20, 520, 1), (25, 10, 12, 2880, 32), (5, 4, 6, 8200, 2), (300, 4, 9, 257, 64), (11, 32, 40, 72, 1)]


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("layout", [(0, 0), (8, 8), (5, 3)])
def test_rows_there_and_back(lcpp, kind, layout):
    """Gather, combine with and without weights, and combine's gradient: contiguous rows, padded rows, rows
    off every vector boundary.  Rows past the last segment keep what they held."""
    dtype, (rel, step) = TYPES[kind], ROUND[kind]
    for t, k, e, h, align in ROWS:
        rng = np.random.default_rng(t * h + k)
        experts = choices(rng, t, k, e, 0.2 if t > 1 else 0.0)
        starts, row_of, pair_of = check_plan(lcpp, experts, e, align)
        end, rows = int(starts[-1]), pair_of.numel()
        hrow, hpair = host(row_of), host(pair_of)
        d = lcpp.DeviceDispatch()

        x = padded(rng.standard_normal((t, h)).astype(np.float32), dtype, *layout)
        out = padded(np.full((rows, h), 9, np.float32), dtype, *layout)
        d.Gather(x, row_of, pair_of, starts, out, t, k, e)
        np.testing.assert_array_equal(host64(out)[:end], ref.gather(host64(x), hpair, k, end))
        assert (host64(out)[end:] == 9).all()

        # garbage in padding rows and past the end must not reach a sum
        values = rng.standard_normal((rows, h)).astype(np.float32)
        values[hpair < 0] = np.nan
        y = padded(values, dtype, *layout)
        y64 = host64(y)
        weights = rng.random((t, k)).astype(np.float32)
        for w in (weights, None):
            got = padded(np.zeros((t, h), np.float32), dtype, *layout)
            d.Combine(y, row_of, None if w is None else cuda(w), got, t, k)
            want = ref.combine(y64, hrow, w)
            size = ref.combine(np.abs(y64), hrow, w)
            assert (np.abs(host64(got) - want) <= 1e-5 * size + rel * np.abs(want) + step).all()

        dy = padded(rng.standard_normal((t, h)).astype(np.float32), dtype, *layout)
        grad_rows = padded(np.full((rows, h), 9, np.float32), dtype, *layout)
        grad_weights = torch.full((t, k), -7.0, device="cuda")
        d.CombineBackward(dy, y, row_of, pair_of, starts, cuda(weights), grad_rows, grad_weights, t, k, e)
        want_rows, want_weights = ref.combine_grad(host64(dy), y64, hrow, hpair, weights.astype(np.float64), end)
        assert (np.abs(host64(grad_rows)[:end] - want_rows) <= (1e-6 + rel) * np.abs(want_rows) + step).all()
        assert (host64(grad_rows)[end:] == 9).all()
        _, size = ref.combine_grad(np.abs(host64(dy)), np.abs(y64), hrow, hpair, np.abs(weights.astype(np.float64)), end)
        assert (np.abs(host64(grad_weights) - want_weights) <= 1e-5 * size + 1e-12).all()
        # in place, and the same bits again
        again = torch.empty_like(grad_weights)
        d.CombineBackward(dy, y, row_of, pair_of, starts, cuda(weights), y, again, t, k, e)
        assert torch.equal(again, grad_weights)
        np.testing.assert_array_equal(host64(y)[:end], host64(grad_rows)[:end])


def test_rows_few_rows_kept(lcpp):
    """Pairs past max_rows have no row: they add nothing and get no gradient."""
    rng = np.random.default_rng(8)
    t, k, e, h = 50, 4, 6, 40
    experts = choices(rng, t, k, e)
    starts, row_of, pair_of = check_plan(lcpp, experts, e, 8, 90)
    rows = cuda(rng.standard_normal((90, h)).astype(np.float32))
    out, w = torch.empty(t, h, device="cuda"), rng.random((t, k)).astype(np.float32)
    d = lcpp.DeviceDispatch()
    d.Combine(rows, row_of, cuda(w), out, t, k)
    np.testing.assert_allclose(host64(out), ref.combine(host64(rows), host(row_of), w), rtol=1e-5, atol=1e-6)
    grad_rows, grad_weights = torch.empty_like(rows), torch.empty(t, k, device="cuda")
    d.CombineBackward(out, rows, row_of, pair_of, starts, cuda(w), grad_rows, grad_weights, t, k, e)
    assert not host(grad_weights)[host(row_of) < 0].any()
    x = cuda(rng.standard_normal((t, h)).astype(np.float32))
    d.Gather(x, row_of, pair_of, starts, rows, t, k, e)
    np.testing.assert_array_equal(host64(rows), ref.gather(host64(x), host(pair_of), k, int(starts[-1])))


def test_combine_gradient_against_differences(lcpp):
    """combine is linear in the rows and in the weights, so a difference quotient of any step is exact in 64
    bits; the kernel's gradient is within 1e-5 of the sum of magnitudes."""
    rng = np.random.default_rng(5)
    t, k, e, h = 6, 3, 5, 10
    experts = choices(rng, t, k, e, 0.0)
    starts, row_of, pair_of = check_plan(lcpp, experts, e, 4)
    n = pair_of.numel()
    rows, dy = rng.standard_normal((n, h)).astype(np.float32), rng.standard_normal((t, h)).astype(np.float32)
    w = rng.random((t, k)).astype(np.float32)
    grad_rows, grad_weights = torch.zeros(n, h, device="cuda"), torch.empty(t, k, device="cuda")
    lcpp.DeviceDispatch().CombineBackward(cuda(dy), cuda(rows), row_of, pair_of, starts, cuda(w), grad_rows,
                                          grad_weights, t, k, e)

    def objective(r, u):
        return (ref.combine(r, host(row_of), u) * dy).sum()

    base = objective(rows.astype(np.float64), w.astype(np.float64))
    for i, j in ((0, 0), (3, 2), (5, 1)):
        up = w.astype(np.float64)
        up[i, j] += 1.0
        assert abs(objective(rows.astype(np.float64), up) - base - float(grad_weights[i, j])) < 1e-4
    for r in range(0, int(starts[-1]), 3):
        up = rows.astype(np.float64)
        up[r, 4] += 1.0
        assert abs(objective(up, w.astype(np.float64)) - base - float(grad_rows[r, 4])) < 1e-4


# ---------------------------------------------------------------------------
# All of them
# ---------------------------------------------------------------------------
def test_on_another_stream_and_in_a_graph(lcpp):
    """The calls enqueue on the stream they are given and can be captured: a replay on new inputs in the same
    buffers gives those inputs' results."""
    rng = np.random.default_rng(12)
    t, e, k, h = 200, 32, 4, 64
    stream = torch.cuda.Stream()
    logits, x = torch.zeros(t, e, device="cuda"), torch.zeros(t, h, device="cuda")
    weights, loss = torch.zeros(t, k, device="cuda"), torch.zeros(1, device="cuda")
    experts, counts, routed = i32(t, k), i32(e), i32(1)
    rows_n = lcpp.DeviceDispatch.MaxRows(t, k, e, 8)
    starts, row_of, pair_of = i32(e + 1), i32(t, k), i32(rows_n)
    rows, out = torch.zeros(rows_n, h, device="cuda"), torch.zeros(t, h, device="cuda")
    temp = lcpp.alloc_temp(max(lcpp.DeviceRouter.GetTempStorageBytes(t, e),
                               lcpp.DeviceDispatch.GetTempStorageBytes(t, k, e)))
    d = lcpp.DeviceDispatch()

    def step(s=None):
        lcpp.DeviceRouter().Forward(temp, logits, weights, experts, counts, routed, loss, t, e, k, stream=s)
        d.Plan(temp, experts, starts, row_of, pair_of, t, k, e, 8, stream=s)
        d.Gather(x, row_of, pair_of, starts, rows, t, k, e, stream=s)
        d.Combine(rows, row_of, weights, out, t, k, stream=s)

    def check():
        # weights sum to 1, so the rows come back as they went
        assert (host64(out) - host64(x)).__abs__().max() <= 1e-5 * np.abs(host64(x)).max()
        assert host(counts).sum() == t * k

    logits.copy_(cuda(rng.standard_normal((t, e)).astype(np.float32)))
    x.copy_(cuda(rng.standard_normal((t, h)).astype(np.float32)))
    torch.cuda.synchronize()
    step(stream)
    stream.synchronize()
    check()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    logits.copy_(cuda(rng.standard_normal((t, e)).astype(np.float32)))
    x.copy_(cuda(rng.standard_normal((t, h)).astype(np.float32)))
    graph.replay()
    torch.cuda.synchronize()
    check()
    np.testing.assert_array_equal(host(experts), ref.choose(host(logits), None, k))
