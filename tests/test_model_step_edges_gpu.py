"""Edges of the model-step operators that tests/test_model_step_gpu.py does not reach, against the same 64-bit
references and with its tolerances (derived at its top)."""
from __future__ import annotations

import ctypes

import numpy as np
import pytest

import model_step_ref as ref
from test_model_step_gpu import COEF, ROUND, SCALE, TYPES, check_extend, check_plan, cuda, host, host64, i32, run_route

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


def test_extend_outputs_between_rows(lcpp):
    """Lengths and counters in the spare columns of the table's own rows: no element is shared."""
    context, new = np.array([30, 0, 17], np.int32), np.array([3, 20, 0], np.int32)
    buffer = i32(3, 24)
    buffer[:, :8] = cuda(np.arange(24, dtype=np.int32).reshape(3, 8))
    flat = buffer.view(-1)
    d_context, d_new, seq, starts = flat[8:11], flat[12:15], flat[32:35], flat[36:40]
    used, free = flat[64:65], np.arange(90, 94, dtype=np.int32)
    d_context.copy_(cuda(context))
    d_new.copy_(cuda(new))
    slots = torch.full((30,), -9, dtype=torch.int64, device="cuda")
    temp = lcpp.alloc_temp(lcpp.DeviceBlockTable.GetTempStorageBytes(3, 30))
    lcpp.DeviceBlockTable().Extend(temp, d_context, d_new, buffer[:, :8], cuda(free), None, used, seq, starts, slots,
                                   None, None, 3, 16)
    table, want, _, _, want_starts, want_seq, want_used = ref.extend(
        context, new, np.arange(24, dtype=np.int32).reshape(3, 8), 8, free, 0, 30, 16)
    np.testing.assert_array_equal(host(buffer)[:, :8], table)
    np.testing.assert_array_equal(host(slots), want)
    np.testing.assert_array_equal(host(starts), want_starts)
    np.testing.assert_array_equal(host(seq), want_seq)
    assert int(used) == want_used


def test_rows_without_columns_share_nothing(lcpp):
    """Rows of no elements (through the C entry point: an empty tensor has no address): what lies between their
    starts is free for other arrays."""
    t, k, e = 6, 2, 4
    experts = np.tile(np.array([[0, 3]], np.int32), (t, 1))
    starts, row_of, pair_of = check_plan(lcpp, experts, e, 2)
    floats = torch.full((400,), 5.0, device="cuda")
    weights, grad_weights = floats[1:1 + t * k], floats[201:201 + t * k]
    rows, grad_rows = floats.data_ptr(), floats[200:].data_ptr()
    torch.cuda.synchronize()
    status = lcpp.lib().lcpp_dispatch_combine_backward(
        rows, 0, rows, 8, row_of.data_ptr(), pair_of.data_ptr(), starts.data_ptr(), weights.data_ptr(), grad_rows, 8,
        grad_weights.data_ptr(), t, k, e, pair_of.numel(), 0, lcpp.F32, torch.cuda.current_stream().cuda_stream)
    assert status == lcpp.OK
    assert not host(grad_weights).any() and (host(floats)[:200] == 5.0).all()


@pytest.mark.parametrize("h", [24, 640, 4104])
def test_combine_gradient_over_the_weights(lcpp, h):
    """The weights' gradient takes the weights' place: the same bits as beside them."""
    rng = np.random.default_rng(h)
    t, k, e = 70, 9, 12
    experts = np.argsort(rng.random((t, e)), axis=1)[:, :k].astype(np.int32)
    experts[rng.random((t, k)) < 0.1] = -1
    starts, row_of, pair_of = check_plan(lcpp, experts, e, 4)
    rows, dy = (cuda(rng.standard_normal((n, h)).astype(np.float32)) for n in (pair_of.numel(), t))
    weights = cuda(rng.random((t, k)).astype(np.float32))
    got, apart = torch.zeros_like(rows), torch.zeros_like(rows)
    grad_weights = torch.empty_like(weights)
    d = lcpp.DeviceDispatch()
    d.CombineBackward(dy, rows, row_of, pair_of, starts, weights, apart, grad_weights, t, k, e)
    d.CombineBackward(dy, rows, row_of, pair_of, starts, weights, got, weights, t, k, e)
    assert torch.equal(weights, grad_weights) and torch.equal(got, apart)


def test_extend_of_changing_request_counts(lcpp):
    """A server's request count changes from step to step: few launch shapes are looked up and kept for all counts,
    and each has its results."""
    def shapes():
        count = ctypes.c_uint64()
        lcpp.check(lcpp.lib().lcpp_diag_launch_shapes(ctypes.byref(count)), "launch_shapes")
        return count.value

    rng = np.random.default_rng(2)
    before = shapes()
    for n in [*range(1, 40), *range(41, 4097, 97), 511, 512, 513, 1024, 1025, 2048, 2049, 4096]:
        context = rng.integers(0, 60, n).astype(np.int32)
        table = rng.permutation(n * 5).astype(np.int32).reshape(n, 5)
        free = (n * 5 + rng.permutation(n)).astype(np.int32)
        check_extend(lcpp, context, None, table, 5, free, None, n + 3, 16, optional=False)
    assert shapes() - before <= 8
    assert lcpp.lib().lcpp_diag_launch_shapes(None) == lcpp.ERR_INVALID_ARG


def route_gradient(L, logits, experts, counts, routed, g, dloss, score, renormalize):
    """(the kernel's gradient, the formula's)"""
    t, e = logits.shape
    k = experts.shape[1]
    out = torch.full_like(logits, -7.0)
    L.DeviceRouter().Backward(logits, experts, counts, routed, None if g is None else cuda(g),
                              None if dloss is None else torch.full((1,), dloss, device="cuda"), out, t, e, k, score,
                              renormalize, SCALE, COEF)
    g64 = np.zeros((t, k)) if g is None else g.astype(np.float64)
    want = ref.route_grad(host64(logits), host(experts), host(counts), int(routed), g64, dloss or 0.0, score,
                          renormalize, SCALE, COEF)
    return host64(out), want


def test_route_grad_of_rows_cut_short(lcpp):
    """A caller drops choices by setting them to -1: without its first one a token has no gradient, whatever
    stands behind it; without a later one it has the remaining ones'."""
    rng = np.random.default_rng(31)
    t, e, k = 60, 20, 4
    for score in (ref.SOFTMAX, ref.SIGMOID):
        for renormalize in (True, False):
            logits = cuda(rng.standard_normal((t, e)).astype(np.float32))
            _, experts, counts, routed, _ = run_route(lcpp, logits, k, score, renormalize)
            experts[:20, 0] = -1
            experts[10:40, 2] = -1
            g = rng.standard_normal((t, k)).astype(np.float32)
            got, want = route_gradient(lcpp, logits, experts, counts, routed, g, 3.0, score, renormalize)
            assert not got[:20].any()
            assert (np.abs(got - want) <= 2e-5 * np.abs(want).max(1, keepdims=True)).all()


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("score", [ref.SOFTMAX, ref.SIGMOID])
@pytest.mark.parametrize("renormalize", [True, False])
def test_route_grad_of_unchosen_leader(lcpp, kind, score, renormalize):
    """A bias keeps the expert with nearly all of a row's share out of the choice: what is left of the slopes
    once its own is taken off is far below them."""
    for e, k in ((5, 1), (16, 2), (64, 6), (256, 8), (1000, 4)):
        rng = np.random.default_rng(e)
        for shift in (0.0, -8.0, -20.0, -60.0):
            gap = rng.choice([4.0, 8.0, 12.0, 16.0, 20.0, 30.0], 150)
            x = rng.standard_normal((150, e))
            off = e // 3
            x[:, off] = x.max(1) + gap
            logits = cuda((x + shift).astype(np.float32)).to(TYPES[kind])
            bias = np.zeros(e, np.float32)
            bias[off] = -np.inf
            _, experts, counts, routed, _ = run_route(lcpp, logits, k, score, renormalize, bias)
            assert (host(experts) != off).all()
            g = rng.standard_normal((150, k)).astype(np.float32)
            for up, dloss in ((g, 3.0), (g, None), (None, 3.0)):
                got, want = route_gradient(lcpp, logits, experts, counts, routed, up, dloss, score, renormalize)
                bound = 2e-5 * np.abs(want).max(1, keepdims=True) + ROUND[kind][0] * np.abs(want)
                assert (np.abs(got - want) <= bound).all(), (e, k, shift, up is None, dloss)


@pytest.mark.parametrize("score", [ref.SOFTMAX, ref.SIGMOID])
@pytest.mark.parametrize("renormalize", [True, False])
@pytest.mark.parametrize("group", [2, 3, 20])
def test_route_grad_of_unchosen_group(lcpp, score, renormalize, group):
    """Several experts that a bias keeps out, and that no token counts for, share a row among them: they have one
    slope, and what is left of it is far below it."""
    rng = np.random.default_rng(group)
    for e, k in ((22, 1), (64, 6), (256, 8), (1000, 2)):
        for low in (-6.0, -9.0, -14.0):
            x = rng.standard_normal((120, e)) + low
            x[:, :group] = rng.choice([0.5, 2.0, 6.0, 16.0], (120, group)) + rng.random((120, group))
            bias = np.zeros(e, np.float32)
            bias[:group] = -np.inf
            logits = cuda(x.astype(np.float32))
            _, experts, counts, routed, _ = run_route(lcpp, logits, k, score, renormalize, bias)
            g = rng.standard_normal((120, k)).astype(np.float32) * 1e-3
            for up in (g, None):
                got, want = route_gradient(lcpp, logits, experts, counts, routed, up, 3.0, score, renormalize)
                assert (np.abs(got - want) <= 2e-5 * np.abs(want).max(1, keepdims=True)).all(), (e, k, low)


@pytest.mark.parametrize("renormalize", [True, False])
def test_route_tiny_sigmoids(lcpp, renormalize):
    """Sigmoids so small that those next to the largest have no 32-bit value of their own: weights and gradient
    keep them as parts of the row's."""
    rng = np.random.default_rng(19)
    for e, k in ((11, 5), (40, 6), (256, 8)):
        x = np.empty((160, e), np.float32)
        x[:] = np.repeat([-20.0, -30.0, -44.7, -45.0, -47.0, -59.0, -61.0, -80.0], 20)[:, None]
        x[:, 2:] -= rng.uniform(25, 42, (160, e - 2)).astype(np.float32)
        x[:, 1] -= 30
        logits = cuda(x)
        weights, experts, counts, routed, loss = run_route(lcpp, logits, k, ref.SIGMOID, renormalize)
        want = ref.route(x, k, ref.SIGMOID, renormalize, SCALE, COEF)
        np.testing.assert_array_equal(host(experts), want[1])
        np.testing.assert_allclose(host64(weights), want[0], rtol=1e-5, atol=0 if renormalize else 1e-37)
        assert abs(float(loss) - want[4]) <= 1e-5 * want[4]
        counts[0] = 0  # no slope of its own for the leading expert's share
        got, want = route_gradient(lcpp, logits, experts, counts, routed, None, 3.0, ref.SIGMOID, renormalize)
        assert (np.abs(got - want) <= 2e-5 * np.abs(want).max(1, keepdims=True)).all()


@pytest.mark.parametrize("score", [ref.SOFTMAX, ref.SIGMOID])
@pytest.mark.parametrize("renormalize", [True, False])
def test_route_grad_beside_led_rows(lcpp, score, renormalize):
    """A row has the same bits beside rows that need more care (an unchosen leader, tiny sigmoids) as without them."""
    rng = np.random.default_rng(23)
    for e, k in ((8, 2), (64, 6), (256, 8)):
        x = rng.standard_normal((90, e)).astype(np.float32) - 3
        mixed = x.copy()
        mixed[::3, 1] = 12.0
        mixed[1::9] -= 80.0
        bias = np.zeros(e, np.float32)
        bias[1] = -np.inf
        g = rng.standard_normal((90, k)).astype(np.float32)
        _, experts, counts, routed, _ = run_route(lcpp, cuda(x), k, score, renormalize, bias)
        chosen = run_route(lcpp, cuda(mixed), k, score, renormalize, bias)[1]
        plain, _ = route_gradient(lcpp, cuda(x), experts, counts, routed, g, 3.0, score, renormalize)
        got, _ = route_gradient(lcpp, cuda(mixed), chosen, counts, routed, g, 3.0, score, renormalize)
        same = (mixed == x).all(1)
        assert same.sum() >= 50 and torch.equal(chosen[cuda(same)], experts[cuda(same)])
        np.testing.assert_array_equal(got[same], plain[same])


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("t", [7, 3000])
@pytest.mark.parametrize("e", [24, 32, 256])
def test_route_switched_off_experts_stay_off(lcpp, kind, t, e):
    """A bias of -inf keeps an expert out of the choice also where its logit is NaN or +inf."""
    rng = np.random.default_rng(t)
    x = rng.standard_normal((t, e)).astype(np.float32)
    off = [4, 9, e - 1]
    x[:, [4, e - 1]] = np.nan
    x[::2, 9] = np.inf
    x[1::3, 9] = np.nan
    bias = np.zeros(e, np.float32)
    bias[off] = -np.inf
    clean = x.copy()
    clean[:, off] = -np.inf
    logits = cuda(x).to(TYPES[kind])
    for k in {1, 4, min(e - 3, 29), min(e, 32)}:
        _, experts, counts, routed, _ = run_route(lcpp, logits, k, ref.SIGMOID, True, bias)
        want = ref.choose(host(cuda(clean).to(TYPES[kind]).float()), None, k)
        np.testing.assert_array_equal(host(experts), want)
        assert int(routed) == t and not host(counts)[off].any()


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("biased", [False, True])
def test_route_rows_of_nan(lcpp, kind, biased):
    """NaN logits are equal to one another: the lower experts come first, however many there are."""
    for e, k in ((12, 2), (8, 8), (256, 8), (1000, 32)):
        x = np.random.default_rng(e).standard_normal((30, e)).astype(np.float32)
        x[:10] = np.nan
        x[10:20, : e // 2] = -np.nan
        x[20:25, 1::2] = np.nan
        bias = np.random.default_rng(k).standard_normal(e).astype(np.float32) if biased else None
        logits = cuda(x).to(TYPES[kind])
        experts = run_route(lcpp, logits, k, ref.SIGMOID, True, bias)[1]
        np.testing.assert_array_equal(host(experts), ref.choose(host(logits.float()), bias, k))


def route_by_score(L, logits, k, score, renormalize, bias, mask=None):
    """Forward with the bias on the scores; (experts, 64-bit sums) after weights, counts and loss were checked
    against those of the experts it chose."""
    weights, experts, counts, routed, loss = run_route(L, logits, k, score + L.BIAS_ON_SCORE, renormalize, bias, mask)
    t, e = logits.shape
    x, chosen = host64(logits), host(experts)
    log_s, share = ref._scores(x, score)
    has, live = chosen >= 0, chosen[:, 0] >= 0
    picked = np.where(has, np.exp(np.take_along_axis(log_s, np.maximum(chosen, 0), 1)), 0.0)
    if renormalize:
        picked /= np.where(live[:, None], picked.sum(1, keepdims=True), 1.0)
    np.testing.assert_allclose(host64(weights), SCALE * picked, rtol=1e-5, atol=1e-9)
    np.testing.assert_array_equal(host(counts), np.bincount(chosen[has], minlength=e))
    assert int(routed) == live.sum() == (t if mask is None else (mask >= 0).sum())
    want = COEF * e * (share[live].sum(0) / live.sum() * host(counts) / (k * live.sum())).sum()
    assert abs(float(loss) - want) <= 1e-5 * want
    return chosen, np.where(np.isneginf(x), -np.inf, np.exp(log_s) + bias.astype(np.float64))


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("score", [ref.SOFTMAX, ref.SIGMOID])
@pytest.mark.parametrize("renormalize", [True, False])
def test_route_bias_on_scores(lcpp, kind, score, renormalize):
    """The largest score + bias.  A score is off by at most 4e-7 (1 at most, a quotient of exponentials good to
    2^-22 each), its sum with a bias below 2 by 2^-23 more: sums that differ by 2e-6 have to be in order."""
    for t, e, k in ((50, 2, 1), (300, 8, 2), (37, 16, 16), (70, 60, 6), (5000, 64, 6), (400, 160, 6), (900, 256, 8),
                    (30, 512, 32), (20, 1000, 10)):
        rng = np.random.default_rng(t + e)
        x = (rng.standard_normal((t, e)) * 2).astype(np.float32)
        bias = (rng.standard_normal(e) * (0.1 if score == ref.SIGMOID else 1.0 / e)).astype(np.float32)
        if e > 16:
            x[rng.random((t, e)) < 0.1] = -np.inf
            bias[e // 2] = -np.inf
        mask = np.where(rng.random(t) < 0.2, -1, 0).astype(np.int32) if t % 20 else None
        logits = cuda(x).to(TYPES[kind])
        chosen, sums = route_by_score(lcpp, logits, k, score, renormalize, bias, mask)
        live = chosen[:, 0] >= 0
        chosen, sums, rows = chosen[live], sums[live], np.nonzero(live)[0]
        order = np.argsort(-sums, axis=1, kind="stable")
        best = np.take_along_axis(sums, order, 1)
        assert (np.abs(np.take_along_axis(sums, chosen, 1) - best[:, :k]) <= 2e-6).all()
        assert all(len(set(c)) == k for c in chosen)
        with np.errstate(invalid="ignore"):
            gap = -np.diff(best, axis=1, append=-np.inf)
        clear = (gap[:, :k] > 2e-6) & (np.concatenate([np.full((len(rows), 1), np.inf), gap[:, :k - 1]], 1) > 2e-6)
        np.testing.assert_array_equal(chosen[clear], order[:, :k][clear])
        assert clear.mean() > 0.9
        if e >= 8 and k < e:  # it is another choice than that of logit + bias
            assert (chosen != ref.choose(host(logits.float()), bias, k)[live]).any(1).mean() > 0.05


@pytest.mark.parametrize("score", [ref.SOFTMAX, ref.SIGMOID])
@pytest.mark.parametrize("e,k", [(40, 5), (256, 8), (1000, 32)])
def test_route_bias_on_equal_scores(lcpp, score, e, k):
    """Few different logits and biases: equal scores have equal bits, so equal sums go to the lower expert, however
    many there are; scores that 32 bits do not tell from 1 are equal."""
    rng = np.random.default_rng(e)
    x = rng.choice([0.0, 1.0, -4.0], (60, e)).astype(np.float32)
    x[:10] = 0.5
    if score == ref.SIGMOID:
        x[20:30] = rng.choice([40.0, 60.0, 90.0], (10, e))
    bias = rng.choice([0.0, 0.25, 0.125], e).astype(np.float32)
    chosen, sums = route_by_score(lcpp, cuda(x), k, score, True, bias)
    rank = np.lexsort((np.broadcast_to(np.arange(e), sums.shape), -np.round(sums, 5)), axis=1)[:, :k]
    np.testing.assert_array_equal(chosen, rank)


def test_route_bias_on_scores_of_broken_rows(lcpp):
    """A NaN logit, or +inf under softmax, makes its own row's weights NaN; masked rows pass nothing on; rows of
    -inf alone are left out; far logits, whose scores are 0 in 32 bits, are told apart by the bias."""
    x = np.random.default_rng(3).standard_normal((40, 12)).astype(np.float32)
    x[3, 5], x[4, 2], x[5] = np.nan, np.inf, -np.inf
    x[6], x[7] = -1e30, -200.0
    bias = np.linspace(0, 1, 12).astype(np.float32)
    for score in (ref.SOFTMAX, ref.SIGMOID):
        weights, experts, counts, routed, _ = run_route(lcpp, cuda(x), 2, score + lcpp.BIAS_ON_SCORE, True, bias)
        bad = np.isnan(host(weights)).any(1)
        assert bad[3] and bad.sum() == (2 if score == ref.SOFTMAX else 1)
        assert host(experts)[3, 0] == (0 if score == ref.SOFTMAX else 5)
        assert (host(experts)[5] == -1).all() and int(routed) == 39 and host(counts).sum() == 78
        np.testing.assert_array_equal(host(experts)[6], [11, 10])
        np.testing.assert_array_equal(host(experts)[7], [11, 10])


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("score", [ref.SOFTMAX, ref.SIGMOID])
@pytest.mark.parametrize("renormalize", [True, False])
def test_route_accuracy(lcpp, kind, score, renormalize):
    """Ordinary logits: an exponential is good to 2^-22 and half a unit of its argument (below 16: 2^-21), a lane's
    sum of 32 to 32 half units (2^-19), a quotient to 2^-22: 3.3e-6 in all for a weight, and so for the loss."""
    rng = np.random.default_rng(29)
    for t, e, k in ((500, 8, 2), (500, 60, 6), (300, 256, 8), (6000, 160, 6), (100, 1000, 10)):
        logits = cuda((rng.standard_normal((t, e)) * 1.5).astype(np.float32)).to(TYPES[kind])
        weights, experts, _, _, loss = run_route(lcpp, logits, k, score, renormalize)
        want = ref.route(host(logits.float()), k, score, renormalize, SCALE, COEF)
        np.testing.assert_array_equal(host(experts), want[1])
        np.testing.assert_allclose(host64(weights), want[0], rtol=3.3e-6, atol=0)
        assert abs(float(loss) - want[4]) <= 3.3e-6 * want[4]


@pytest.mark.parametrize("score", [ref.SOFTMAX, ref.SIGMOID])
@pytest.mark.parametrize("t", [40, 4000, 60_001])
@pytest.mark.parametrize("logit", [-12.0, -30.0, -45.0, -60.0, -75.0])
def test_route_loss_of_small_shares(lcpp, score, t, logit):
    """A bias sends every token to an expert with next to no share: the loss keeps its digits however many blocks
    add to it."""
    rng = np.random.default_rng(5)
    x = rng.standard_normal((t, 16)).astype(np.float32)
    x[:, 3] = logit
    bias = np.zeros(16, np.float32)
    bias[3] = 100.0
    loss = run_route(lcpp, cuda(x), 1, score, True, bias)[4]
    want = ref.route(x, 1, score, True, SCALE, COEF, bias)[4]
    assert abs(float(loss) - want) <= 1e-5 * want


# one block of 256 threads up to 256 pairs and 256 experts, one of 1024 up to 2048 pairs, several beyond
@pytest.mark.parametrize("pairs", [255, 256, 257, 1023, 1024, 1025, 2047, 2048, 2049, 3073])
@pytest.mark.parametrize("e", [255, 256, 257, 1024])
def test_plan_borders(lcpp, pairs, e):
    rng = np.random.default_rng(pairs * e)
    experts = rng.integers(-1, e, (pairs, 1)).astype(np.int32)
    check_plan(lcpp, experts, e, 16)
    check_plan(lcpp, experts, e, 1, pairs // 2)


@pytest.mark.parametrize("kind,t,h,k", [("bf16", 1300, 2048, 8), ("f32", 2400, 1024, 2), ("f16", 2700, 904, 5),
                                        ("bf16", 400, 8192, 3), ("bf16", 500, 2881, 3)])
def test_combine_gradient_of_long_batches(lcpp, kind, t, h, k):
    """Enough columns in all for the lanes that take several accesses each."""
    rng = np.random.default_rng(h)
    e, dtype, (rel, step) = 24, TYPES[kind], ROUND[kind]
    experts = np.argsort(rng.random((t, e)), axis=1)[:, :k].astype(np.int32)
    experts[rng.random((t, k)) < 0.1] = -1
    starts, row_of, pair_of = check_plan(lcpp, experts, e, 16)
    end, n = int(starts[-1]), pair_of.numel()
    rows, dy = (cuda(rng.standard_normal(s).astype(np.float32)).to(dtype) for s in ((n, h), (t, h)))
    w = rng.random((t, k)).astype(np.float32)
    grad_rows, grad_weights = torch.full_like(rows, 9), torch.full((t, k), -7.0, device="cuda")
    lcpp.DeviceDispatch().CombineBackward(dy, rows, row_of, pair_of, starts, cuda(w), grad_rows, grad_weights, t, k, e)
    want_rows, want_weights = ref.combine_grad(host64(dy), host64(rows), host(row_of), host(pair_of),
                                               w.astype(np.float64), end)
    assert (np.abs(host64(grad_rows)[:end] - want_rows) <= (1e-6 + rel) * np.abs(want_rows) + step).all()
    assert (host64(grad_rows)[end:] == 9).all()
    _, size = ref.combine_grad(np.abs(host64(dy)), np.abs(host64(rows)), host(row_of), host(pair_of),
                               w.astype(np.float64), end)
    assert (np.abs(host64(grad_weights) - want_weights) <= 1e-5 * size + 1e-12).all()
