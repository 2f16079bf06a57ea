"""DeviceRotary, DevicePagedAttention and DeviceCacheEviction against 64-bit references (tests/cache_ref.py).

Tolerances.  Whole numbers, copied rows and scores that move are exact.
Rotary: cosine and sine are off by at most 4e-7 (half a unit of the fraction of a turn, 2^-25, times 2 pi, is 1.9e-7;
sincospi adds 2^-23), and two products and a sum by 2^-24 each: 6e-7 of |a| + |b|, then the type's rounding.
Attention: a logit's dot product adds D terms in 32 bits, off by at most 2^-22 of the sum of their magnitudes (10 here:
2.4e-6), its exponential by 2^-22 and half a unit of an argument below 32 (1.9e-6); a term kept as two bfloat16 numbers
is off by 2^-17 (7.6e-6); a lane adds at most 256 terms in a row (2^-16, 1.5e-5): 3e-5 of sum p |v| with the quotient's
2^-23, then the type's rounding.  lse and scores are sums of the same terms: 2e-5 and 4e-5 relative."""
from __future__ import annotations

import math

import numpy as np
import pytest

import cache_ref as ref

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
KINDS = ["bf16", "f16", "f32"]


def rounding(t, value):
    """Half a step of the type at each value, float16's smallest step below its normal numbers."""
    return torch.finfo(t).eps / 2 * value + (2.0 ** -25 if t == torch.float16 else 0.0)


def randn(seed, dtype, *shape):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(*shape, device="cuda", generator=g).to(dtype)


def i32(values):
    return torch.tensor(np.asarray(values), dtype=torch.int32, device="cuda")


def host64(t):
    return t.detach().double().cpu().numpy()


def strided(t, where):
    """The tensor's values in a view whose elements lie elsewhere: a copy, rows of a wider buffer, heads first, or a
    start that no vector access is aligned to."""
    a, b, c = t.shape
    if where == "plain":
        return t.clone()
    if where == "wide":
        out = torch.zeros(a, b + 3, c + 16 // t.element_size(), dtype=t.dtype, device=t.device)[:, 1:b + 1, :c]
    elif where == "heads":
        out = torch.zeros(b, a, c, dtype=t.dtype, device=t.device).transpose(0, 1)
    else:
        out = torch.zeros(a * b * (c + 1) + 1, dtype=t.dtype, device=t.device)[1:].view(a, b, c + 1)[:, :, :c]
    out.copy_(t)
    return out


# ---------------------------------------------------------------------------
# DeviceRotary
# ---------------------------------------------------------------------------
def check_turn(out, x, positions, frequencies, layout, scale, inverse=False):
    want, size = ref.turn(host64(x), positions, host64(frequencies), layout, scale, inverse)
    assert (np.abs(host64(out) - want) <= 6e-7 * size + rounding(out.dtype, np.abs(want))).all()
    turned = 2 * frequencies.numel()
    assert torch.equal(out[:, :, turned:], x[:, :, turned:])


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("layout", [ref.HALF, ref.INTERLEAVED])
@pytest.mark.parametrize("dim,rotary", [(64, 64), (128, 128), (80, 40), (192, 64), (256, 256), (96, 6), (10, 4),
                                        (7, 2), (64, 0), (256, 250), (1, 0), (2, 2)])
def test_rotary(lcpp, kind, layout, dim, rotary):
    for t, heads, kv, where, scale in ((1, 1, 1, "plain", 1.0), (37, 5, 2, "wide", 0.75), (130, 4, 4, "heads", 1.0),
                                       (700, 3, 1, "odd", 1.25)):
        q, k = (strided(randn(t + i, TYPES[kind], t, h, dim), where) for i, h in enumerate((heads, kv)))
        positions = np.random.default_rng(t).integers(-5, 100_000, t)
        f = lcpp.DeviceRotary.Frequencies(rotary)
        for inverse in (False, True):
            call = lcpp.DeviceRotary().Backward if inverse else lcpp.DeviceRotary().Forward
            q_out, k_out = (strided(torch.full_like(x, 7), where) for x in (q, k))
            call(q, k, q_out, k_out, i32(positions), f, t, layout=layout, scale=scale)
            for out, x in ((q_out, q), (k_out, k)):
                check_turn(out, x, positions, f, layout, scale, inverse)
            a, b = strided(q, where), strided(k, where)
            call(a, b, a, b, i32(positions), f, t, layout=layout, scale=scale)
            assert torch.equal(a, q_out) and torch.equal(b, k_out)
            call(q, None, a, None, i32(positions), f, t, layout=layout, scale=scale)
            assert torch.equal(a, q_out)


@pytest.mark.parametrize("layout", [ref.HALF, ref.INTERLEAVED])
def test_rotary_far_positions(lcpp, layout):
    """Angles of the last positions that 32 bits hold: an angle of 2^31 radians is off by 2^-23 in 64 bits."""
    positions = np.array([2 ** 31 - 1, -2 ** 31, 10 ** 9 + 7, 16_777_217, 1_000_003], np.int64)
    x = randn(3, torch.float32, 5, 2, 64)
    out, f = torch.empty_like(x), lcpp.DeviceRotary.Frequencies(64)
    lcpp.DeviceRotary().Forward(x, None, out, None, i32(positions), f, 5, layout=layout)
    want, size = ref.turn(host64(x), positions, host64(f), layout)
    assert (np.abs(host64(out) - want) <= (6e-7 + 3 * 2.0 ** -23) * size + 2.0 ** -24).all()


@pytest.mark.parametrize("tokens", [1, 511, 512, 2370, 9473])
@pytest.mark.parametrize("heads", [1, 3, 64])
def test_rotary_block_sizes(lcpp, tokens, heads):
    """From one token in a block to sixteen, and heads that need several rounds."""
    x = randn(tokens, torch.bfloat16, tokens, heads, 16)
    out, f = torch.zeros_like(x), lcpp.DeviceRotary.Frequencies(8, base=100.0)
    positions = np.arange(tokens) * 3
    lcpp.DeviceRotary().Forward(x, None, out, None, i32(positions), f, tokens, layout=ref.INTERLEAVED)
    check_turn(out, x, positions, f, ref.INTERLEAVED, 1.0)


def test_rotary_gradient(lcpp):
    """Backward is the transpose of Forward: <Forward(x), y> = <x, Backward(y)>, and differences of Forward agree."""
    for layout in (ref.HALF, ref.INTERLEAVED):
        x, y = randn(1, torch.float32, 40, 3, 32), randn(2, torch.float32, 40, 3, 32)
        positions, f = i32(np.arange(40) * 101), lcpp.DeviceRotary.Frequencies(24)
        turned, back = torch.empty_like(x), torch.empty_like(x)
        lcpp.DeviceRotary().Forward(x, None, turned, None, positions, f, 40, layout=layout, scale=1.5)
        lcpp.DeviceRotary().Backward(y, None, back, None, positions, f, 40, layout=layout, scale=1.5)
        a, b = float((turned.double() * y.double()).sum()), float((x.double() * back.double()).sum())
        assert abs(a - b) <= 1e-6 * float((turned.abs().double() * y.abs().double()).sum())
        moved, step = torch.empty_like(x), 0.5  # Forward is linear
        nudge = torch.zeros_like(x)
        nudge[7, 1, 5] = nudge[30, 2, 31] = step
        lcpp.DeviceRotary().Forward(x + nudge, None, moved, None, positions, f, 40, layout=layout, scale=1.5)
        slope = ((moved.double() - turned.double()) * y.double()).sum((1, 2)) / step
        assert abs(float(slope[7]) - float(back[7, 1, 5])) <= 1e-4
        assert abs(float(slope[30]) - float(back[30, 2, 31])) <= 1e-4


def test_rotary_in_a_fused_projection(lcpp):
    """Queries and keys turned in place in the rows that also hold the values, which stay."""
    t, h, kv, d = 33, 4, 2, 64
    rows = randn(5, torch.bfloat16, t, (h + 2 * kv) * d)
    before = rows.clone()
    q, k, v = (x.unflatten(1, (-1, d)) for x in rows.split((h * d, kv * d, kv * d), 1))
    f, positions = lcpp.DeviceRotary.Frequencies(d), np.arange(t)
    lcpp.DeviceRotary().Forward(q, k, q, k, i32(positions), f, t)
    was = before.split((h * d, kv * d, kv * d), 1)
    check_turn(q.contiguous(), was[0].unflatten(1, (-1, d)), positions, f, ref.HALF, 1.0)
    check_turn(k.contiguous(), was[1].unflatten(1, (-1, d)), positions, f, ref.HALF, 1.0)
    assert torch.equal(v, was[2].unflatten(1, (-1, d)))


def test_rotary_requests(lcpp):
    """Tokens of no request stay as they are; requests' offsets are added."""
    t = 50
    x = randn(8, torch.float32, t, 2, 16)
    request = np.random.default_rng(0).integers(-1, 4, t)
    offset, positions = np.array([0, 1000, 7]), np.arange(t)
    f, out = lcpp.DeviceRotary.Frequencies(16), torch.full_like(x, 9)
    lcpp.DeviceRotary().Forward(x, None, out, None, i32(positions), f, t, d_token_request=i32(request),
                                d_position_offset=i32(offset))
    live = (request >= 0) & (request < 3)
    assert (host64(out)[~live] == 9).all() and 0 < live.sum() < t
    at = positions[live] + offset[request[live]]
    check_turn(out[torch.tensor(live)], x[torch.tensor(live)], at, f, ref.HALF, 1.0)
    out.fill_(9)
    lcpp.DeviceRotary().Forward(x, None, out, None, i32(positions), f, t, d_token_request=i32(request))
    assert (host64(out)[request < 0] == 9).all()
    check_turn(out[torch.tensor(request >= 0)], x[torch.tensor(request >= 0)], positions[request >= 0], f, ref.HALF, 1.0)


def make_cache(kind, pages, block, heads, dim, layout, seed=0):
    """Keys and values [pages, block, heads, dim] in one of the memory orders."""
    dtype = TYPES[kind]
    if layout == "tokens":
        return randn(seed, dtype, pages, block, heads, dim), randn(seed + 1, dtype, pages, block, heads, dim)
    if layout == "heads":
        return tuple(randn(seed + i, dtype, pages, heads, block, dim).transpose(1, 2) for i in range(2))
    if layout == "both":  # keys and values of a page side by side
        both = randn(seed, dtype, pages, 2, block, heads, dim)
        return both[:, 0], both[:, 1]
    if layout == "pairs":  # of a head
        both = randn(seed, dtype, pages, block, heads, 2, dim)
        return both[:, :, :, 0], both[:, :, :, 1]
    flat = [randn(seed + i, dtype, pages * block * heads * (dim + 1) + 1)[1:] for i in range(2)]
    return tuple(x.view(pages, block, heads, dim + 1)[..., :dim] for x in flat)


LAYOUTS = ["tokens", "heads", "both", "pairs", "odd"]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("cache", LAYOUTS)
@pytest.mark.parametrize("t,block,dim,rotary,layout", [(1, 1, 64, 64, 0), (70, 16, 128, 128, 0), (333, 24, 80, 40, 1),
                                                       (50, 7, 9, 4, 1), (1200, 64, 192, 64, 0)])
def test_append(lcpp, kind, cache, t, block, dim, rotary, layout):
    h, kv = 6, 3
    pages = t // block + 3
    rng = np.random.default_rng(t)
    slots = rng.permutation(pages * block)[:t]
    slots[rng.random(t) < 0.2] = -1
    if t > 40:
        slots[7], slots[9] = pages * block, 2 ** 45
    live = (slots >= 0) & (slots < pages * block)
    rows = randn(t, TYPES[kind], t, (h + 2 * kv) * dim)
    q, k, v = (x.unflatten(1, (-1, dim)) for x in rows.split((h * dim, kv * dim, kv * dim), 1))
    kc, vc = make_cache(kind, pages, block, kv, dim, cache)
    want_k, want_v = kc.clone(), vc.clone()
    request, offset = rng.integers(0, 4, t), np.array([0, 50, 9000, 3])
    positions, f = rng.integers(0, 5000, t), lcpp.DeviceRotary.Frequencies(rotary, base=1e5)
    q_out = torch.full((t, h, dim), 5, dtype=TYPES[kind], device="cuda")
    slot_positions, scores = i32(np.full(pages * block, -3)), torch.full((pages * block,), 4.0, device="cuda")
    lcpp.DeviceRotary().Append(q, k, v, q_out, kc, vc, torch.tensor(slots, device="cuda"), i32(positions), f, t,
                               layout=layout, d_token_request=i32(request), d_position_offset=i32(offset),
                               d_slot_positions=slot_positions, d_slot_scores=scores)
    at = positions + offset[request]
    mask = torch.tensor(live)
    check_turn(q_out[mask], q[mask], at[live], f, layout, 1.0)
    assert (host64(q_out)[~live] == 5).all()
    s = torch.tensor(slots[live], device="cuda")
    check_turn(kc[s // block, s % block], k[mask], at[live], f, layout, 1.0)
    assert torch.equal(vc[s // block, s % block], v[mask])
    untouched = torch.ones(pages * block, dtype=torch.bool, device="cuda")
    untouched[s] = False
    rest = untouched.nonzero()[:, 0]
    assert torch.equal(kc[rest // block, rest % block], want_k[rest // block, rest % block])
    assert torch.equal(vc[rest // block, rest % block], want_v[rest // block, rest % block])
    assert (slot_positions[rest] == -3).all() and (scores[rest] == 4).all()
    assert (scores[s] == 0).all() and torch.equal(slot_positions[s], i32(at[live]))
    # without queries and the arrays beside the cache
    kc2, vc2 = (x.clone() for x in (want_k, want_v))
    lcpp.DeviceRotary().Append(None, k, v, None, kc2, vc2, torch.tensor(slots, device="cuda"), i32(at), f, t,
                               layout=layout)
    assert torch.equal(kc2, kc) and torch.equal(vc2, vc)


# ---------------------------------------------------------------------------
# DevicePagedAttention
# ---------------------------------------------------------------------------
def make_table(rng, lens, width, block, spare=3):
    held = [-(-max(0, n) // block) for n in lens]
    order = rng.permutation(sum(held) + spare)
    table, at = np.full((len(lens), width), -1, np.int32), 0
    for r, n in enumerate(held):
        table[r, :min(n, width)] = order[at:at + n][:width]
        at += n
    return table, len(order)


def decode(L, q, kc, vc, table, lens, where="plain", scores=None, lse=True, **options):
    n, h, d = q.shape
    out = strided(torch.full_like(q, 3), where)
    d_lse = torch.full((n, h), 77.0, device="cuda") if lse else None
    slots = kc.shape[0] * kc.shape[1]
    after = None if scores is None else torch.full((slots,), -8.0, device="cuda")
    temp = L.alloc_temp(L.DevicePagedAttention.GetTempStorageBytes(n, h, kc.shape[2], d, 0 if scores is None else slots))
    temp.fill_(0xFF)  # NaN, should anything be read before it is written
    L.DevicePagedAttention().Decode(temp, strided(q, where), kc, vc, table, lens, out, n, d_lse_out=d_lse,
                                    d_scores=scores, d_scores_out=after, **options)
    return out, d_lse, after


def check_decode(L, q, kc, vc, table, lens, where="plain", scores=None, scale=None, window=0, softcap=0.0, decay=1.0):
    out, lse, after = decode(L, q, kc, vc, i32(table), i32(lens), where, scores, scale=scale, window=window,
                             softcap=softcap, score_decay=decay)
    s64 = None if scores is None else scores.double()
    want, size, want_lse, want_after = ref.attend(q.double(), kc.double(), vc.double(), torch.tensor(table), lens,
                                                  q.shape[2] ** -0.5 if scale is None else scale, window, softcap, s64,
                                                  decay)
    error = (out.double() - want).abs()
    assert (error <= 3e-5 * size + rounding(out.dtype, want.abs()) + 1e-30).all(), float((error - 3e-5 * size).max())
    empty = torch.isneginf(want_lse)
    assert torch.equal(torch.isneginf(lse), empty) and (out[empty] == 0).all()
    assert ((lse.double() - want_lse)[~empty].abs() <= 2e-5 * (1 + want_lse[~empty].abs())).all()
    if scores is not None:
        touched = torch.zeros_like(after, dtype=torch.bool)
        for r, n in enumerate(lens):
            token = np.arange(max(0, min(n, table.shape[1] * kc.shape[1])))
            page = table[r, token // kc.shape[1]].astype(np.int64)
            ok = (page >= 0) & (page < kc.shape[0])
            touched[torch.tensor((page * kc.shape[1] + token % kc.shape[1])[ok], device="cuda")] = True
        assert (after[~touched] == -8).all()
        error = (after.double() - want_after)[touched].abs()
        assert (error <= 4e-5 * want_after[touched].abs() + 1e-12).all()
    return out, lse, after


SHAPES = [  # (lengths, query heads, kv heads, dim, page size)
    ([1], 1, 1, 64, 1),
    ([0, 1, 15, 16, 17, 0], 4, 2, 128, 16),
    ([700], 32, 8, 128, 16),
    ([33, 250, 0, 64, 5], 7, 7, 80, 24),
    ([500, 3, 900], 20, 1, 64, 8),
    ([300, 129], 24, 2, 192, 32),
    ([260, 1, 77], 40, 1, 128, 64),
    ([90, 200], 16, 1, 256, 16),
    ([41, 300], 36, 2, 256, 7),
    ([100, 99], 70, 1, 64, 16),
    ([65, 130, 31], 6, 2, 8, 16),
    ([20, 50], 3, 1, 1, 4),
    ([77, 12], 5, 1, 250, 16),
]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("shape", range(len(SHAPES)))
@pytest.mark.parametrize("cache", LAYOUTS)
def test_decode(lcpp, kind, shape, cache):
    lens, h, kv, d, block = SHAPES[shape]
    rng = np.random.default_rng(shape)
    table, pages = make_table(rng, lens, max(lens) // block + 3, block)
    kc, vc = make_cache(kind, pages, block, kv, d, cache, seed=shape)
    q = randn(shape + 50, TYPES[kind], len(lens), h, d)
    scores = torch.rand(pages * block, device="cuda") if cache in ("tokens", "odd") else None
    check_decode(lcpp, q, kc, vc, table, lens, {"tokens": "plain", "odd": "odd"}.get(cache, "wide"), scores, decay=0.5)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("h,kv", [(8, 8), (16, 2), (12, 1)])
def test_decode_ragged_batch(lcpp, kind, d, h, kv):
    """Requests from empty to long ones, split over blocks in the middle of units, with and without a window."""
    rng = np.random.default_rng(d + h)
    lens = [int(n) for n in np.exp(rng.uniform(0, 8.3, 40))]
    lens[3] = lens[17] = lens[39] = 0
    table, pages = make_table(rng, lens, 5000 // 16, 16)
    kc, vc = make_cache(kind, pages, 16, kv, d, "tokens", seed=d)
    q = randn(d, TYPES[kind], len(lens), h, d)
    scores = torch.rand(pages * 16, device="cuda")
    check_decode(lcpp, q, kc, vc, table, lens, scores=scores)
    check_decode(lcpp, q, kc, vc, table, lens, window=257, scores=scores, decay=0.0)
    check_decode(lcpp, q, kc, vc, table, lens, window=1)
    check_decode(lcpp, q, kc, vc, table, lens, softcap=2.0, scale=0.3)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("n", [40_000, 150_001])
def test_decode_one_long_request(lcpp, kind, n):
    """One request over the whole GPU, under one kv head: every block has a part of it.  A lane adds up to 40 terms."""
    table, pages = make_table(np.random.default_rng(n), [n], n // 64 + 1, 64)
    kc, vc = make_cache(kind, pages, 64, 1, 64, "tokens")
    q = randn(1, TYPES[kind], 1, 8, 64)
    check_decode(lcpp, q, kc, vc, table, [n], scores=torch.zeros(pages * 64, device="cuda"))


@pytest.mark.parametrize("kind", KINDS)
def test_decode_many_requests(lcpp, kind):
    """More requests than a block has threads, most of them short, some empty."""
    rng = np.random.default_rng(4)
    lens = [int(n) for n in rng.integers(0, 40, 3001)]
    table, pages = make_table(rng, lens, 3, 16)
    kc, vc = make_cache(kind, pages, 16, 1, 64, "tokens")
    check_decode(lcpp, randn(4, TYPES[kind], 3001, 2, 64), kc, vc, table, lens,
                 scores=torch.rand(pages * 16, device="cuda"))


@pytest.mark.parametrize("kind", KINDS)
def test_decode_of_garbage_outside(lcpp, kind):
    """NaN, infinities and the lowest values in slots that no request holds, behind the last token of a page too, are
    never used; lengths below zero and past the table count as its ends; page ids out of range are passed over."""
    rng = np.random.default_rng(6)
    lens = [37, 5, 128, 90]
    table, pages = make_table(rng, lens, 8, 16)
    kc, vc = make_cache(kind, pages, 16, 2, 128, "tokens")
    held = np.zeros(pages * 16, bool)
    for r, n in enumerate(lens):
        held[(table[r, np.arange(n) // 16] * 16 + np.arange(n) % 16)] = True
    free = torch.tensor(np.nonzero(~held)[0], device="cuda")
    for x in (kc, vc):
        for i, bad in enumerate((float("nan"), float("inf"), -float("inf"), torch.finfo(x.dtype).min)):
            x.view(-1, 2, 128)[free[i::4]] = bad
    q = randn(9, TYPES[kind], 4, 8, 128)
    scores = torch.rand(pages * 16, device="cuda")
    args = dict(scores=scores, decay=1.0)

    def clean(x):
        return torch.nan_to_num(x, 0.0, 0.0, 0.0)

    def compare(lens, table):
        out, lse, after = decode(lcpp, q, kc, vc, i32(table), i32(lens), scores=scores)
        same = decode(lcpp, q, clean(kc), clean(vc), i32(table), i32(lens), scores=scores)
        assert torch.equal(out, same[0]) and torch.equal(lse, same[1]) and torch.equal(after, same[2])
        return out

    compare(lens, table)
    check_decode(lcpp, q, clean(kc), clean(vc), table, lens, **args)
    broken = table.copy()
    broken[0, 1], broken[1, 0], broken[2, 3], broken[2, 7] = -1, -5, pages, 2 ** 31 - 1
    compare(lens, broken)
    check_decode(lcpp, q, clean(kc), clean(vc), broken, lens, **args)
    check_decode(lcpp, q, clean(kc), clean(vc), broken, [-3, 5, 2 ** 31 - 1, 0], **args)


@pytest.mark.parametrize("kind", KINDS)
def test_decode_of_extreme_values(lcpp, kind):
    """Infinite and NaN logits act as in the formula on their own head only; logits that are all -inf leave the row
    empty; equal, far apart and large logits keep their digits."""
    dtype = TYPES[kind]
    n, d = 70, 64
    table = np.arange(5, dtype=np.int32)[None]
    kc, vc = make_cache(kind, 5, 16, 4, d, "tokens")
    q = torch.zeros(1, 4, d, dtype=dtype, device="cuda")
    q[0, :, 0] = 1
    kc[..., 0] = 0
    flat = kc.view(80, 4, d)
    flat[20, 0, 0] = float("nan")
    flat[20, 1, 0] = float("inf")
    flat[:70, 2, 0] = -float("inf")
    flat[:70, 3, 0] = torch.linspace(-200, 200, 70, device="cuda").to(dtype)
    out, lse, _ = decode(lcpp, q, kc, vc, i32(table), i32([n]), scale=1.0)
    assert out[0, :2].isnan().all() and lse[0, :2].isnan().all()
    assert (out[0, 2] == 0).all() and float(lse[0, 2]) == -math.inf
    want, size, want_lse, _ = ref.attend(q.double()[:, 3:], kc.double()[:, :, 3:], vc.double()[:, :, 3:],
                                         torch.tensor(table), [n], 1.0)
    assert ((out[0, 3].double() - want[0, 0]).abs() <= 1e-4 * size[0, 0] + rounding(dtype, want[0, 0].abs())).all()
    assert abs(float(lse[0, 3]) - float(want_lse)) <= 2e-5 * float(want_lse)
    # +inf in one token under one head of four that share keys
    kc, vc = make_cache(kind, 5, 16, 1, d, "tokens")
    kc[..., 0] = 0
    kc.view(80, d)[33, 0] = float("inf")
    q = randn(2, dtype, 1, 4, d)
    q[0, :, 0] = torch.tensor([0.5, -0.5, 0.0, 1.0])
    out, lse, _ = decode(lcpp, q, kc, vc, i32(table), i32([n]))
    assert out[0, [0, 2, 3]].isnan().all()  # inf - inf, 0 * inf
    q[0, 1, 0] = -0.5
    kept = kc.double().clone()
    kept.view(80, d)[33] = 0
    x = (kept.view(80, d)[:n] @ q[0, 1].double()) / 8
    x[33] = -math.inf
    p = torch.softmax(x, 0)
    want = p @ vc.view(80, d)[:n].double()
    size = p @ vc.view(80, d)[:n].double().abs()
    assert ((out[0, 1].double() - want).abs() <= 3e-5 * size + rounding(dtype, want.abs())).all()


@pytest.mark.parametrize("kind", KINDS)
def test_decode_rising_logits(lcpp, kind):
    """Logits that rise tile by tile, by less and by more than the reference may lag, and that fall again."""
    d, n = 64, 2000
    table = np.arange(125, dtype=np.int32)[None]
    kc, vc = make_cache(kind, 125, 16, 1, d, "tokens")
    kc.zero_()
    q = torch.zeros(1, 8, d, dtype=TYPES[kind], device="cuda")
    q[0, :, 0] = torch.tensor([1, 0.5, 0.25, 0.125, -1, -0.5, 2, 0])
    for step in (4.0, 0.05, 7.9, -3.0):
        ramp = torch.arange(2000, device="cuda") // 16 * step
        kc.view(-1, d)[:, 0] = ramp.to(kc.dtype)
        x = (kc.double().view(-1, d) @ q[0].double().T).T  # exact
        p = torch.softmax(x, 1)
        out, lse, _ = decode(lcpp, q, kc, vc, i32(table), i32([n]), scale=1.0)
        want, size = p @ vc.double().view(-1, d), p @ vc.double().view(-1, d).abs()
        # an argument of up to 2000 is off by half a unit of 2^-13 in base 2
        slack = 3e-5 + float(x.abs().max()) * 1.45 * 2.0 ** -23
        assert ((out[0].double() - want).abs() <= slack * size + rounding(out.dtype, want.abs())).all()
        want_lse = torch.logsumexp(x, 1)
        assert ((lse[0].double() - want_lse).abs() <= 2e-5 + 2e-7 * want_lse.abs()).all()


def test_decode_long_offsets(lcpp):
    """A cache of more than 2^32 elements: pages at its end."""
    pages, block, kv, d = 8200, 128, 32, 128  # 4.3e9 elements, 8.6 GB each for keys and values
    kc, vc = (torch.zeros(pages, block, kv, d, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    ids = np.array([[pages - 1, 3, pages - 2]], np.int32)
    small_k, small_v = make_cache("bf16", 3, block, kv, d, "tokens")
    kc[ids[0].tolist()], vc[ids[0].tolist()] = small_k, small_v
    q = randn(5, torch.bfloat16, 1, kv, d)
    out, lse, _ = decode(lcpp, q, kc, vc, i32(ids), i32([300]))
    same = decode(lcpp, q, small_k, small_v, i32([[0, 1, 2]]), i32([300]))
    assert torch.equal(out, same[0]) and torch.equal(lse, same[1])
    # and written to and moved there
    x = randn(6, torch.bfloat16, 2, kv, d)
    slots = torch.tensor([pages * block - 1, (pages - 2) * block], device="cuda")
    f = lcpp.DeviceRotary.Frequencies(0)
    lcpp.DeviceRotary().Append(None, x, x, None, kc, vc, slots, i32([0, 0]), f, 2)
    assert torch.equal(kc[pages - 1, block - 1], x[0]) and torch.equal(vc[pages - 2, 0], x[1])
    moves = torch.tensor([[[pages * block - 1, pages * block - 5]]], device="cuda")
    lcpp.DeviceCacheEviction().Move(moves, i32([1]), kc, vc, 1)
    assert torch.equal(kc[pages - 1, block - 5], x[0]) and torch.equal(vc[pages - 1, block - 5], x[0])


def test_decode_shared_pages(lcpp):
    """Requests that begin with the same pages, without scores."""
    rng = np.random.default_rng(8)
    kc, vc = make_cache("bf16", 40, 16, 2, 128, "tokens")
    table = rng.integers(0, 40, (6, 12)).astype(np.int32)
    table[:, :5] = table[0, :5]
    check_decode(lcpp, randn(3, torch.bfloat16, 6, 8, 128), kc, vc, table, [100, 80, 190, 16, 17, 81])


def test_decode_is_repeatable_and_in_place(lcpp):
    """Equal inputs give equal bits; scores may be updated where they are; another stream, a captured graph."""
    rng = np.random.default_rng(2)
    lens = [900, 20, 4000, 333]
    table, pages = make_table(rng, lens, 260, 16)
    kc, vc = make_cache("bf16", pages, 16, 2, 128, "heads")
    q = randn(1, torch.bfloat16, 4, 8, 128)
    scores = torch.rand(pages * 16, device="cuda")
    first = decode(lcpp, q, kc, vc, i32(table), i32(lens), scores=scores)
    for _ in range(3):
        again = decode(lcpp, q, kc, vc, i32(table), i32(lens), scores=scores)
        assert all(torch.equal(a, b) for a, b in zip(first, again))
    held = first[2] != -8
    d_table, d_lens, out = i32(table), i32(lens), torch.zeros_like(q)
    temp = lcpp.alloc_temp(lcpp.DevicePagedAttention.GetTempStorageBytes(4, 8, 2, 128, pages * 16))

    def call(scores, stream=None):
        lcpp.DevicePagedAttention().Decode(temp, q, kc, vc, d_table, d_lens, out, 4, d_scores=scores,
                                           d_scores_out=scores, stream=stream)
    own = scores.clone()
    call(own)
    assert torch.equal(own[held], first[2][held]) and torch.equal(own[~held], scores[~held])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    out.zero_()
    own = scores.clone()
    torch.cuda.synchronize()
    call(own, side)
    side.synchronize()
    assert torch.equal(out, first[0]) and torch.equal(own[held], first[2][held])
    out.zero_()
    own = scores.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(own)
    d_lens.copy_(i32([1, 20, 3999, 0]))  # a replay reads the lengths of its own time
    graph.replay()
    torch.cuda.synchronize()
    want = decode(lcpp, q, kc, vc, d_table, d_lens)
    assert torch.equal(out, want[0])


# ---------------------------------------------------------------------------
# DeviceCacheEviction
# ---------------------------------------------------------------------------
def check_plan(L, lens, table, scores, positions, evicted, budget, trigger, first, recent, block, pages, room, used=None,
               free=None, width=None):
    n = len(lens)
    d_table = i32(table)
    out_lens, out_evicted, counts = i32(np.full(n, -7)), i32(np.full(n, -7)), i32(np.full(n, -7))
    moves = torch.full((n, room, 2), -9, dtype=torch.int64, device="cuda")
    d_free = None if free is None else i32(free)
    d_used, used_out = (None, None) if used is None else (i32([used]), i32([-1]))
    L.DeviceCacheEviction().Plan(
        i32(lens), d_table, torch.tensor(scores, device="cuda"), out_lens, counts, moves, n, block, budget,
        trigger=trigger, keep_first=first, keep_recent=recent,
        d_positions=None if positions is None else i32(positions), d_evicted=None if evicted is None else i32(evicted),
        d_evicted_out=out_evicted, d_free_blocks=d_free, d_free_used=d_used, d_free_used_out=used_out)
    gone = np.zeros(n, np.int64) if evicted is None else evicted
    want_lens, want_evicted, want_moves, freed = ref.evict(lens, table, scores, positions, gone, budget, trigger, first,
                                                           recent, block, pages, room)
    np.testing.assert_array_equal(out_lens.cpu(), want_lens)
    np.testing.assert_array_equal(out_evicted.cpu(), want_evicted)
    np.testing.assert_array_equal(counts.cpu(), [len(m) for m in want_moves])
    want = np.full((n, room, 2), -9, np.int64)
    for r, m in enumerate(want_moves):
        want[r, :len(m)] = np.array(m, np.int64).reshape(-1, 2)
    np.testing.assert_array_equal(moves.cpu(), want)
    if free is not None:
        expect, before = np.array(free, np.int32), max(0, min(used, len(free)))
        at = before - len(freed)
        for i, page in enumerate(freed):
            if at + i >= 0:
                expect[at + i] = page
        np.testing.assert_array_equal(d_free.cpu(), expect)
        assert int(used_out) == max(0, at)
    return moves, counts, out_lens


def eviction_case(seed, lens, block, ties=False):
    rng = np.random.default_rng(seed)
    width = max(1, -(-max(lens) // block))
    table, pages = make_table(rng, lens, width, block)
    scores = np.exp(rng.uniform(-8, 3, pages * block)).astype(np.float32)
    if ties:
        scores = rng.choice(np.array([0.0, -0.0, 0.5, 1.0], np.float32), pages * block)
    evicted = rng.integers(0, 50, len(lens))
    positions = np.zeros(pages * block, np.int64)
    for r, n in enumerate(lens):
        slot = table[r, np.arange(n) // block].astype(np.int64) * block + np.arange(n) % block
        positions[slot] = np.sort(rng.permutation(n + evicted[r])[:n]) if n else 0
    return table, pages, scores, positions, evicted


@pytest.mark.parametrize("ties", [False, True])
@pytest.mark.parametrize("lens,block,budget,trigger,first,recent", [
    ([1, 2, 3, 10], 1, 2, 2, 0, 0),
    ([100, 64, 65, 0, 300, 63], 16, 64, 64, 4, 16),
    ([100, 64, 65, 80, 300, 63], 16, 64, 80, 0, 64),
    ([500, 1000, 999], 24, 333, 400, 333, 0),
    ([4096, 5000, 9000, 33], 64, 1, 1, 0, 0),
    ([4096, 5000, 9000, 33], 64, 4000, 4000, 7, 1000),
    ([50_000], 16, 4096, 4096, 4, 512),
    ([130_000, 100], 128, 60_000, 60_000, 10, 1000),
])
def test_plan(lcpp, ties, lens, block, budget, trigger, first, recent):
    table, pages, scores, positions, evicted = eviction_case(len(lens) + budget, lens, block, ties)
    room = max(1, min(budget, max(lens) - budget))
    free = np.arange(1000, 1000 + 2 * pages + 5)
    check_plan(lcpp, lens, table, scores, positions, evicted, budget, trigger, first, recent, block, pages, room,
               pages + 2, free)
    check_plan(lcpp, lens, table, scores, None, None, budget, trigger, first, recent, block, pages, room)


def test_plan_without_room_in_shared_memory(lcpp):
    """More tokens to a block than its shared memory holds keys for: many requests, of which one is very long."""
    lens = [200_000] + [3] * 400
    table, pages, scores, positions, evicted = eviction_case(1, lens, 64)
    check_plan(lcpp, lens, table, scores, positions, evicted, 70_000, 70_000, 5, 300, 64, pages, 70_000)
    table, pages, scores, positions, evicted = eviction_case(2, lens, 64, ties=True)
    check_plan(lcpp, lens, table, scores, positions, evicted, 70_000, 70_000, 5, 300, 64, pages, 70_000)


def test_plan_many_requests(lcpp):
    rng = np.random.default_rng(5)
    lens = [int(n) for n in rng.integers(0, 60, 3000)]
    table, pages, scores, positions, evicted = eviction_case(3, lens, 8)
    check_plan(lcpp, lens, table, scores, positions, evicted, 30, 32, 2, 8, 8, pages, 30, 2 * pages,
               np.arange(2 * pages + 1))


def test_plan_special_scores(lcpp):
    """NaN stays before +inf, both before the rest, negative scores and -inf leave first, both zeros are equal."""
    lens = [200, 200]
    table, pages, scores, positions, evicted = eviction_case(4, lens, 16)
    rng = np.random.default_rng(0)
    special = np.array([np.nan, np.inf, -np.inf, 0.0, -0.0, -1.5, 1e-45, 3.4e38], np.float32)
    scores = rng.choice(special, pages * 16).astype(np.float32)
    scores[rng.random(pages * 16) < 0.05] = -np.float32(np.nan)
    for budget in (10, 60, 120, 190):
        check_plan(lcpp, lens, table, scores, positions, evicted, budget, budget, 3, 5, 16, pages, 200)


def test_plan_leaves_requests(lcpp):
    """Broken page ids, too few entries for the moves, free lists that are too short, lengths past the table."""
    lens = [100, 90, 120, 100]
    table, pages, scores, positions, evicted = eviction_case(6, lens, 16)
    table[1, 2], table[2, 0] = -1, pages
    check_plan(lcpp, lens, table, scores, positions, evicted, 40, 40, 0, 4, 16, pages, 40, 3, np.arange(50))
    table[1, 2], table[2, 0] = 0, 0
    for room in (1, 10, 20, 26):
        check_plan(lcpp, lens, table, scores, positions, evicted, 40, 40, 0, 4, 16, pages, room, 200, np.arange(50))
    check_plan(lcpp, [100, -5, 2 ** 31 - 1, 100], table, scores, positions, evicted, 40, 40, 0, 4, 16, pages, 90)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("cache", LAYOUTS)
@pytest.mark.parametrize("block,heads,dim", [(16, 4, 128), (24, 3, 80), (5, 1, 7), (64, 8, 256)])
def test_move(lcpp, kind, cache, block, heads, dim):
    pages = 900 // block + 2
    kc, vc = make_cache(kind, pages, block, heads, dim, cache)
    rng = np.random.default_rng(block)
    slots = rng.permutation(pages * block)[:800].reshape(2, 400)
    counts, room = np.array([150, 0, 1, 200, -4]), 200
    moves = np.full((5, room, 2), 3, np.int64)  # entries past the counts are not looked at
    at = 0
    for r, c in enumerate(counts):
        c = max(0, c)
        moves[r, :c] = slots[:, at:at + c].T
        at += c
    moves[0, 5, 0], moves[0, 6, 1], moves[3, 0, 1] = -1, pages * block, 2 ** 50
    scores, positions = torch.rand(pages * block, device="cuda"), i32(rng.integers(0, 999, pages * block))
    want = [x.clone() for x in (kc, vc, scores, positions)]
    for r, c in enumerate(counts):
        for src, dst in moves[r, :max(0, c)]:
            if 0 <= src < pages * block and 0 <= dst < pages * block:
                for x, y in zip(want[:2], (kc, vc)):
                    x[dst // block, dst % block] = y[src // block, src % block]
                want[2][dst], want[3][dst] = scores[src], positions[src]
    lcpp.DeviceCacheEviction().Move(torch.tensor(moves, device="cuda"), i32(counts), kc, vc, 5, d_scores=scores,
                                    d_positions=positions)
    for got, expect in zip((kc, vc, scores, positions), want):
        assert torch.equal(got, expect)
    lcpp.DeviceCacheEviction().Move(torch.tensor(moves, device="cuda"), i32([0] * 5), kc, vc, 5)
    assert torch.equal(kc, want[0])


# ---------------------------------------------------------------------------
# Together
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("cache,order", [("f32", "tokens"), ("bf16", "heads")])
def test_serving_loop(lcpp, cache, order):
    """Prompts, then steps of Extend, Append, Decode and now and then Plan and Move, against a model that keeps each
    request's tokens in lists.  The choice of tokens to evict is read back: scores that differ in the last digits may
    order differently."""
    L = lcpp
    torch.manual_seed(0)
    n, h, kv, d, block, width, budget = 5, 8, 2, 64, 8, 16, 40
    dtype, pages = TYPES[cache], 60
    kc, vc = make_cache(cache, pages, block, kv, d, order)
    slots_total = pages * block
    free, used = i32(np.random.default_rng(1).permutation(pages)), i32([0])
    table = torch.full((n, width), -1, dtype=torch.int32, device="cuda")
    lens, evicted = i32(np.zeros(n)), i32(np.zeros(n))
    scores, slot_positions = torch.zeros(slots_total, device="cuda"), i32(np.zeros(slots_total))
    f = L.DeviceRotary.Frequencies(d)
    attention_temp = L.alloc_temp(L.DevicePagedAttention.GetTempStorageBytes(n, h, kv, d, slots_total))
    kept = [[] for _ in range(n)]  # (position, key, value) in the cache's order, 64 bits
    mass = [[] for _ in range(n)]
    rng = np.random.default_rng(3)
    for step in range(30):
        new = rng.integers(1, 30, n) if step == 0 else np.ones(n, np.int64)
        tokens = int(new.sum()) + 2
        temp = L.alloc_temp(L.DeviceBlockTable.GetTempStorageBytes(n, tokens))
        used_out, seq, starts = i32([0]), i32(np.zeros(n)), i32(np.zeros(n + 1))
        slots = torch.zeros(tokens, dtype=torch.int64, device="cuda")
        positions, requests = i32(np.zeros(tokens)), i32(np.zeros(tokens))
        L.DeviceBlockTable().Extend(temp, lens, i32(new), table, free, used, used_out, seq, starts, slots, positions,
                                    requests, n, block)
        assert (seq.cpu().numpy() == lens.cpu().numpy() + new).all()
        lens, used = seq, used_out
        q, k, v = (torch.randn(tokens, x, d, device="cuda").to(dtype) for x in (h, kv, kv))
        L.DeviceRotary().Append(q, k, v, q, kc, vc, slots, positions, f, tokens, d_token_request=requests,
                                d_position_offset=evicted, d_slot_positions=slot_positions, d_slot_scores=scores)
        last = (starts[1:] - 1).long()
        out = torch.empty(n, h, d, dtype=dtype, device="cuda")
        L.DevicePagedAttention().Decode(attention_temp, q[last], kc, vc, table, lens, out, n, d_scores=scores,
                                        d_scores_out=scores)
        at = starts.cpu().numpy()
        for r in range(n):
            # the model's own cache: keys as they were written (checked against the formula by test_append)
            s = slots[at[r]:at[r + 1]]
            for x in s.tolist():
                kept[r].append((int(slot_positions[x]), kc[x // block, x % block].double(), vc[x // block, x % block].double()))
                mass[r].append(0.0)
            keys, values = torch.stack([x[1] for x in kept[r]]), torch.stack([x[2] for x in kept[r]])
            x = torch.einsum("kgd,tkd->kgt", q[last[r]].double().view(kv, h // kv, d), keys) * d ** -0.5
            p = torch.softmax(x, -1)
            want = torch.einsum("kgt,tkd->kgd", p, values).reshape(h, d)
            size = torch.einsum("kgt,tkd->kgd", p, values.abs()).reshape(h, d)
            assert ((out[r].double() - want).abs() <= 3e-5 * size + rounding(dtype, want.abs())).all()
            mass[r] = [a + b for a, b in zip(mass[r], p.sum((0, 1)).tolist())]
            got = scores[(table[r].long()[torch.arange(len(mass[r]), device="cuda") // block] * block
                          + torch.arange(len(mass[r]), device="cuda") % block)]
            np.testing.assert_allclose(got.cpu(), mass[r], rtol=4e-5)
            total = len(kept[r]) + int(evicted[r])
            assert sorted(x[0] for x in kept[r])[-1] == total - 1
        if step % 4 == 3:
            counts, moves = i32(np.zeros(n)), torch.zeros(n, budget, 2, dtype=torch.int64, device="cuda")
            cut, gone, back = i32(np.zeros(n)), i32(np.zeros(n)), i32([0])
            ev = L.DeviceCacheEviction()
            ev.Plan(lens, table, scores, cut, counts, moves, n, block, budget - 8, trigger=budget - 1, keep_first=2,
                    keep_recent=6, d_positions=slot_positions, d_evicted=evicted, d_evicted_out=gone,
                    d_free_blocks=free, d_free_used=used, d_free_used_out=back)
            ev.Move(moves, counts, kc, vc, n, d_scores=scores, d_positions=slot_positions)
            for r in range(n):
                row = [int(table[r, i // block]) * block + i % block for i in range(len(kept[r]))]
                for src, dst in moves[r, :int(counts[r])].tolist():
                    kept[r][row.index(dst)], mass[r][row.index(dst)] = kept[r][row.index(src)], mass[r][row.index(src)]
                del kept[r][int(cut[r]):], mass[r][int(cut[r]):]
                for i, x in enumerate(kept[r]):
                    assert int(slot_positions[row[i]]) == x[0]
            lens, evicted, used = cut, gone, back
            held = sum(-(-int(x) // block) for x in lens)
            assert int(used) == held
            assert len(set(free[int(used):].tolist()) |
                       {int(p) for r in range(n) for p in table[r, :-(-int(lens[r]) // block)]}) == pages
    assert max(int(x) for x in evicted) > 0


@pytest.mark.parametrize("n", [4093, 4095, 4096, 8192, 16384, 32768])
def test_plan_where_a_run_fills_its_room(lcpp, n):
    """A block's keys take all of the shared memory that was asked for, and the last four are not always whole."""
    table, pages, scores, positions, evicted = eviction_case(n, [n], 4096)
    check_plan(lcpp, [n], table, scores, positions, evicted, n // 3, n // 2, 5, 100, 4096, pages, n // 3)


def test_plan_of_places(lcpp):
    """Without positions, places count: what left the requests before does not shift the last ones."""
    lens = [100, 64, 65, 300]
    table, pages, scores, _, _ = eviction_case(9, lens, 16)
    kept = check_plan(lcpp, lens, table, scores, None, None, 50, 64, 3, 20, 16, pages, 50)
    gone, gone_out, counts, cut = i32([7, 0, 900, 41]), i32([0] * 4), i32([0] * 4), i32([0] * 4)
    moves = torch.full((4, 50, 2), -9, dtype=torch.int64, device="cuda")
    lcpp.DeviceCacheEviction().Plan(i32(lens), i32(table), torch.tensor(scores, device="cuda"), cut, counts, moves, 4, 16,
                                    50, trigger=64, keep_first=3, keep_recent=20, d_evicted=gone, d_evicted_out=gone_out)
    assert torch.equal(moves, kept[0]) and torch.equal(counts, kept[1]) and torch.equal(cut, kept[2])
    assert torch.equal(gone_out, gone + i32(lens) - cut)


def test_steps_in_a_graph(lcpp):
    """Append, Decode, Plan and Move captured together on a stream of their own and replayed on other lengths, slots and
    values, next to the same calls one by one."""
    L, n, h, kv, d, block, width, budget = lcpp, 3, 8, 2, 64, 16, 8, 60
    pages = n * width
    table = i32(np.random.default_rng(2).permutation(pages).reshape(n, width))
    f = L.DeviceRotary.Frequencies(d)

    def state():
        kc, vc = make_cache("bf16", pages, block, kv, d, "tokens", 5)
        return dict(kc=kc, vc=vc, rows=randn(7, torch.bfloat16, n, (h + 2 * kv) * d), lens=i32([100, 20, 128]),
                    slots=torch.zeros(n, dtype=torch.int64, device="cuda"), positions=i32([99, 19, 127]),
                    gone=i32([3, 0, 9]), held=i32(np.arange(pages * block) % 140),
                    scores=randn(8, torch.float32, pages * block).abs(), q=torch.zeros(n, h, d, dtype=torch.bfloat16, device="cuda"),
                    out=torch.zeros(n, h, d, dtype=torch.bfloat16, device="cuda"), cut=i32([0] * n), counts=i32([0] * n),
                    gone_out=i32([0] * n), moves=torch.zeros(n, budget, 2, dtype=torch.int64, device="cuda"),
                    temp=L.alloc_temp(L.DevicePagedAttention.GetTempStorageBytes(n, h, kv, d, pages * block)))

    def step(s, stream=None):
        q, k, v = (x.unflatten(1, (-1, d)) for x in s["rows"].split((h * d, kv * d, kv * d), 1))
        L.DeviceRotary().Append(q, k, v, s["q"], s["kc"], s["vc"], s["slots"], s["positions"], f, n,
                                d_token_request=i32_rows, d_position_offset=s["gone"], d_slot_positions=s["held"],
                                d_slot_scores=s["scores"], stream=stream)
        L.DevicePagedAttention().Decode(s["temp"], s["q"], s["kc"], s["vc"], table, s["lens"], s["out"], n,
                                        d_scores=s["scores"], d_scores_out=s["scores"], stream=stream)
        L.DeviceCacheEviction().Plan(s["lens"], table, s["scores"], s["cut"], s["counts"], s["moves"], n, block, budget,
                                     keep_recent=8, d_positions=s["held"], d_evicted=s["gone"], d_evicted_out=s["gone_out"],
                                     stream=stream)
        L.DeviceCacheEviction().Move(s["moves"], s["counts"], s["kc"], s["vc"], n, d_scores=s["scores"],
                                     d_positions=s["held"], stream=stream)

    def other(s, lens, seed):
        at = i32(lens).long() - 1
        s["lens"].copy_(i32(lens))
        s["positions"].copy_(at)
        s["slots"].copy_(table.long().gather(1, (at // block)[:, None])[:, 0] * block + at % block)
        s["rows"].copy_(randn(seed, torch.bfloat16, n, (h + 2 * kv) * d))

    i32_rows = i32(np.arange(n))
    one, two = state(), state()
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    other(two, [100, 20, 128], 7)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=side):
        step(two, side)
    for lens, seed in (([100, 20, 128], 11), ([61, 128, 1], 12), ([60, 60, 90], 13)):
        other(one, lens, seed)
        other(two, lens, seed)
        step(one)
        graph.replay()
        torch.cuda.synchronize()
        for name in one:
            if name != "temp":
                assert torch.equal(one[name], two[name]), name
        assert one["cut"].tolist() == [min(x, budget) for x in lens]


@pytest.mark.parametrize("ties", [False, True])
def test_plan_of_more_tokens_than_a_cluster_holds(lcpp, ties):
    """Keys that no block of the largest cluster has room for are read again."""
    lens = [350_001, 3, 320_000]
    table, pages, scores, positions, evicted = eviction_case(11, lens, 128, ties)
    check_plan(lcpp, lens, table, scores, positions, evicted, 100_000, 100_000, 5, 300, 128, pages, 100_000)
    check_plan(lcpp, lens, table, scores, None, None, 330_000, 330_000, 0, 0, 128, pages, 20_001)


def test_decode_of_more_tokens_than_slots(lcpp):
    """Lengths far past the pages there are: outputs hold, scores of the requests in front too, no memory is left."""
    rng = np.random.default_rng(3)
    pages, block = 30, 16
    kc, vc = make_cache("bf16", pages, block, 2, 64, "tokens")
    table = np.full((3, 4000), -1, np.int32)
    ids = rng.permutation(pages)
    table[0, :7], table[1, :9], table[2, 3990:3996] = ids[:7], ids[7:16], ids[16:22]
    lens, q = [100, 60_000, 64_000], randn(1, torch.bfloat16, 3, 8, 64)
    out, lse, after = decode(lcpp, q, kc, vc, i32(table), i32(lens), scores=torch.zeros(pages * block, device="cuda"))
    plain = decode(lcpp, q, kc, vc, i32(table), i32(lens))
    assert torch.equal(out, plain[0]) and torch.equal(lse, plain[1])
    want, want_lse, _ = decode(lcpp, q[:1], kc, vc, i32(table[:1, :7]), i32(lens[:1]))
    assert ((out[0].float() - want[0].float()).abs() <= 6e-5 + 2 ** -7 * want[0].float().abs()).all()
    assert ((lse[0] - want_lse[0]).abs() <= 4e-5 * (1 + want_lse[0].abs())).all()
    first = torch.tensor(ids[:7].astype(np.int64), device="cuda")[:, None] * block + torch.arange(block, device="cuda")
    first = first.view(-1)[:100]
    total = float(after[first].double().sum())
    assert abs(total - 8) <= 8 * 4e-5  # each head hands out 1
    rest = torch.ones(pages * block, dtype=torch.bool, device="cuda")
    rest[first] = False
    assert (after[rest] == -8).all()


def test_broadcast_inputs(lcpp):
    """Inputs whose heads or tokens are one row repeated (stride 0); as outputs and as a written cache they are refused."""
    t, d = 37, 128
    x, f = randn(1, torch.bfloat16, t, 1, d), lcpp.DeviceRotary.Frequencies(d)
    positions = np.arange(t) * 3
    out = torch.zeros(t, 6, d, dtype=torch.bfloat16, device="cuda")
    lcpp.DeviceRotary().Forward(x.expand(t, 6, d), None, out, None, i32(positions), f, t)
    check_turn(out, x.expand(t, 6, d).contiguous(), positions, f, ref.HALF, 1.0)
    row = x[:1, :1].expand(t, 2, d)
    same = torch.zeros(t, 2, d, dtype=torch.bfloat16, device="cuda")
    lcpp.DeviceRotary().Backward(None, row, None, same, i32(positions), f, t)
    check_turn(same, row.contiguous(), positions, f, ref.HALF, 1.0, inverse=True)
    with pytest.raises(lcpp.LcppError):
        lcpp.DeviceRotary().Forward(out, None, x.expand(t, 6, d), None, i32(positions), f, t)

    rng = np.random.default_rng(0)
    lens = [100, 1, 60]
    table, pages = make_table(rng, lens, 10, 16)
    kc, vc = make_cache("bf16", pages, 16, 1, d, "tokens")
    shared = [c.expand(pages, 16, 4, d) for c in (kc, vc)]
    q = randn(2, torch.bfloat16, 3, 8, d)
    got = decode(lcpp, q, *shared, i32(table), i32(lens))
    want = decode(lcpp, q, *(c.contiguous() for c in shared), i32(table), i32(lens))
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    check_decode(lcpp, randn(3, torch.bfloat16, 1, 8, d).expand(3, 8, d), kc, vc, table, lens)
    one = randn(4, torch.bfloat16, 3, 4, d)
    slots = torch.tensor([0, 1, 2], device="cuda")
    with pytest.raises(lcpp.LcppError):
        lcpp.DeviceRotary().Append(None, one, one, None, *shared, slots, i32([0, 1, 2]), f, 3)
    with pytest.raises(lcpp.LcppError):
        lcpp.DeviceCacheEviction().Move(torch.zeros(3, 1, 2, dtype=torch.int64, device="cuda"), i32([0] * 3), *shared, 3)


def test_plan_without_room_for_moves(lcpp):
    """No moves at all fit: requests whose tokens happen to lie in front are cut, the others stay."""
    lens, budget, block = [90, 90], 40, 16
    table, pages, _, _, _ = eviction_case(12, lens, block)
    scores = np.zeros(pages * block, np.float32)
    for r in range(2):
        slot = table[r, np.arange(90) // block].astype(np.int64) * block + np.arange(90) % block
        scores[slot] = np.arange(90)[::-1] if r == 0 else np.arange(90)
    cut, counts = i32([-7, -7]), i32([-7, -7])
    moves = torch.zeros(2, 0, 2, dtype=torch.int64, device="cuda")
    lcpp.DeviceCacheEviction().Plan(i32(lens), i32(table), torch.tensor(scores, device="cuda"), cut, counts, moves, 2, block,
                                    budget)
    assert cut.tolist() == [budget, 90] and counts.tolist() == [0, 0]


def test_two_streams_at_once(lcpp):
    """Calls on two streams with temp storage of their own do not disturb one another."""
    rng = np.random.default_rng(4)
    lens = [3000, 700, 41, 1800]
    table, pages = make_table(rng, lens, 200, 16)
    kc, vc = make_cache("bf16", pages, 16, 2, 128, "tokens")
    qs = [randn(s, torch.bfloat16, 4, 16, 128) for s in range(2)]
    want = [decode(lcpp, q, kc, vc, i32(table), i32(lens), scores=torch.zeros(pages * 16, device="cuda")) for q in qs]
    streams = [torch.cuda.Stream() for _ in qs]
    d_table, d_lens, f = i32(table), i32(lens), lcpp.DeviceRotary.Frequencies(128)
    temps = [lcpp.alloc_temp(lcpp.DevicePagedAttention.GetTempStorageBytes(4, 16, 2, 128, pages * 16)) for _ in qs]
    outs, scores = [torch.zeros_like(q) for q in qs], [torch.full((pages * 16,), -8.0, device="cuda") for _ in qs]
    turned = [torch.zeros_like(q) for q in qs]
    torch.cuda.synchronize()
    for _ in range(20):
        for i, s in enumerate(streams):
            lcpp.DevicePagedAttention().Decode(temps[i], qs[i], kc, vc, d_table, d_lens, outs[i], 4, d_scores_out=scores[i],
                                               stream=s)
            lcpp.DeviceRotary().Forward(qs[i], None, turned[i], None, d_lens, f, 4, stream=s)
    torch.cuda.synchronize()
    for i in range(2):
        assert torch.equal(outs[i], want[i][0]) and torch.equal(scores[i], want[i][2])
        check_turn(turned[i], qs[i], np.array(lens), f, ref.HALF, 1.0)
