"""The paged cache's operators where numbers end: infinite values, sums beyond 32 bits, rows that are empty by their
logits.  References and tolerances as in tests/test_cache_ops_gpu.py."""
from __future__ import annotations

import math

import numpy as np
import pytest

import cache_ref as ref
from test_cache_ops_gpu import (KINDS, TYPES, check_decode, check_plan, decode, eviction_case, i32, make_cache, make_table,
                                randn)

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

MIXES = {
    # units that a block has whole and units that blocks divide; some empty ones
    "ragged": [int(n) for n in np.random.default_rng(0).integers(0, 90, 220)] + [900, 0, 2500],
    "one": [70],
    "long": [20_000],
}


def compare(out, lse, q, kc, vc, table, lens, **options):
    """Infinities and NaN where the formula has them, and its numbers elsewhere."""
    want, size, want_lse, _ = ref.attend(q.double(), kc.double(), vc.double(), torch.tensor(table), lens,
                                         options.pop("scale", q.shape[2] ** -0.5), **options)
    out = out.double()
    assert torch.equal(out.isnan(), want.isnan())
    assert torch.equal(torch.where(out.isinf(), out, 0), torch.where(want.isinf(), want, 0))
    sure = want.isfinite()
    error = (out - want)[sure].abs()
    assert (error <= (3e-5 * size + torch.finfo(q.dtype).eps / 2 * want.abs())[sure] + 2.0 ** -25).all()
    assert ((lse.double() - want_lse)[want_lse.isfinite()].abs() <= 2e-5 * (1 + want_lse[want_lse.isfinite()].abs())).all()
    return want


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("mix", MIXES)
@pytest.mark.parametrize("h,kv,d,block,options", [(8, 2, 64, 16, {}), (3, 1, 128, 24, {"window": 60}),
                                                  (40, 1, 128, 16, {"softcap": 3.0}), (6, 3, 250, 7, {})])
def test_decode_of_infinite_values(lcpp, kind, mix, h, kv, d, block, options):
    """A value of +inf or -inf that is looked at gives its column that infinity, both of them or a NaN give NaN; other
    columns, heads and requests keep their numbers."""
    lens = MIXES[mix]
    rng = np.random.default_rng(d + len(lens))
    table, pages = make_table(rng, lens, max(lens) // block + 2, block)
    kc, vc = make_cache(kind, pages, block, kv, d, "tokens", seed=d)
    for r, n in enumerate(lens):
        if not n or (r % 3 and mix == "ragged"):
            continue
        # columns 0, 1 and 5 of several tokens: inf, -inf, NaN; column 3: both infinities; the last: inf in the first token
        for column, token, value in ((0, n - 1, math.inf), (0, n // 2, math.inf), (1, n - 1, -math.inf),
                                     (3, n - 1, math.inf), (3, n // 3, -math.inf), (5, n // 2, math.nan),
                                     (d - 1, 0, math.inf)):
            vc[table[r, token // block], token % block, (r + column) % kv, column] = value
    q = randn(d + 1, TYPES[kind], len(lens), h, d)
    out, lse, _ = decode(lcpp, q, kc, vc, i32(table), i32(lens), **options)
    want = compare(out, lse, q, kc, vc, table, lens, **options)
    assert want.isinf().any() and want.isfinite().any()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("mix", MIXES)
def test_decode_of_the_largest_values(lcpp, kind, mix):
    """The mean of the type's largest numbers is a number, although their sum is none in 32 bits; equal ones give
    themselves."""
    lens, h, kv, d, block = MIXES[mix], 8, 2, 64, 16
    table, pages = make_table(np.random.default_rng(1), lens, max(lens) // block + 2, block)
    kc, vc = make_cache(kind, pages, block, kv, d, "tokens", seed=3)
    top = torch.finfo(TYPES[kind]).max
    vc[..., 0], vc[..., 1] = top, -top
    vc[..., 2] = torch.where(vc[..., 2] > 0, top, -top)
    vc[..., 3] *= top / 8
    q = randn(4, TYPES[kind], len(lens), h, d)
    out, lse, _ = decode(lcpp, q, kc, vc, i32(table), i32(lens))
    live = torch.tensor(lens, device="cuda") > 0
    assert (out[live][..., 0] == top).all() and (out[live][..., 1] == -top).all() and out.isfinite().all()
    compare(out, lse, q, kc, vc, table, lens)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("mix", MIXES)
def test_decode_of_rows_without_weight(lcpp, kind, mix):
    """A row whose logits are all -inf gets zeros and lse -inf, whatever its values hold."""
    lens, d, block = MIXES[mix], 64, 16
    table, pages = make_table(np.random.default_rng(2), lens, max(lens) // block + 2, block)
    kc, vc = make_cache(kind, pages, block, 2, d, "tokens", seed=5)
    q = randn(6, TYPES[kind], len(lens), 4, d)
    kc[..., 0, 0] = -math.inf  # of the first kv head
    q[..., 0] = 1
    plain = vc.clone()
    for i, bad in enumerate((math.inf, -math.inf, math.nan)):
        vc[..., 0, i::4] = bad
    out, lse, _ = decode(lcpp, q, kc, vc, i32(table), i32(lens))
    assert (out[:, :2] == 0).all() and (lse[:, :2] == -math.inf).all()
    other, other_lse, _ = decode(lcpp, q, kc, plain, i32(table), i32(lens))
    assert torch.equal(out[:, 2:], other[:, 2:]) and torch.equal(lse, other_lse)


@pytest.mark.parametrize("kind", KINDS)
def test_heads_side_by_side_in_each_head(lcpp, kind):
    """Queries, keys and values of a head next to one another: outputs beside inputs and beside one another."""
    t, h, d = 33, 4, 64
    rows = randn(1, TYPES[kind], t, h, 3, d)
    before, positions, f = rows.clone(), i32(np.arange(t) * 7), lcpp.DeviceRotary.Frequencies(d)
    want_q, want_k = (before[:, :, i].contiguous() for i in range(2))
    lcpp.DeviceRotary().Forward(want_q, want_k, want_q, want_k, positions, f, t)
    lcpp.DeviceRotary().Forward(rows[:, :, 0], rows[:, :, 1], rows[:, :, 0], rows[:, :, 1], positions, f, t)
    assert torch.equal(rows[:, :, 0], want_q) and torch.equal(rows[:, :, 1], want_k)
    assert torch.equal(rows[:, :, 2], before[:, :, 2])
    # the turned queries into the place of the values
    lcpp.DeviceRotary().Forward(before[:, :, 0], None, before[:, :, 2], None, positions, f, t)
    assert torch.equal(before[:, :, 2], want_q)

    lens, block = [70, 0, 9], 16
    table, pages = make_table(np.random.default_rng(0), lens, 6, block)
    kc, vc = make_cache(kind, pages, block, 2, d, "tokens")
    both = randn(3, TYPES[kind], 3, h, 2, d)
    q = both[:, :, 0].contiguous()
    want, lse, _ = decode(lcpp, q, kc, vc, i32(table), i32(lens))
    temp = lcpp.alloc_temp(lcpp.DevicePagedAttention.GetTempStorageBytes(3, h, 2, d))
    lcpp.DevicePagedAttention().Decode(temp, both[:, :, 0], kc, vc, i32(table), i32(lens), both[:, :, 1], 3)
    assert torch.equal(both[:, :, 1], want) and torch.equal(both[:, :, 0], q)
    for bad in (both.view(3, h, 2 * d)[..., d // 2:d // 2 + d], both.view(3, 2 * h, d)[:, h - 1:2 * h - 1]):
        with pytest.raises(lcpp.LcppError):
            lcpp.DevicePagedAttention().Decode(temp, both[:, :, 0], kc, vc, i32(table), i32(lens), bad, 3)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("block", [16, 7])
def test_cache_without_pages(lcpp, kind, block):
    """No page at all, whatever the tables and lengths say: rows are empty, nothing is written, nothing moves."""
    kc, vc = (torch.zeros(0, block, 2, 64, dtype=TYPES[kind], device="cuda") for _ in range(2))
    table, lens = i32([[0, 3, -1], [5, 1, 0]]), i32([40, 9])
    none = torch.zeros(0, device="cuda")
    for scores in (None, none):
        out, lse, _ = decode(lcpp, randn(1, TYPES[kind], 2, 4, 64), kc, vc, table, lens, scores=scores)
        assert (out == 0).all() and (lse == -math.inf).all()
    x, f = randn(2, TYPES[kind], 3, 2, 64), lcpp.DeviceRotary.Frequencies(64)
    q = torch.full_like(x, 5)
    lcpp.DeviceRotary().Append(x, x, x, q, kc, vc, torch.tensor([0, 1, -1], device="cuda"), i32([0, 1, 2]), f, 3)
    assert (q == 5).all()  # tokens whose slot lies outside the cache are left out
    lcpp.DeviceCacheEviction().Move(torch.zeros(2, 1, 2, dtype=torch.int64, device="cuda"), i32([1, 1]), kc, vc, 2)
    cut, counts = i32([-7, -7]), i32([-7, -7])
    lcpp.DeviceCacheEviction().Plan(i32([20, 9]), table, none, cut, counts,
                                    torch.zeros(2, 4, 2, dtype=torch.int64, device="cuda"), 2, block, 4)
    assert cut.tolist() == [20, 9] and counts.tolist() == [0, 0]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("block", [1, 7, 24])
def test_windows_that_begin_inside_pages(lcpp, kind, block):
    """A window's first tile has rows before it, and rows in several pages; with scores."""
    lens = [300, 1, 9, 0, 158, 33, 64]
    table, pages = make_table(np.random.default_rng(block), lens, max(lens) // block + 2, block)
    kc, vc = make_cache(kind, pages, block, 2, 80, "heads", seed=block)
    q, scores = randn(block, TYPES[kind], len(lens), 6, 80), torch.rand(pages * block, device="cuda")
    for window in (1, 9, 17, 23, 100, 299):
        check_decode(lcpp, q, kc, vc, table, lens, scores=scores, window=window, decay=0.5)


@pytest.mark.parametrize("ties", [False, True])
@pytest.mark.parametrize("lens", [[2048, 2049, 4096, 3], [5000, 4999], [50_000, 20_000]])
def test_plan_of_pages_of_one_token(lcpp, lens, ties):
    """Runs of more pages than a block keeps the ids of, which are then read where they are needed, and of just as many."""
    table, pages, scores, positions, evicted = eviction_case(len(lens), lens, 1, ties)
    n = min(x for x in lens if x > 3)
    check_plan(lcpp, lens, table, scores, positions, evicted, n // 2, n - 1, 5, 100, 1, pages, max(lens), 2 * pages,
               np.arange(2 * pages + 1))
    table[0, lens[0] - 2] = -1  # a request with a broken page stays as it is
    check_plan(lcpp, lens, table, scores, None, None, n // 2, n - 1, 5, 100, 1, pages, max(lens))


@pytest.mark.parametrize("ties", [False, True])
def test_plan_of_more_keys_than_a_block_holds(lcpp, ties):
    """A long request among many short ones: keys past what the largest cluster's blocks have room for are read again."""
    lens = [330_000] + [3] * 200
    table, pages, scores, positions, evicted = eviction_case(1, lens, 64, ties)
    check_plan(lcpp, lens, table, scores, positions, evicted, 70_000, 70_000, 5, 300, 64, pages, 70_000)
