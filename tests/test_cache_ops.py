"""Refusals of DeviceRotary, DevicePagedAttention and DeviceCacheEviction, which need no device: bad arguments give a
status before any work is enqueued, the Python classes refuse tensors of another type, size, layout or place.  And the
frequencies, which the host computes."""
from __future__ import annotations

import ctypes
import math

import numpy as np
import pytest

torch = pytest.importorskip("torch")

BIG = 1 << 30


def p(i):
    return ctypes.c_void_p(0x10000000 * (i + 1))  # never dereferenced


def status(call, *args):
    return call(*(ctypes.byref(a) if isinstance(a, ctypes.Structure) else a for a in args))


def put(structure, changes):
    for name, value in changes.items():
        target, *path = name.split("."), None
        at = structure
        for part in target[:-1]:
            at = getattr(at, part)
        setattr(at, target[-1], value)
    return structure


def rotary_args(L, **changes):
    # 8 tokens, 4 and 2 heads of 64 columns, 32 of them turned
    q = L.HeadRows(0x10000000, 0x20000000, 256, 64, 256, 64, 4)
    k = L.HeadRows(0x30000000, 0x40000000, 128, 64, 128, 64, 2)
    return put(L.RotaryArgs(q, k, 0x50000000, 0x60000000, 0x70000000, 0x80000000, 8, 3, 64, 32, 0, 1.0, L.BF16), changes)


def cache(L):
    # 10 pages of 16 tokens, 2 heads of 64 columns
    return L.KVCache(0xA0000000, 0xB0000000, 2048, 128, 64, 10, 16, 2, 64, L.BF16)


def append_args(L, **changes):
    return put(L.CacheAppendArgs(cache(L), 0xC0000000, 128, 64, 0xD0000000, 0xE0000000, 0xF0000000), changes)


BAD_ROTARY = [
    {"head_dim": 0}, {"head_dim": 257}, {"rotary_dim": 31}, {"rotary_dim": 66}, {"layout": 2}, {"layout": -1},
    {"num_tokens": 1 << 31}, {"positions": None}, {"frequencies": None}, {"token_request": None},
    {"q.in_": None}, {"q.out": None}, {"positions": 0x50000002}, {"frequencies": 0x80000004}, {"q.in_": 0x10000001},
    {"token_request": 0x60000001}, {"position_offset": 0x70000002}, {"q.num_heads": 1 << 23},
    {"q.in_token_stride": 1 << 45},
    {"q.out_head_stride": 63}, {"q.out_token_stride": 255},  # rows that share memory
    {"q.out": 0x30000000},  # the keys
    {"q.out": 0x10000002},  # neither in place nor apart
    {"q.out": 0x10000000, "q.out_token_stride": 512},
    {"q.out": 0x40000000}, {"q.out": 0x50000000}, {"q.out": 0x80000000},
]


@pytest.mark.parametrize("change", BAD_ROTARY)
def test_rotary_refuses(lcpp, change):
    for call in (lcpp.lib().lcpp_rotary_forward, lcpp.lib().lcpp_rotary_backward):
        assert status(call, rotary_args(lcpp, **change), None) == lcpp.ERR_INVALID_ARG


def test_rotary_refuses_more(lcpp):
    lib = lcpp.lib()
    assert lib.lcpp_rotary_forward(None, None) == lcpp.ERR_INVALID_ARG
    assert status(lib.lcpp_rotary_forward, rotary_args(lcpp, dtype=lcpp.F64), None) == lcpp.ERR_UNSUPPORTED_DTYPE
    # nothing to do: no tokens, no heads
    assert status(lib.lcpp_rotary_forward, rotary_args(lcpp, num_tokens=0), None) == lcpp.OK
    assert status(lib.lcpp_rotary_forward, rotary_args(lcpp, **{"q.num_heads": 0, "k.num_heads": 0}), None) == lcpp.OK


@pytest.mark.parametrize("change", [
    {"cache.block_size": 0}, {"cache.num_kv_heads": 3}, {"cache.head_dim": 128}, {"cache.dtype": 2},
    {"cache.num_pages": 0xffffffff, "cache.block_size": 0xffffffff}, {"cache.k": None}, {"cache.v": None},
    {"cache.page_stride": 2047}, {"cache.token_stride": 127}, {"cache.head_stride": 63}, {"cache.page_stride": 1 << 45},
    {"v": None}, {"slots": None}, {"slots": 0xD0000004}, {"slot_positions": 0xE0000002}, {"slot_scores": 0xF0000001},
    {"v": 0xC0000001}, {"cache.k": 0xA0000001},
    {"cache.v": 0xA0000000}, {"cache.v": 0xA0000080},  # keys and values that share memory
    {"cache.k": 0x10000000}, {"cache.k": 0x20000000}, {"cache.k": 0xC0000000}, {"cache.v": 0xD0000000},
    {"slot_scores": 0xE0000010}, {"slot_scores": 0xA0000000}, {"slot_positions": 0x10000000},
])
def test_append_refuses(lcpp, change):
    assert status(lcpp.lib().lcpp_rotary_append, rotary_args(lcpp), append_args(lcpp, **change), None) == lcpp.ERR_INVALID_ARG


@pytest.mark.parametrize("change", [c for c in BAD_ROTARY if c != {"q.out": 0x40000000}])  # the keys go to the cache
def test_append_refuses_rotary(lcpp, change):
    assert status(lcpp.lib().lcpp_rotary_append, rotary_args(lcpp, **change), append_args(lcpp), None) == lcpp.ERR_INVALID_ARG
    assert status(lcpp.lib().lcpp_rotary_append, rotary_args(lcpp), None, None) == lcpp.ERR_INVALID_ARG


def attention_args(L, **changes):
    # 4 requests of up to 8 pages, 4 query heads
    return put(L.PagedAttentionArgs(cache(L), 0x10000000, 256, 64, 0x20000000, 256, 64, 0x30000000, 8, 8, 4, 0x40000000,
                                    4, 0, 0.125, 0.0, 0x50000000, 0x60000000, 0x70000000, 1.0), changes)


@pytest.mark.parametrize("change", [
    {"num_requests": (1 << 20) + 1}, {"num_heads": 0}, {"num_heads": 5}, {"num_heads": 1 << 17}, {"table_stride": 7},
    {"table_stride": 1 << 45}, {"cache.block_size": 0}, {"cache.num_kv_heads": 0}, {"cache.head_dim": 0},
    {"cache.head_dim": 257}, {"softcap": -1.0}, {"softcap": math.nan}, {"softcap": math.inf}, {"scale": math.nan},
    {"scale": math.inf}, {"score_decay": math.nan}, {"q": None}, {"out": None}, {"block_table": None},
    {"seq_lens": None}, {"cache.k": None}, {"cache.v": None}, {"slot_scores_out": None}, {"q": 0x10000001},
    {"out": 0x20000001}, {"cache.v": 0xB0000001}, {"block_table": 0x30000002}, {"seq_lens": 0x40000001},
    {"lse_out": 0x50000002}, {"slot_scores": 0x60000001}, {"slot_scores_out": 0x70000002}, {"out_head_stride": 63},
    {"out_request_stride": 255}, {"out_request_stride": 0}, {"q_head_stride": 1 << 45},
    {"out": 0x10000000}, {"out": 0xA0000000}, {"out": 0xB0000000}, {"out": 0x30000000}, {"out": 0x40000000},
    {"lse_out": 0x20000004}, {"lse_out": 0x60000000}, {"slot_scores_out": 0x60000004}, {"slot_scores_out": 0xB0000000},
])
def test_decode_refuses(lcpp, change):
    call = lcpp.lib().lcpp_paged_attention_decode
    assert status(call, p(15), BIG, attention_args(lcpp, **change), None) == lcpp.ERR_INVALID_ARG


def test_decode_refuses_temp(lcpp):
    call = lcpp.lib().lcpp_paged_attention_decode
    a = attention_args(lcpp)
    assert status(call, None, BIG, a, None) == lcpp.ERR_INVALID_ARG
    assert status(call, ctypes.c_void_p(0x100000010), BIG, a, None) == lcpp.ERR_INVALID_ARG
    assert status(call, p(15), BIG, None, None) == lcpp.ERR_INVALID_ARG
    assert status(call, p(15), 4096, a, None) == lcpp.ERR_TEMP_TOO_SMALL
    assert status(call, ctypes.c_void_p(0x20000000), BIG, a, None) == lcpp.ERR_INVALID_ARG  # the output
    assert status(call, p(15), BIG, attention_args(lcpp, **{"cache.dtype": lcpp.F64}), None) == lcpp.ERR_UNSUPPORTED_DTYPE
    assert status(call, p(15), 0, attention_args(lcpp, num_requests=0), None) == lcpp.OK
    size = lcpp.DevicePagedAttention.GetTempStorageBytes
    assert size(4, 4, 2, 64, 160) > size(4, 4, 2, 64) > 0
    assert size(4, 64, 2, 64) >= size(4, 4, 2, 64)
    for bad in ((4, 5, 2, 64), (4, 0, 1, 64), (4, 4, 0, 64), (4, 4, 2, 0), (4, 4, 2, 257), ((1 << 20) + 1, 4, 2, 64),
                (4, 4, 2, 64, 1 << 40)):
        with pytest.raises(lcpp.LcppError):
            size(*bad)


def evict_args(L, **changes):
    return put(L.CacheEvictArgs(0x10000000, 0x20000000, 8, 8, 4, 10, 16, 0x30000000, 0x40000000, 0x50000000, 32, 40, 4, 8,
                                32, 0x60000000, 0x70000000, 0x80000000, 0x90000000, 32, 0xA0000000, 0xB0000000,
                                0xC0000000, 50), changes)


@pytest.mark.parametrize("change", [
    {"block_size": 0}, {"budget": 0}, {"budget": 1 << 31, "trigger": 1 << 31}, {"trigger": 31}, {"keep_first": 25},
    {"keep_first": 0xffffffff, "keep_recent": 0xffffffff}, {"num_requests": (1 << 20) + 1}, {"table_stride": 7},
    {"moves_stride": 31}, {"num_pages": 0xffffffff, "block_size": 0xffffffff}, {"seq_lens": None}, {"block_table": None},
    {"slot_scores": None}, {"seq_lens_out": None}, {"move_counts_out": None}, {"moves_out": None}, {"free_used": None},
    {"free_used_out": None}, {"free_blocks": None}, {"moves_out": 0x90000008}, {"seq_lens": 0x10000002},
    {"slot_positions": 0x40000001}, {"free_blocks": 0xA0000002},
    {"seq_lens_out": 0x10000000}, {"seq_lens_out": 0x30000000}, {"evicted_out": 0x50000004}, {"move_counts_out": 0x20000000},
    {"moves_out": 0x20000070}, {"free_used_out": 0xB0000000}, {"free_blocks": 0x20000040}, {"free_blocks": 0x10000000},
    {"free_used": 0xA0000004}, {"moves_out": 0x60000000},
])
def test_plan_refuses(lcpp, change):
    assert status(lcpp.lib().lcpp_cache_evict_plan, evict_args(lcpp, **change), None) == lcpp.ERR_INVALID_ARG
    assert lcpp.lib().lcpp_cache_evict_plan(None, None) == lcpp.ERR_INVALID_ARG


@pytest.mark.parametrize("change", [
    {"block_size": 0}, {"k": None}, {"v": None}, {"v": 0xA0000000}, {"page_stride": 100}, {"k": 0xA0000001},
])
def test_move_refuses(lcpp, change):
    call, c = lcpp.lib().lcpp_cache_evict_move, put(cache(lcpp), change)
    assert status(call, c, p(0), 32, 32, p(1), 4, p(2), p(3), None) == lcpp.ERR_INVALID_ARG


def test_move_refuses_more(lcpp):
    call, c = lcpp.lib().lcpp_cache_evict_move, cache(lcpp)
    good = (p(0), 32, 32, p(1), 4, p(2), p(3))
    for i, value in ((0, None), (0, ctypes.c_void_p(0x10000008)), (1, 31), (3, None), (3, ctypes.c_void_p(0x20000002)),
                     (4, (1 << 20) + 1), (5, ctypes.c_void_p(0x30000001)), (6, ctypes.c_void_p(0x40000002)),
                     (5, p(3)), (5, p(0)), (6, ctypes.c_void_p(0xA0000000)), (5, ctypes.c_void_p(0xB0000010))):
        bad = good[:i] + (value,) + good[i + 1:]
        assert status(call, c, *bad, None) == lcpp.ERR_INVALID_ARG, (i, value)
    assert status(call, None, *good, None) == lcpp.ERR_INVALID_ARG
    assert status(call, put(cache(lcpp), {"dtype": lcpp.F64}), *good, None) == lcpp.ERR_UNSUPPORTED_DTYPE
    assert status(call, c, p(0), 32, 32, p(1), 0, None, None, None) == lcpp.OK
    assert status(call, c, None, 0, 0, p(1), 4, None, None, None) == lcpp.OK


def test_structures_are_packed_as_they_lie(lcpp):
    """The Python classes put arguments together in one step; it has to agree with the structures' layout."""
    for make, pack in ((rotary_args, lcpp._pack_rotary), (append_args, lcpp._pack_append),
                       (attention_args, lcpp._pack_attention), (evict_args, lcpp._pack_evict)):
        a = make(lcpp)

        def values(s):
            for name, kind in s._fields_:
                x = getattr(s, name)
                if isinstance(x, ctypes.Structure):
                    yield from values(x)
                else:
                    yield x or 0
        packed = pack(*values(a))
        assert len(packed) == ctypes.sizeof(a)
        assert bytes(a) == packed


def test_python_refuses_numbers(lcpp):
    """Numbers that the call's fields do not hold."""
    fields = [1, 1, 64, 64, 64, 2, 16, 1, 64, 0]
    assert len(lcpp._pack_cache(*fields)) == ctypes.sizeof(lcpp.KVCache)
    for at, value in ((5, -1), (6, 2 ** 32), (2, -64), (0, 2 ** 64), (8, 1.5)):
        with pytest.raises(lcpp.LcppError):
            lcpp._pack_cache(*(value if i == at else x for i, x in enumerate(fields)))


def test_python_refuses_tensors(lcpp):
    """Tensors of the host, of other types, shapes and layouts."""
    L, bf, i32 = lcpp, torch.bfloat16, torch.int32
    q, k = torch.zeros(8, 4, 64, dtype=bf), torch.zeros(8, 2, 64, dtype=bf)
    pos, f, slots = torch.zeros(8, dtype=i32), torch.zeros(16, dtype=torch.float64), torch.zeros(8, dtype=torch.int64)
    kc, vc = torch.zeros(10, 16, 2, 64, dtype=bf), torch.zeros(10, 16, 2, 64, dtype=bf)
    table, lens, lse = torch.zeros(4, 8, dtype=i32), torch.zeros(4, dtype=i32), torch.zeros(4, 4)
    temp = torch.zeros(1, dtype=torch.uint8)
    rot, att, ev = L.DeviceRotary(), L.DevicePagedAttention(), L.DeviceCacheEviction()
    calls = [
        lambda: rot.Forward(q, k, q, k, pos, f, 8),  # host tensors
        lambda: rot.Forward(None, None, None, None, pos, f, 8),
        lambda: rot.Forward(q[0], k, q, k, pos, f, 8),
        lambda: rot.Forward(q, k.float(), q, k, pos, f, 8),
        lambda: rot.Forward(q, k[:, :, :32], q, k, pos, f, 8),
        lambda: rot.Forward(q, k, q[:7], k, pos, f, 8),
        lambda: rot.Forward(q, k, q[:, :3], k, pos, f, 8),
        lambda: rot.Forward(q.transpose(1, 2).contiguous().transpose(1, 2), k, q, k, pos, f, 8),
        lambda: rot.Append(q, k, k, q, kc, vc, slots, pos, f, 8),
        lambda: rot.Append(q, k, k, q, kc, vc[:9], slots, pos, f, 8),
        lambda: rot.Append(q, k, k, q, kc[0], vc[0], slots, pos, f, 8),
        lambda: rot.Append(q, k, k, q, kc, vc.transpose(1, 2).contiguous().transpose(1, 2), slots, pos, f, 8),
        lambda: att.Decode(temp, q[:4], kc, vc, table, lens, q[4:], 4),
        lambda: att.Decode(temp, q[:4], kc, vc.float(), table, lens, q[4:], 4),
        lambda: ev.Plan(lens, table, lse.view(-1), lens, lens, slots.view(4, 1, 2), 4, 16, 2),
        lambda: ev.Plan(lens, table, lse.view(-1), lens, lens, slots.view(4, 2), 4, 16, 2),
        lambda: ev.Plan(lens, table.float(), lse.view(-1), lens, lens, slots.view(4, 1, 2), 4, 16, 2),
        lambda: ev.Move(slots.view(4, 1, 2), lens, kc, vc, 4),
        lambda: ev.Move(slots.view(4, 1, 2).int(), lens, kc, vc, 4),
    ]
    for i, call in enumerate(calls):
        with pytest.raises(L.LcppError):
            call()
    with pytest.raises(TypeError):
        rot.Forward(q.double(), None, q.double(), None, pos, f, 8)


# ---------------------------------------------------------------------------
# Frequencies
# ---------------------------------------------------------------------------
def frequencies(L, dim, *args):
    out = (ctypes.c_double * max(1, dim // 2))(*[-7.0] * max(1, dim // 2))
    L.check(L.lib().lcpp_rotary_frequencies(out, dim, *args), "frequencies")
    return np.array(out[:dim // 2])


@pytest.mark.parametrize("dim", [2, 6, 64, 128, 250, 256])
@pytest.mark.parametrize("base", [100.0, 1e4, 5e5])
def test_frequencies(lcpp, dim, base):
    i = np.arange(dim // 2)
    plain = base ** (-2.0 * i / dim)
    np.testing.assert_allclose(frequencies(lcpp, dim, base, lcpp.ROTARY_PLAIN, 1, 0, 0, 0), plain, rtol=1e-14)
    np.testing.assert_allclose(frequencies(lcpp, dim, base, lcpp.ROTARY_LINEAR, 8, 0, 0, 0), plain / 8, rtol=1e-14)
    if dim > 2:
        got = frequencies(lcpp, dim, base, lcpp.ROTARY_BASE, 4, 0, 0, 0)
        np.testing.assert_allclose(got, (base * 4 ** (dim / (dim - 2))) ** (-2.0 * i / dim), rtol=1e-13)
        assert abs(got[-1] - plain[-1] / 4) <= 1e-13 * plain[-1]  # the slowest one is stretched by the factor
    got = frequencies(lcpp, dim, base, lcpp.ROTARY_BY_ROTATIONS, 8, 8192, 1, 4)
    turns = 8192 * plain / (2 * math.pi)
    for f, was, n in zip(got, plain, turns):
        if n >= 4:
            assert f == pytest.approx(was, rel=1e-14)
        elif n <= 1:
            assert f == pytest.approx(was / 8, rel=1e-14)
        else:
            share = (n - 1) / 3
            assert f == pytest.approx(share * was + (1 - share) * was / 8, rel=1e-13)


def test_frequencies_refuse(lcpp):
    call, out = lcpp.lib().lcpp_rotary_frequencies, (ctypes.c_double * 128)()
    good = (out, 64, 1e4, lcpp.ROTARY_BY_ROTATIONS, 8.0, 8192.0, 1.0, 4.0)
    assert call(*good) == lcpp.OK and call(out, 0, 1e4, 0, 1.0, 0.0, 0.0, 0.0) == lcpp.OK
    for i, value in ((0, None), (1, 63), (1, 258), (2, 0.0), (2, -1.0), (2, math.inf), (2, math.nan), (3, 4), (3, -1),
                     (4, 0.5), (4, math.nan), (4, math.inf), (5, 0.0), (5, math.inf), (6, 0.0), (6, 4.0), (7, math.inf)):
        assert call(*(good[:i] + (value,) + good[i + 1:])) == lcpp.ERR_INVALID_ARG, (i, value)
    assert call(out, 2, 1e4, lcpp.ROTARY_BASE, 8.0, 0.0, 0.0, 0.0) == lcpp.ERR_INVALID_ARG
