"""The model-step operators' refusals, which need no device: every bad argument gives a status before any
work is enqueued, and the Python classes refuse tensors of the wrong type, size or layout."""
from __future__ import annotations

import ctypes

import pytest

torch = pytest.importorskip("torch")

BIG = 1 << 20


def p(i):
    return ctypes.c_void_p(0x100000 * (i + 1))  # never dereferenced


def table_args(lcpp, **changes):
    a = lcpp.BlockTableArgs(0x1000000, 0x2000000, 0x3000000, 8, 8, 4, 16, 10, 0x4000000, 0x5000000, 0x6000000,
                            0x7000000, 0x8000000, 0x9000000, 0xA000000, 0xB000000, 32)
    for name, value in changes.items():
        setattr(a, name, value)
    return a


@pytest.mark.parametrize("change", [
    {"block_size": 0}, {"max_tokens": (1 << 31) - 1}, {"num_requests": (1 << 20) + 1}, {"table_stride": 7},
    {"context_lens": None}, {"block_table": None}, {"free_blocks": None}, {"free_used_out": None},
    {"seq_lens_out": None}, {"query_starts_out": None}, {"slots_out": None},
    {"slots_out": 0x9000004}, {"positions_out": 0xA000002}, {"new_lens": 0x2000001},
    {"free_used_out": 0x5000000}, {"free_used_out": 0x1000008}, {"seq_lens_out": 0x1000000},
    {"seq_lens_out": 0x1000004}, {"seq_lens_out": 0x2000000},
])
def test_block_table_refuses(lcpp, change):
    a = table_args(lcpp, **change)
    assert lcpp.lib().lcpp_block_table_extend(p(0), BIG, a, None) == lcpp.ERR_INVALID_ARG


def test_block_table_refuses_temp(lcpp):
    lib = lcpp.lib()
    assert lib.lcpp_block_table_extend(None, BIG, table_args(lcpp), None) == lcpp.ERR_INVALID_ARG
    assert lib.lcpp_block_table_extend(ctypes.c_void_p(0x100010), BIG, table_args(lcpp), None) == lcpp.ERR_INVALID_ARG
    assert lib.lcpp_block_table_extend(p(0), 16, table_args(lcpp), None) == lcpp.ERR_TEMP_TOO_SMALL
    assert lib.lcpp_block_table_extend(p(0), BIG, None, None) == lcpp.ERR_INVALID_ARG
    need = lcpp.DeviceBlockTable.GetTempStorageBytes(5000, 32)
    many = table_args(lcpp, num_requests=5000)
    assert lib.lcpp_block_table_extend(p(0), need - 1, many, None) == lcpp.ERR_TEMP_TOO_SMALL
    for n, tokens in (((1 << 20) + 1, 1), (1, (1 << 31) - 1)):
        with pytest.raises(lcpp.LcppError):
            lcpp.DeviceBlockTable.GetTempStorageBytes(n, tokens)


def config(lcpp, experts=16, k=4, score=0):
    return lcpp.RouterConfig(experts, k, score, 1, 1.0, 1.0)


def forward(lcpp, temp=p(0), bytes=BIG, logits=p(1), stride=16, dtype=2, bias=None, mask=None, weights=p(2),
            experts=p(3), counts=p(4), routed=p(5), loss=p(6), tokens=10, cfg=None):
    return lcpp.lib().lcpp_router_forward(temp, bytes, logits, stride, dtype, bias, mask, weights, experts, counts,
                                          routed, loss, tokens, cfg or config(lcpp), None)


def backward(lcpp, logits=p(1), stride=16, dtype=2, experts=p(2), counts=p(3), routed=p(4), gw=p(5), gl=p(6),
             out=p(7), out_stride=16, tokens=10, cfg=None):
    return lcpp.lib().lcpp_router_backward(logits, stride, dtype, experts, counts, routed, gw, gl, out, out_stride,
                                           tokens, cfg or config(lcpp), None)


def test_router_refuses(lcpp):
    bad, odd = lcpp.ERR_INVALID_ARG, ctypes.c_void_p(0x100002)
    for cfg in (config(lcpp, 0, 0), config(lcpp, 1025, 4), config(lcpp, 16, 0), config(lcpp, 16, 17),
                config(lcpp, 64, 33), config(lcpp, 16, 4, 2)):
        assert forward(lcpp, cfg=cfg, stride=2000) == bad
        assert backward(lcpp, cfg=cfg, stride=2000, out_stride=2000) == bad
    for name in ("temp", "logits", "weights", "experts", "counts", "routed", "loss"):
        assert forward(lcpp, **{name: None}) == bad
        assert forward(lcpp, **{name: odd}) == bad
    for name in ("bias", "mask"):
        assert forward(lcpp, **{name: odd}) == bad
    assert forward(lcpp, stride=15) == bad
    assert forward(lcpp, tokens=1 << 31, stride=16) == bad
    assert forward(lcpp, tokens=1 << 29) == bad  # 4 entries each: 2^31 pairs
    for dtype in (lcpp.U32, lcpp.I32, lcpp.F64, lcpp.U8, lcpp.NONE, 99):
        assert forward(lcpp, dtype=dtype) == lcpp.ERR_UNSUPPORTED_DTYPE
        assert backward(lcpp, dtype=dtype) == lcpp.ERR_UNSUPPORTED_DTYPE
    assert forward(lcpp, bytes=64) == lcpp.ERR_TEMP_TOO_SMALL
    for name in ("logits", "experts", "counts", "routed", "out"):
        assert backward(lcpp, **{name: None}) == bad
        assert backward(lcpp, **{name: odd}) == bad
    assert backward(lcpp, gw=odd) == bad and backward(lcpp, gl=odd) == bad
    assert backward(lcpp, stride=15) == bad and backward(lcpp, out_stride=15) == bad
    # partly overlapping rows, or the same rows with another stride
    assert backward(lcpp, out=ctypes.c_void_p(0x200040)) == bad
    assert backward(lcpp, out=p(1), out_stride=17) == bad
    assert backward(lcpp, tokens=0) == lcpp.OK
    for tokens, experts in ((1 << 31, 4), (10, 0), (10, 1025)):
        with pytest.raises(lcpp.LcppError):
            lcpp.DeviceRouter.GetTempStorageBytes(tokens, experts)


def test_dispatch_refuses(lcpp):
    lib, bad, odd = lcpp.lib(), lcpp.ERR_INVALID_ARG, ctypes.c_void_p(0x100002)

    def plan(temp=p(0), bytes=BIG, experts=p(1), starts=p(2), row_of=p(3), pair_of=p(4), tokens=10, k=4, e=16,
             align=8, rows=200):
        return lib.lcpp_dispatch_plan(temp, bytes, experts, starts, row_of, pair_of, tokens, k, e, align, rows, None)

    for change in ({"k": 0}, {"k": 33}, {"e": 0}, {"e": 1025}, {"align": 0}, {"rows": 1 << 31}, {"tokens": 1 << 29},
                   {"align": 1 << 30}, {"temp": None}, {"temp": ctypes.c_void_p(0x100010)}):
        assert plan(**change) == bad
    for name in ("experts", "starts", "row_of", "pair_of"):
        assert plan(**{name: None}) == bad
        assert plan(**{name: odd}) == bad
    assert plan(row_of=p(1)) == bad and plan(pair_of=ctypes.c_void_p(0x200010)) == bad and plan(starts=p(1)) == bad
    assert plan(bytes=64) == lcpp.ERR_TEMP_TOO_SMALL
    assert plan(tokens=100_000, bytes=256, starts=p(40), row_of=p(50), pair_of=p(90)) == lcpp.ERR_TEMP_TOO_SMALL

    def gather(x=p(1), xs=64, row_of=p(50), pair_of=p(51), starts=p(52), rows=p(100), rs=64, tokens=10, k=4, e=16,
               max_rows=200, h=64, dtype=lcpp.BF16):
        return lib.lcpp_dispatch_gather(x, xs, row_of, pair_of, starts, rows, rs, tokens, k, e, max_rows, h, dtype, None)

    def combine(rows=p(100), rs=64, row_of=p(50), w=p(51), out=p(200), os=64, tokens=10, k=4, max_rows=200, h=64,
                dtype=lcpp.BF16):
        return lib.lcpp_dispatch_combine(rows, rs, row_of, w, out, os, tokens, k, max_rows, h, dtype, None)

    def back(g=p(1), gs=64, rows=p(100), rs=64, row_of=p(50), pair_of=p(51), starts=p(52), w=p(53), out=p(200), os=64,
             gw=p(54), tokens=10, k=4, e=16, max_rows=200, h=64, dtype=lcpp.BF16):
        return lib.lcpp_dispatch_combine_backward(g, gs, rows, rs, row_of, pair_of, starts, w, out, os, gw, tokens, k,
                                                  e, max_rows, h, dtype, None)

    byte = ctypes.c_void_p(0x100001)
    for call, names in ((gather, ("x", "row_of", "pair_of", "starts", "rows")), (combine, ("rows", "row_of", "out")),
                        (back, ("g", "rows", "row_of", "pair_of", "starts", "w", "out", "gw"))):
        for name in names:
            assert call(**{name: None}) == bad, name
            assert call(**{name: byte}) == bad, name
        for change in ({"k": 0}, {"k": 33}, {"max_rows": 1 << 31}, {"tokens": 1 << 31}, {"h": 1 << 31}):
            assert call(**change) == bad, change
        for dtype in (lcpp.U32, lcpp.I64, lcpp.F64, lcpp.U8, lcpp.NONE, 55):
            assert call(dtype=dtype) == lcpp.ERR_UNSUPPORTED_DTYPE
    assert gather(xs=63) == bad and gather(rs=63) == bad and combine(rs=63) == bad and combine(os=63) == bad
    assert back(gs=63) == bad and back(rs=63) == bad and back(os=63) == bad
    assert combine(w=byte) == bad
    # inputs that a block may still read while another writes
    assert gather(rows=ctypes.c_void_p(0x200400)) == bad
    assert combine(out=ctypes.c_void_p(p(100).value + 128)) == bad
    assert back(out=ctypes.c_void_p(p(100).value + 128)) == bad and back(out=p(100), os=72) == bad
    assert back(out=p(1)) == bad
    with pytest.raises(lcpp.LcppError):
        lcpp.DeviceDispatch.MaxRows(10, 4, 16, 0)
    assert lcpp.DeviceDispatch.MaxRows(10, 4, 16, 8) == 40 + 16 * 7
    assert lcpp.DeviceDispatch.MaxRows(1, 4, 16, 8) == 4 + 4 * 7


def test_other_entry_points_reject_the_row_types(lcpp):
    lib = lcpp.lib()
    for dtype in (lcpp.F16, lcpp.BF16):
        assert lib.lcpp_radix_sort_keys(p(0), BIG, p(1), p(2), 10, 0, 8, 0, dtype, None) == lcpp.ERR_UNSUPPORTED_DTYPE
        assert lib.lcpp_scan_inclusive_sum(p(0), BIG, p(1), p(2), 10, dtype, None) == lcpp.ERR_UNSUPPORTED_DTYPE
        assert lib.lcpp_reduce_sum(p(0), BIG, p(1), p(2), 10, dtype, None) == lcpp.ERR_UNSUPPORTED_DTYPE
        assert lib.lcpp_select_unique(p(0), BIG, p(1), p(2), p(3), 10, dtype, None) == lcpp.ERR_UNSUPPORTED_DTYPE


def test_python_classes_refuse_tensors(lcpp):
    """Type, size and layout are looked at before the library is called (CPU tensors never get that far)."""
    i32, f32 = torch.int32, torch.float32
    t, e, k = 6, 8, 2
    logits = torch.zeros(t, e)
    good = {"w": torch.zeros(t, k), "x": torch.zeros(t, k, dtype=i32), "c": torch.zeros(e, dtype=i32),
            "n": torch.zeros(1, dtype=i32), "l": torch.zeros(1)}

    def forward(logits=logits, **changes):
        a = {**good, **changes}
        lcpp.DeviceRouter().Forward(torch.zeros(4096, dtype=torch.uint8), logits, a["w"], a["x"], a["c"], a["n"],
                                    a["l"], t, e, k)

    for change in ({"w": torch.zeros(t, k, dtype=torch.float64)}, {"x": torch.zeros(t, k, dtype=torch.int64)},
                   {"c": torch.zeros(e - 1, dtype=i32)}, {"x": torch.zeros(t, 2 * k, dtype=i32)[:, ::2]},
                   {"logits": torch.zeros(e, t).t()}, {"logits": torch.zeros(t - 1, e)}):
        with pytest.raises(lcpp.LcppError) as err:
            forward(**change)
        assert err.value.status == lcpp.ERR_INVALID_ARG
    with pytest.raises(lcpp.LcppError, match="CUDA tensor"):
        forward()
    with pytest.raises(TypeError):
        forward(logits=torch.zeros(t, e, dtype=torch.float64))
    with pytest.raises(lcpp.LcppError):
        lcpp.DeviceDispatch().Combine(torch.zeros(9, 16), torch.zeros(t, k, dtype=i32), torch.zeros(t, k),
                                      torch.zeros(t, 16, dtype=torch.bfloat16), t, k)
    with pytest.raises(lcpp.LcppError):
        lcpp.DeviceBlockTable().Extend(torch.zeros(256, dtype=torch.uint8), torch.zeros(3, dtype=i32), None,
                                       torch.zeros(2, 4, dtype=i32), torch.zeros(4, dtype=i32), None,
                                       torch.zeros(1, dtype=i32), torch.zeros(3, dtype=i32), torch.zeros(4, dtype=i32),
                                       torch.zeros(3, dtype=torch.int64), None, None, 3, 16)
