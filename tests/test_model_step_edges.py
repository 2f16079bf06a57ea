"""What the model-step operators' Python classes and entry points refuse or hand on, beyond
tests/test_model_step.py; no device needed."""
from __future__ import annotations

import pytest

torch = pytest.importorskip("torch")


class OnDevice:
    """A CPU tensor that says it is a CUDA tensor; only a stand-in for the library ever sees its address."""

    is_cuda = True

    def __init__(self, tensor):
        self.tensor = tensor

    def __getattr__(self, name):
        return getattr(self.tensor, name)


class Recorder:
    """Stands in for the library and keeps the arguments of lcpp_block_table_extend."""

    def lcpp_block_table_extend(self, temp, temp_bytes, args, stream):
        self.args = args
        return 0


def table_stride(lcpp, monkeypatch, table, n):
    recorder = Recorder()
    monkeypatch.setattr(lcpp, "lib", lambda: recorder)
    i32 = torch.int32
    stream = type("Stream", (), {"cuda_stream": 0})()
    a = [OnDevice(torch.zeros(s, dtype=i32)) for s in (n, 4, 1, n, n + 1)]
    lcpp.DeviceBlockTable().Extend(None, a[0], None, OnDevice(table), a[1], None, a[2], a[3], a[4],
                                   OnDevice(torch.zeros(n, dtype=torch.int64)), None, None, n, 16, stream)
    return recorder.args.table_stride, recorder.args.table_width


def test_table_rows_keep_their_stride(lcpp, monkeypatch):
    """Rows that share memory go to the library as they are, which refuses them (a stride below the width): taken
    for rows of their own, they would be read and written past the table's end."""
    i32 = torch.int32
    assert table_stride(lcpp, monkeypatch, torch.zeros(5, 8, dtype=i32), 5) == (8, 8)
    assert table_stride(lcpp, monkeypatch, torch.zeros(5, 8, dtype=i32)[:, :6], 5) == (8, 6)
    assert table_stride(lcpp, monkeypatch, torch.zeros(1, 8, dtype=i32).expand(5, 8), 5) == (0, 8)
    assert table_stride(lcpp, monkeypatch, torch.zeros(40, dtype=i32).as_strided((5, 8), (3, 1)), 5) == (3, 8)
    # one request takes one row, whatever follows it
    assert table_stride(lcpp, monkeypatch, torch.zeros(1, 8, dtype=i32).expand(5, 8), 1) == (8, 8)
    assert table_stride(lcpp, monkeypatch, torch.zeros(8, dtype=i32).as_strided((1, 8), (0, 1)), 1) == (8, 8)


def p(i):
    return 0x1000000 * (i + 1)  # never dereferenced


def test_block_table_refuses_every_overlap(lcpp):
    """Each output, temp storage and the table over each other and over each input, from the front and from
    behind: another block may still read what one has written."""
    n, tokens, need = 4, 32, lcpp.DeviceBlockTable.GetTempStorageBytes(4, 32)
    names = ["context_lens", "new_lens", "block_table", "free_blocks", "free_used", "free_used_out", "seq_lens_out",
             "query_starts_out", "slots_out", "positions_out", "token_request_out"]
    sizes = [n * 4, n * 4, n * 8 * 4, 40, 4, 4, n * 4, (n + 1) * 4, tokens * 8, tokens * 4, tokens * 4]

    def extend(temp=p(20), **changes):
        a = lcpp.BlockTableArgs(p(0), p(1), p(2), 8, 8, n, 16, 10, *(p(i) for i in range(3, 11)), tokens)
        for name, value in changes.items():
            setattr(a, name, value)
        return lcpp.lib().lcpp_block_table_extend(temp, need, a, None)

    place = dict(zip(names, range(11)))
    for name in ["block_table"] + names[5:]:
        for other, size in zip(names, sizes):
            if other == name:
                continue
            mine = sizes[place[name]]
            for at in (p(place[other]) + (size - 1) // 8 * 8, p(place[other]) - (mine - 1) // 8 * 8):
                assert extend(**{name: at}) == lcpp.ERR_INVALID_ARG, (name, other)
    for name, size in zip(names, sizes):
        assert extend(temp=p(place[name])) == lcpp.ERR_INVALID_ARG, name
    # wider rows: an element, and an array that starts between rows and runs into one
    for at in (p(2) + 16 * 4, p(2) + 12 * 4):
        assert extend(table_stride=16, query_starts_out=at) == lcpp.ERR_INVALID_ARG


def overlaps(names, sizes, place, written, size_of):
    """(name, address) of each written array put over the last and the first bytes of every other one."""
    for name in written:
        for other, size in zip(names, sizes):
            if other != name:
                yield name, place[other] + (size - 1) // 4 * 4
                yield name, place[other] - (size_of[name] - 1) // 4 * 4


def test_router_refuses_every_overlap(lcpp):
    t, e, k = 10, 16, 4
    cfg, lib = lcpp.RouterConfig(e, k, 0, 1, 1.0, 1.0), lcpp.lib()
    names = ["logits", "bias", "mask", "weights", "experts", "counts", "routed", "loss"]
    sizes = [t * e * 4, e * 4, t * 4, t * k * 4, t * k * 4, e * 4, 4, 4]
    place, size_of = {n: p(i) for i, n in enumerate(names)}, dict(zip(names, sizes))

    def forward(temp=p(20), stride=e, **changes):
        a = {**place, **changes}
        return lib.lcpp_router_forward(temp, 1 << 16, a["logits"], stride, 2, *(a[n] for n in names[1:]), t, cfg, None)

    for name, at in overlaps(names, sizes, place, names[3:], size_of):
        assert forward(**{name: at}) == lcpp.ERR_INVALID_ARG, name
    for name in names:
        assert forward(temp=place[name]) == lcpp.ERR_INVALID_ARG, name
    # logits in wider rows: an array that runs from the spare columns into a row
    assert forward(stride=24, experts=place["logits"] + 20 * 4) == lcpp.ERR_INVALID_ARG

    names = ["experts", "counts", "routed", "grad_weights", "grad_loss", "out"]
    sizes = [t * k * 4, e * 4, 4, t * k * 4, 4, t * e * 4]
    place, size_of = {n: p(i) for i, n in enumerate(names)}, dict(zip(names, sizes))
    for _, at in overlaps(names, sizes, place, ["out"], size_of):
        assert lib.lcpp_router_backward(p(20), e, 2, *(place[n] for n in names[:-1]), at, e, t, cfg, None) == \
            lcpp.ERR_INVALID_ARG


def test_dispatch_refuses_every_overlap(lcpp):
    t, k, e, rows, h, lib, bad = 10, 4, 16, 60, 64, lcpp.lib(), lcpp.ERR_INVALID_ARG
    sizes_of = {"experts": t * k * 4, "starts": (e + 1) * 4, "row_of": t * k * 4, "pair_of": rows * 4,
                "x": t * h * 2, "rows": rows * h * 2, "weights": t * k * 4, "out": t * h * 2, "grad_rows": rows * h * 2,
                "grad_weights": t * k * 4, "grad_out": t * h * 2}
    place = {n: p(i) for i, n in enumerate(sizes_of)}

    def check(call, names, written):
        for name, at in overlaps(names, [sizes_of[n] for n in names], place, written, sizes_of):
            assert call(**{**place, name: at}) == bad, (name, hex(at))

    def plan(experts, starts, row_of, pair_of, temp=p(20), **_):
        return lib.lcpp_dispatch_plan(temp, 1 << 16, experts, starts, row_of, pair_of, t, k, e, 1, rows, None)

    names = ["experts", "starts", "row_of", "pair_of"]
    check(plan, names, names[1:])
    for name in names:
        assert plan(**place, temp=place[name]) == bad

    def gather(x, row_of, pair_of, starts, rows, **_):
        return lib.lcpp_dispatch_gather(x, h, row_of, pair_of, starts, rows, h, t, k, e, 60, h, lcpp.BF16, None)

    check(gather, ["x", "row_of", "pair_of", "starts", "rows"], ["rows"])

    def combine(rows, row_of, weights, out, **_):
        return lib.lcpp_dispatch_combine(rows, h, row_of, weights, out, h, t, k, 60, h, lcpp.BF16, None)

    check(combine, ["rows", "row_of", "weights", "out"], ["out"])

    def back(grad_out, rows, row_of, pair_of, starts, weights, grad_rows, grad_weights, **_):
        return lib.lcpp_dispatch_combine_backward(grad_out, h, rows, h, row_of, pair_of, starts, weights, grad_rows, h,
                                                  grad_weights, t, k, e, 60, h, lcpp.BF16, None)

    check(back, ["grad_out", "rows", "row_of", "pair_of", "starts", "weights", "grad_rows", "grad_weights"],
          ["grad_rows", "grad_weights"])


def test_router_bias_on_scores_is_a_flag(lcpp):
    """The flag goes with either score, in the gradient's configuration too, and makes no other value valid."""
    lib = lcpp.lib()
    for score, status in ((lcpp.BIAS_ON_SCORE, lcpp.OK), (lcpp.BIAS_ON_SCORE + lcpp.SCORE_SIGMOID, lcpp.OK),
                          (lcpp.BIAS_ON_SCORE + 2, lcpp.ERR_INVALID_ARG), (0x20, lcpp.ERR_INVALID_ARG)):
        cfg = lcpp.RouterConfig(16, 4, score, 1, 1.0, 1.0)
        assert lib.lcpp_router_backward(None, 16, 2, None, None, None, None, None, None, 16, 0, cfg, None) == status
