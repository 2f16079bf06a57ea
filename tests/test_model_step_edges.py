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
