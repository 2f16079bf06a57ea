"""What the paged cache's Python classes and entry points refuse or hand on, beyond tests/test_cache_ops.py; no device
needed: a stand-in takes the library's calls."""
from __future__ import annotations

import pytest

torch = pytest.importorskip("torch")


class Recorder:
    """Stands in for the library and keeps its calls."""

    def __init__(self):
        self.calls = []

    def lcpp_status_string(self, status):
        return b""

    def __getattr__(self, name):
        def call(*args):
            self.calls.append((name, args))
            return 0
        return call


class Elsewhere:
    """A tensor that says it lies on another device."""

    def __init__(self, tensor):
        self.tensor = tensor

    def get_device(self):
        return 3

    def __getattr__(self, name):
        return getattr(self.tensor, name)


@pytest.fixture
def recorder(lcpp, monkeypatch):
    """CPU tensors pass as the current device's, whose number is theirs."""
    lib = Recorder()
    monkeypatch.setattr(lcpp, "lib", lambda: lib)
    monkeypatch.setattr(lcpp, "_device", lambda: -1)
    monkeypatch.setattr(lcpp, "_queue", lambda stream, device=None: 0)
    return lib


def decode_args():
    i32 = torch.int32
    q = torch.zeros(4, 4, 64)
    return [q, torch.zeros(10, 16, 2, 64), torch.zeros(10, 16, 2, 64), torch.zeros(4, 8, dtype=i32),
            torch.zeros(4, dtype=i32), torch.zeros_like(q), 4]


def test_decode_takes_temp_of_its_device(lcpp, recorder):
    """Temp storage of the host or of another device would be written by the kernels all the same."""
    temp, call = torch.zeros(1024, dtype=torch.uint8), lcpp.DevicePagedAttention().Decode
    call(temp, *decode_args())
    assert [name for name, _ in recorder.calls] == ["lcpp_paged_attention_decode"]
    assert recorder.calls[0][1][:2] == (temp.data_ptr(), 1024)
    for bad in (Elsewhere(temp), torch.zeros(1, dtype=torch.uint8).expand(1 << 30)):
        with pytest.raises(lcpp.LcppError):
            call(bad, *decode_args())
    assert len(recorder.calls) == 1


@pytest.mark.parametrize("k,v", [
    # one kv head: heads first in the page, and tokens first
    (torch.zeros(10, 1, 16, 64).transpose(1, 2), torch.zeros(10, 16, 1, 64)),
    # one page, and the first of several that lie further apart
    (torch.zeros(1, 16, 2, 64), torch.zeros(3, 20, 2, 64)[:1, :16]),
    # pages of one token
    (torch.zeros(10, 2, 64)[:, None], torch.zeros(10, 1, 2, 64)),
    (torch.zeros(10, 16, 2, 1), torch.zeros(10, 16, 2, 3)[..., :1].contiguous()),
])
def test_strides_of_single_entries_do_not_matter(lcpp, k, v):
    """Keys and values need equal strides where there is a second entry to step to."""
    fields = lcpp._kv_cache(k, v, -1)
    assert fields[:2] == (k.data_ptr(), v.data_ptr()) and fields[5:9] == tuple(k.shape)
    for i in range(3):
        assert k.shape[i] == 1 or fields[2 + i] == k.stride(i) == v.stride(i)


def test_strides_of_keys_and_values_agree(lcpp):
    k = torch.zeros(10, 16, 2, 64)
    for v in (torch.zeros(10, 2, 16, 64).transpose(1, 2), torch.zeros(10, 17, 2, 64)[:, :16], torch.zeros(10, 16, 2, 65)[..., :64],
              torch.zeros(10, 16, 2, 64, dtype=torch.float16), torch.zeros(9, 16, 2, 64)):
        with pytest.raises(lcpp.LcppError):
            lcpp._kv_cache(k, v, -1)


def test_append_of_one_tensor_as_queries_and_keys(lcpp, recorder):
    """Queries that are the keys' own tensor are turned into their output, as those of an equal tensor are."""
    x, out, cache = torch.zeros(8, 2, 64), torch.zeros(8, 2, 64), torch.zeros(2, 10, 16, 2, 64)
    slots, positions, f = torch.zeros(8, dtype=torch.int64), torch.zeros(8, dtype=torch.int32), torch.zeros(32, dtype=torch.float64)
    for keys in (x, x[:]):
        lcpp.DeviceRotary().Append(x, keys, x, out, cache[0], cache[1], slots, positions, f, 8)
    (_, (one, *_)), (_, (two, *_)) = recorder.calls
    assert lcpp.RotaryArgs.from_buffer_copy(two).q.out == out.data_ptr() and one == two


@pytest.mark.parametrize("shift", [64 - 32, 128 + 32, 192 - 2, 192 * 3, 768 - 32, 192 + 32])
def test_rows_inside_each_head_that_overlap_are_refused(lcpp, shift):
    """Heads of [tokens, 4, 3, 64]: an output that is not one of the three in every head shares memory with the queries
    (or, behind the third, with those of the next head or token)."""
    at = 0x10000000
    q = lcpp.HeadRows(at, at, 768, 192, 768, 192, 4)
    k = lcpp.HeadRows(0x50000000, at + 2 * shift, 128, 64, 768, 192, 2)
    args = lcpp.RotaryArgs(q, k, 0x60000000, None, None, 0x70000000, 8, 0, 64, 64, 0, 1.0, lcpp.BF16)
    assert lcpp.lib().lcpp_rotary_forward(bytes(args), None) == lcpp.ERR_INVALID_ARG


@pytest.mark.parametrize("scale,softcap", [(1.0, 1e-40), (3e38, 0.0), (-3e38, 0.0), (1.0, 3e38), (1e30, 1e-10)])
def test_decode_refuses_factors_beyond_32_bits(lcpp, scale, softcap):
    """Factors that are no numbers where the kernel multiplies by them."""
    cache = lcpp.KVCache(0xA0000000, 0xB0000000, 2048, 128, 64, 10, 16, 2, 64, lcpp.BF16)
    args = lcpp.PagedAttentionArgs(cache, 0x10000000, 256, 64, 0x20000000, 256, 64, 0x30000000, 8, 8, 4, 0x40000000, 4, 0,
                                   scale, softcap, 0x50000000, 0x60000000, 0x70000000, 1.0)
    assert lcpp.lib().lcpp_paged_attention_decode(0x100000000, 1 << 30, bytes(args), None) == lcpp.ERR_INVALID_ARG
