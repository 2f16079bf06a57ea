"""Python front end of liblcpp_b200 (sm_100a sort / scan / reduce).

A thin ctypes layer over the C ABI in ``include/lcpp_b200.h`` plus class
wrappers that mirror the reference's Device-level modules
(``DeviceRadixSort``, ``DeviceScan``, ``DeviceReduce`` in
``src/lcpp/device/``): same method names, same argument order, CUB-style
temp-storage queries.  Device buffers are torch CUDA tensors (torch is only
the allocator and stream provider here); every call enqueues on the current
torch CUDA stream unless a stream is given.

There is no CPU fallback: if ``liblcpp_b200.so`` has not been built, importing
the library raises.
"""
from __future__ import annotations

import ctypes
from pathlib import Path

_HERE = Path(__file__).resolve().parent
LIB_PATH = _HERE / "liblcpp_b200.so"

# lcpp_status
OK, ERR_INVALID_ARG, ERR_TEMP_TOO_SMALL, ERR_UNSUPPORTED_DTYPE = 0, 1, 2, 3
ERR_CUDA, ERR_LOOKBACK_TIMEOUT, ERR_COMM, ERR_INTERNAL = 4, 5, 6, 7
# lcpp_dtype
U32, I32, F32, U64, I64, F64, NONE = 0, 1, 2, 3, 4, 5, 255
U8 = 6  # 1-byte (bool) selection flags only
F16, BF16 = 7, 8  # logits and token rows of the model-step operators only
# lcpp_router_score
SCORE_SOFTMAX, SCORE_SIGMOID = 0, 1
BIAS_ON_SCORE = 0x10  # added to either: a bias joins the score instead of the logit
# lcpp_rotary_layout, lcpp_rotary_scaling
ROTARY_HALF, ROTARY_INTERLEAVED = 0, 1
ROTARY_PLAIN, ROTARY_LINEAR, ROTARY_BASE, ROTARY_BY_ROTATIONS = 0, 1, 2, 3
# lcpp_op
OP_SUM, OP_MIN, OP_MAX = 0, 1, 2
# lcpp_testgen_dist
GEN_U32_UNIFORM, GEN_U32_AND3, GEN_U32_CONST, GEN_U64_UNIFORM = 0, 1, 2, 3
GEN_I32_SCAN, GEN_F32_UNIT, GEN_I64_UNIFORM, GEN_U32_INDEX = 4, 5, 6, 7
GEN_F32_NORMAL, GEN_U32_ZIPF = 8, 9

# lcpp_kernel_kind
KERNEL_SORT_HISTOGRAM, KERNEL_SORT_ONESWEEP, KERNEL_SCAN, KERNEL_REDUCE, KERNEL_SEGMENT_BLOCK = 0, 1, 2, 3, 4
KERNEL_MERGE = 5
KERNEL_ARG_REDUCE = 6
KERNEL_BY_KEY = 7
KERNEL_SELECT = 8
KERNEL_BLOCK_TABLE, KERNEL_ROUTER, KERNEL_DISPATCH = 9, 10, 11
KERNEL_ROTARY, KERNEL_PAGED_ATTENTION, KERNEL_CACHE_EVICTION = 12, 13, 14

_lib = None


class KernelTime(ctypes.Structure):
    _fields_ = [("kind", ctypes.c_int), ("ms", ctypes.c_float), ("items", ctypes.c_uint64)]


class DistSortTimes(ctypes.Structure):
    """lcpp_dist_sort_times (include/lcpp_b200_dist.h)."""
    _fields_ = [("local_sort_ms", ctypes.c_float), ("splitters_ms", ctypes.c_float),
                ("host_wait_ms", ctypes.c_float), ("exchange_merge_ms", ctypes.c_float),
                ("local_merge_ms", ctypes.c_float), ("total_ms", ctypes.c_float), ("host_ms", ctypes.c_float),
                ("peer_exchange", ctypes.c_int)]


class BlockTableArgs(ctypes.Structure):
    """lcpp_block_table_args (include/lcpp_b200_model.h)."""
    _fields_ = [("context_lens", ctypes.c_void_p), ("new_lens", ctypes.c_void_p), ("block_table", ctypes.c_void_p),
                ("table_stride", ctypes.c_uint64), ("table_width", ctypes.c_uint32),
                ("num_requests", ctypes.c_uint32), ("block_size", ctypes.c_uint32), ("num_free", ctypes.c_uint32),
                ("free_blocks", ctypes.c_void_p), ("free_used", ctypes.c_void_p), ("free_used_out", ctypes.c_void_p),
                ("seq_lens_out", ctypes.c_void_p), ("query_starts_out", ctypes.c_void_p),
                ("slots_out", ctypes.c_void_p), ("positions_out", ctypes.c_void_p),
                ("token_request_out", ctypes.c_void_p), ("max_tokens", ctypes.c_uint64)]


class RouterConfig(ctypes.Structure):
    """lcpp_router_config (include/lcpp_b200_model.h)."""
    _fields_ = [("num_experts", ctypes.c_uint32), ("top_k", ctypes.c_uint32), ("score", ctypes.c_int32),
                ("renormalize", ctypes.c_int32), ("weight_scale", ctypes.c_float), ("loss_coef", ctypes.c_float)]


class HeadRows(ctypes.Structure):
    """lcpp_head_rows (include/lcpp_b200_model.h)."""
    _fields_ = [("in_", ctypes.c_void_p), ("out", ctypes.c_void_p), ("in_token_stride", ctypes.c_uint64),
                ("in_head_stride", ctypes.c_uint64), ("out_token_stride", ctypes.c_uint64),
                ("out_head_stride", ctypes.c_uint64), ("num_heads", ctypes.c_uint32)]


class KVCache(ctypes.Structure):
    """lcpp_kv_cache (include/lcpp_b200_model.h)."""
    _fields_ = [("k", ctypes.c_void_p), ("v", ctypes.c_void_p), ("page_stride", ctypes.c_uint64),
                ("token_stride", ctypes.c_uint64), ("head_stride", ctypes.c_uint64), ("num_pages", ctypes.c_uint32),
                ("block_size", ctypes.c_uint32), ("num_kv_heads", ctypes.c_uint32), ("head_dim", ctypes.c_uint32),
                ("dtype", ctypes.c_int)]


class RotaryArgs(ctypes.Structure):
    """lcpp_rotary_args (include/lcpp_b200_model.h)."""
    _fields_ = [("q", HeadRows), ("k", HeadRows), ("positions", ctypes.c_void_p), ("token_request", ctypes.c_void_p),
                ("position_offset", ctypes.c_void_p), ("frequencies", ctypes.c_void_p),
                ("num_tokens", ctypes.c_uint64), ("num_requests", ctypes.c_uint32), ("head_dim", ctypes.c_uint32),
                ("rotary_dim", ctypes.c_uint32), ("layout", ctypes.c_int32), ("scale", ctypes.c_float),
                ("dtype", ctypes.c_int)]


class CacheAppendArgs(ctypes.Structure):
    """lcpp_cache_append_args (include/lcpp_b200_model.h)."""
    _fields_ = [("cache", KVCache), ("v", ctypes.c_void_p), ("v_token_stride", ctypes.c_uint64),
                ("v_head_stride", ctypes.c_uint64), ("slots", ctypes.c_void_p), ("slot_positions", ctypes.c_void_p),
                ("slot_scores", ctypes.c_void_p)]


class PagedAttentionArgs(ctypes.Structure):
    """lcpp_paged_attention_args (include/lcpp_b200_model.h)."""
    _fields_ = [("cache", KVCache), ("q", ctypes.c_void_p), ("q_request_stride", ctypes.c_uint64),
                ("q_head_stride", ctypes.c_uint64), ("out", ctypes.c_void_p), ("out_request_stride", ctypes.c_uint64),
                ("out_head_stride", ctypes.c_uint64), ("block_table", ctypes.c_void_p),
                ("table_stride", ctypes.c_uint64), ("table_width", ctypes.c_uint32),
                ("num_requests", ctypes.c_uint32), ("seq_lens", ctypes.c_void_p), ("num_heads", ctypes.c_uint32),
                ("window", ctypes.c_uint32), ("scale", ctypes.c_float), ("softcap", ctypes.c_float),
                ("lse_out", ctypes.c_void_p), ("slot_scores", ctypes.c_void_p), ("slot_scores_out", ctypes.c_void_p),
                ("score_decay", ctypes.c_float)]


class CacheEvictArgs(ctypes.Structure):
    """lcpp_cache_evict_args (include/lcpp_b200_model.h)."""
    _fields_ = [("seq_lens", ctypes.c_void_p), ("block_table", ctypes.c_void_p), ("table_stride", ctypes.c_uint64),
                ("table_width", ctypes.c_uint32), ("num_requests", ctypes.c_uint32), ("num_pages", ctypes.c_uint32),
                ("block_size", ctypes.c_uint32), ("slot_scores", ctypes.c_void_p),
                ("slot_positions", ctypes.c_void_p), ("evicted", ctypes.c_void_p), ("budget", ctypes.c_uint32),
                ("trigger", ctypes.c_uint32), ("keep_first", ctypes.c_uint32), ("keep_recent", ctypes.c_uint32),
                ("max_moves", ctypes.c_uint32), ("seq_lens_out", ctypes.c_void_p), ("evicted_out", ctypes.c_void_p),
                ("move_counts_out", ctypes.c_void_p), ("moves_out", ctypes.c_void_p), ("moves_stride", ctypes.c_uint64),
                ("free_blocks", ctypes.c_void_p), ("free_used", ctypes.c_void_p), ("free_used_out", ctypes.c_void_p), ("num_free", ctypes.c_uint32)]


class LcppError(RuntimeError):
    def __init__(self, status: int, what: str):
        self.status = status
        name = lib().lcpp_status_string(status).decode() if _lib is not None else str(status)
        super().__init__(f"{what}: {name}")


def lib() -> ctypes.CDLL:
    """Load liblcpp_b200.so (raises when it has not been built)."""
    global _lib
    if _lib is not None:
        return _lib
    if not LIB_PATH.exists():
        raise ImportError(
            f"{LIB_PATH} is missing: build it with "
            "`python luisacompute-parallelprimitive_b200/build.py` (no CPU fallback exists)")
    l = ctypes.CDLL(str(LIB_PATH))
    vp, sz, u64, i = ctypes.c_void_p, ctypes.c_size_t, ctypes.c_uint64, ctypes.c_int
    szp = ctypes.POINTER(ctypes.c_size_t)
    ip = ctypes.POINTER(ctypes.c_int)
    vpa = ctypes.c_void_p * 2
    u32, cfg, f64 = ctypes.c_uint32, ctypes.POINTER(RouterConfig), ctypes.c_double
    sigs = {
        "lcpp_status_string": ([i], ctypes.c_char_p),
        "lcpp_version": ([], i),
        "lcpp_radix_sort_keys_temp_bytes": ([i, u64, szp], i),
        "lcpp_radix_sort_pairs_temp_bytes": ([i, i, u64, szp], i),
        "lcpp_radix_sort_keys": ([vp, sz, vp, vp, u64, i, i, i, i, vp], i),
        "lcpp_radix_sort_pairs": ([vp, sz, vp, vp, vp, vp, u64, i, i, i, i, i, vp], i),
        "lcpp_radix_sort_keys_double_buffer": ([vp, sz, vpa, ip, u64, i, i, i, i, vp], i),
        "lcpp_radix_sort_pairs_double_buffer": ([vp, sz, vpa, vpa, ip, u64, i, i, i, i, i, vp], i),
        "lcpp_radix_sort_decomposed_temp_bytes": ([u64, szp], i),
        "lcpp_radix_sort_decomposed_keys": ([vp, sz, vp, vp, u64, ctypes.c_uint32, vp, i, i, i, i, vp], i),
        "lcpp_radix_sort_decomposed_pairs": ([vp, sz, vp, vp, vp, vp, u64, ctypes.c_uint32, vp, i, i, i, i, i, vp],
                                             i),
        "lcpp_radix_sort_decomposed_keys_double_buffer": ([vp, sz, vpa, ip, u64, ctypes.c_uint32, vp, i, i, i, i, vp],
                                                          i),
        "lcpp_radix_sort_decomposed_pairs_double_buffer": ([vp, sz, vpa, vpa, ip, u64, ctypes.c_uint32, vp, i, i, i,
                                                            i, i, vp], i),
        "lcpp_segmented_radix_sort_keys_temp_bytes": ([i, u64, szp], i),
        "lcpp_segmented_radix_sort_pairs_temp_bytes": ([i, i, u64, szp], i),
        "lcpp_segmented_radix_sort_keys": ([vp, sz, vp, vp, u64, u64, vp, vp, i, i, i, i, vp], i),
        "lcpp_segmented_radix_sort_pairs": ([vp, sz, vp, vp, vp, vp, u64, u64, vp, vp, i, i, i, i, i, vp], i),
        "lcpp_segmented_radix_sort_keys_double_buffer": ([vp, sz, vpa, ip, u64, u64, vp, vp, i, i, i, i, vp], i),
        "lcpp_segmented_radix_sort_pairs_double_buffer": ([vp, sz, vpa, vpa, ip, u64, u64, vp, vp, i, i, i, i, i,
                                                           vp], i),
        "lcpp_scan_temp_bytes": ([i, u64, szp], i),
        "lcpp_scan_exclusive": ([vp, sz, vp, vp, u64, i, vp, i, vp], i),
        "lcpp_scan_inclusive": ([vp, sz, vp, vp, u64, i, i, vp], i),
        "lcpp_scan_inclusive_init": ([vp, sz, vp, vp, u64, i, vp, i, vp], i),
        "lcpp_scan_exclusive_sum": ([vp, sz, vp, vp, u64, i, vp], i),
        "lcpp_scan_inclusive_sum": ([vp, sz, vp, vp, u64, i, vp], i),
        "lcpp_scan_inclusive_sum_noalloc": ([vp, vp, u64, i, vp], i),
        "lcpp_reduce_temp_bytes": ([i, u64, szp], i),
        "lcpp_reduce_arg_temp_bytes": ([i, u64, szp], i),
        "lcpp_scan_by_key_temp_bytes": ([i, i, u64, szp], i),
        "lcpp_scan_exclusive_by_key": ([vp, sz, vp, vp, vp, u64, i, vp, i, i, vp], i),
        "lcpp_scan_inclusive_by_key": ([vp, sz, vp, vp, vp, u64, i, i, i, vp], i),
        "lcpp_scan_inclusive_by_key_init": ([vp, sz, vp, vp, vp, u64, i, vp, i, i, vp], i),
        "lcpp_scan_exclusive_sum_by_key": ([vp, sz, vp, vp, vp, u64, i, i, vp], i),
        "lcpp_scan_inclusive_sum_by_key": ([vp, sz, vp, vp, vp, u64, i, i, vp], i),
        "lcpp_reduce_by_key_temp_bytes": ([i, i, u64, szp], i),
        "lcpp_reduce_by_key": ([vp, sz, vp, vp, vp, vp, vp, u64, i, i, i, vp], i),
        "lcpp_scan_transform_temp_bytes": ([u64, szp], i),
        "lcpp_scan_exclusive_sum_transform": ([vp, sz, vp, vp, u64, i, vp, i, vp], i),
        "lcpp_scan_exclusive_sum_adjacent": ([vp, sz, vp, vp, u64, i, vp], i),
        "lcpp_select_temp_bytes": ([u64, szp], i),
        "lcpp_partition_temp_bytes": ([u64, szp], i),
        "lcpp_partition_three_way_temp_bytes": ([u64, szp], i),
        "lcpp_select_flagged": ([vp, sz, vp, vp, vp, vp, u64, i, i, vp], i),
        "lcpp_select_flagged_if": ([vp, sz, vp, vp, vp, vp, u64, i, i, vp, i, vp], i),
        "lcpp_select_if": ([vp, sz, vp, vp, vp, u64, i, vp, i, vp], i),
        "lcpp_select_unique": ([vp, sz, vp, vp, vp, u64, i, vp], i),
        "lcpp_select_unique_by_key": ([vp, sz, vp, vp, vp, vp, vp, u64, i, i, vp], i),
        "lcpp_partition_flagged": ([vp, sz, vp, vp, vp, vp, u64, i, i, vp], i),
        "lcpp_partition_if": ([vp, sz, vp, vp, vp, u64, i, vp, i, vp], i),
        "lcpp_partition_if_three_way": ([vp, sz, vp, vp, vp, vp, vp, u64, i, vp, i, vp, i, vp], i),
        "lcpp_reduce_argmin": ([vp, sz, vp, vp, vp, u64, i, vp], i),
        "lcpp_reduce_argmax": ([vp, sz, vp, vp, vp, u64, i, vp], i),
        "lcpp_reduce": ([vp, sz, vp, vp, u64, i, vp, i, vp], i),
        "lcpp_reduce_sum": ([vp, sz, vp, vp, u64, i, vp], i),
        "lcpp_reduce_min": ([vp, sz, vp, vp, u64, i, vp], i),
        "lcpp_reduce_max": ([vp, sz, vp, vp, u64, i, vp], i),
        "lcpp_device_status": ([vp, vp], i),
        "lcpp_testgen_fill": ([vp, u64, u64, u64, i, vp], i),
        "lcpp_dist_search_sorted": ([vp, u64, vp, u64, i, vp, i, vp], i),
        "lcpp_dist_merge_temp_bytes": ([u64, szp], i),
        "lcpp_dist_merge_sorted": ([vp, sz, vp, u64, vp, u64, vp, i, vp], i),
        "lcpp_dist_merge_batch_temp_bytes": ([i, ctypes.POINTER(u64), ctypes.POINTER(u64), szp], i),
        "lcpp_dist_merge_sorted_batch": ([vp, sz, i, ctypes.POINTER(vp), ctypes.POINTER(u64), ctypes.POINTER(vp),
                                          ctypes.POINTER(u64), ctypes.POINTER(vp), i, vp], i),
        "lcpp_dist_ipc_alloc": ([sz, ctypes.POINTER(ctypes.c_void_p), vp], i),
        "lcpp_dist_ipc_open": ([vp, ctypes.POINTER(ctypes.c_void_p)], i),
        "lcpp_dist_ipc_close": ([vp], i),
        "lcpp_dist_ipc_free": ([vp], i),
        "lcpp_comm_unique_id": ([vp], i),
        "lcpp_comm_init": ([vp, i, i, ctypes.POINTER(ctypes.c_void_p)], i),
        "lcpp_comm_from_nccl": ([vp, ctypes.POINTER(ctypes.c_void_p)], i),
        "lcpp_comm_destroy": ([vp], i),
        "lcpp_comm_rank": ([vp, ip, ip], i),
        "lcpp_dist_sort_keys_temp_bytes": ([vp, i, u64, szp], i),
        "lcpp_dist_sort_keys": ([vp, vp, sz, vp, vp, u64, i, i, ctypes.POINTER(DistSortTimes), vp], i),
        "lcpp_dist_scan_temp_bytes": ([vp, i, u64, szp], i),
        "lcpp_dist_inclusive_sum": ([vp, vp, sz, vp, vp, u64, i, vp], i),
        "lcpp_dist_exclusive_sum": ([vp, vp, sz, vp, vp, u64, i, vp], i),
        "lcpp_dist_reduce_temp_bytes": ([vp, i, u64, szp], i),
        "lcpp_dist_reduce": ([vp, vp, sz, vp, vp, u64, i, vp, i, vp], i),
        "lcpp_block_table_temp_bytes": ([u64, u64, szp], i),
        "lcpp_block_table_extend": ([vp, sz, ctypes.POINTER(BlockTableArgs), vp], i),
        "lcpp_router_temp_bytes": ([u64, u32, szp], i),
        "lcpp_router_forward": ([vp, sz, vp, u64, i, vp, vp, vp, vp, vp, vp, vp, u64, cfg, vp], i),
        "lcpp_router_backward": ([vp, u64, i, vp, vp, vp, vp, vp, vp, u64, u64, cfg, vp], i),
        "lcpp_dispatch_temp_bytes": ([u64, u32, u32, szp], i),
        "lcpp_dispatch_max_rows": ([u64, u32, u32, u32, ctypes.POINTER(u64)], i),
        "lcpp_dispatch_plan": ([vp, sz, vp, vp, vp, vp, u64, u32, u32, u32, u64, vp], i),
        "lcpp_dispatch_gather": ([vp, u64, vp, vp, vp, vp, u64, u64, u32, u32, u64, u64, i, vp], i),
        "lcpp_dispatch_combine": ([vp, u64, vp, vp, vp, u64, u64, u32, u64, u64, i, vp], i),
        "lcpp_dispatch_combine_backward": ([vp, u64, vp, u64, vp, vp, vp, vp, vp, u64, vp, u64, u32, u32, u64, u64,
                                            i, vp], i),
        "lcpp_rotary_frequencies": ([vp, u32, f64, i, f64, f64, f64, f64], i),
        "lcpp_rotary_forward": ([vp, vp], i),
        "lcpp_rotary_backward": ([vp, vp], i),
        "lcpp_rotary_append": ([vp, vp, vp], i),
        "lcpp_paged_attention_temp_bytes": ([u32, u32, u32, u32, u64, szp], i),
        "lcpp_paged_attention_decode": ([vp, sz, vp, vp], i),
        "lcpp_cache_evict_plan": ([vp, vp], i),
        "lcpp_cache_evict_move": ([vp, vp, u64, u32, vp, u32, vp, vp, vp], i),
        "lcpp_diag_timing_enable": ([i], i),
        "lcpp_diag_launch_shapes": ([ctypes.POINTER(u64)], i),
        "lcpp_diag_wait_timeout_probe": ([vp, sz, u64, vp], i),
        "lcpp_diag_timing_read": ([ctypes.POINTER(KernelTime), i, ip], i),
    }
    for name, (args, res) in sigs.items():
        f = getattr(l, name)
        f.argtypes = args
        f.restype = res
    _lib = l
    return l


def check(status: int, what: str) -> None:
    if status != OK:
        raise LcppError(status, what)


# ---------------------------------------------------------------------------
# torch helpers (plumbing only)
# ---------------------------------------------------------------------------
_torch_module = None


def _torch():
    global _torch_module
    if _torch_module is None:
        import torch
        _torch_module = torch
    return _torch_module


def dtype_code(t) -> int:
    torch = _torch()
    m = {torch.uint32: U32, torch.int32: I32, torch.float32: F32, torch.uint64: U64,
         torch.int64: I64, torch.float64: F64}
    if t.dtype not in m:
        raise TypeError(f"unsupported dtype {t.dtype}")
    return m[t.dtype]


def _ptr(t):
    return None if t is None else ctypes.c_void_p(t.data_ptr())


def _stream(stream):
    torch = _torch()
    if stream is None:
        stream = torch.cuda.current_stream()
    return ctypes.c_void_p(stream.cuda_stream)


def _host_scalar(value, code):
    import numpy as np
    np_t = {U32: np.uint32, I32: np.int32, F32: np.float32, U64: np.uint64, I64: np.int64,
            F64: np.float64}[code]
    arr = np.array([value], dtype=np_t)
    return arr, ctypes.c_void_p(arr.ctypes.data)


def alloc_temp(nbytes: int, device=None):
    """A 256-byte aligned uint8 CUDA tensor of at least nbytes (>= 1)."""
    torch = _torch()
    return torch.empty(max(int(nbytes), 1), dtype=torch.uint8, device=device or "cuda")


# ---------------------------------------------------------------------------
# Reference-shaped module wrappers
# ---------------------------------------------------------------------------
class DoubleBuffer:
    """Mirror of the reference's DoubleBuffer<T> (src/lcpp/common/util_type.h:57-74)."""

    def __init__(self, current, alternate, selector: int = 0):
        self.d_buffers = [current, alternate]
        self.selector = selector

    def current(self):
        return self.d_buffers[self.selector]

    def alternate(self):
        return self.d_buffers[self.selector ^ 1]


def _bit_range(rest):
    """(begin_bit, end_bit) from trailing positional arguments; end None = key width."""
    if len(rest) > 2:
        raise TypeError("too many arguments")
    begin = rest[0] if len(rest) >= 1 else 0
    end = rest[1] if len(rest) == 2 else None
    return begin, end


class Clause(ctypes.Structure):
    """One clause of a C-ABI predicate (lcpp_clause in include/lcpp_b200.h)."""
    _fields_ = [("kind", ctypes.c_int32), ("negate", ctypes.c_int32), ("a", ctypes.c_uint64),
                ("b", ctypes.c_uint64)]


CLAUSE_LT, CLAUSE_LE, CLAUSE_GT, CLAUSE_GE, CLAUSE_EQ, CLAUSE_NE, CLAUSE_MOD_EQ, CLAUSE_BITS_ANY = range(8)


def _bits(value, code: int) -> int:
    import struct
    if code == F32:
        return struct.unpack("<I", struct.pack("<f", float(value)))[0]
    if code == F64:
        return struct.unpack("<Q", struct.pack("<d", float(value)))[0]
    width = {U8: 8, U32: 32, I32: 32, U64: 64, I64: 64}[code]
    return int(value) & ((1 << width) - 1)


class Pred:
    """A predicate for DeviceSelect / DevicePartition through the C ABI: the
    AND (`&`) of up to 4 clauses, each negatable (`~`).  Examples: the
    reference tests' `value % 2 == 0` is Pred.mod_eq(2, 0), `value < 7` is
    Pred.lt(7), `flag > 0 & flag % 2 != 0` is Pred.gt(0) & ~Pred.mod_eq(2, 0)."""

    def __init__(self, clauses=()):
        self.clauses = list(clauses)  # (kind, negate, a, b)

    def __and__(self, other: "Pred") -> "Pred":
        return Pred(self.clauses + other.clauses)

    def __invert__(self) -> "Pred":
        if len(self.clauses) != 1:
            raise ValueError("~ applies to a single clause")
        k, n, a, b = self.clauses[0]
        return Pred([(k, 1 - n, a, b)])

    @staticmethod
    def lt(a): return Pred([(CLAUSE_LT, 0, a, 0)])
    @staticmethod
    def le(a): return Pred([(CLAUSE_LE, 0, a, 0)])
    @staticmethod
    def gt(a): return Pred([(CLAUSE_GT, 0, a, 0)])
    @staticmethod
    def ge(a): return Pred([(CLAUSE_GE, 0, a, 0)])
    @staticmethod
    def eq(a): return Pred([(CLAUSE_EQ, 0, a, 0)])
    @staticmethod
    def ne(a): return Pred([(CLAUSE_NE, 0, a, 0)])
    @staticmethod
    def mod_eq(m, r): return Pred([(CLAUSE_MOD_EQ, 0, m, r)])
    @staticmethod
    def bits_any(mask): return Pred([(CLAUSE_BITS_ANY, 0, mask, 0)])

    def encode(self, code: int):
        """(ctypes array, count) for values of dtype `code`."""
        arr = (Clause * max(1, len(self.clauses)))()
        for j, (k, n, a, b) in enumerate(self.clauses):
            arr[j] = Clause(k, n, _bits(a, code), _bits(b, code))
        return arr, len(self.clauses)


def flag_code(t) -> int:
    """dtype code of a selection-flag tensor (bool and uint8 are LCPP_U8)."""
    torch = _torch()
    if t.dtype in (torch.bool, torch.uint8):
        return U8
    return dtype_code(t)


class KeyMember(ctypes.Structure):
    _fields_ = [("offset", ctypes.c_uint32), ("dtype", ctypes.c_int)]


class Decomposer:
    """The reference's decomposer for struct keys (device_radix_sort.h:556-940):
    the key struct's size in bytes and its members, most significant first, as
    (byte offset, dtype code) pairs."""

    def __init__(self, key_bytes: int, members):
        self.key_bytes = int(key_bytes)
        self.members = [(int(o), int(d)) for o, d in members]
        self.bits = sum(8 * (4 if d in (U32, I32, F32) else 8) for _, d in self.members)
        arr = (KeyMember * len(self.members))(*[KeyMember(o, d) for o, d in self.members])
        self._arr = arr


class DeviceRadixSort:
    """Mirror of lcpp::DeviceRadixSort (src/lcpp/device/device_radix_sort.h:50-1489)."""

    @staticmethod
    def GetDecomposedTempStorageBytes(num_items: int) -> int:
        out = ctypes.c_size_t()
        check(lib().lcpp_radix_sort_decomposed_temp_bytes(num_items, ctypes.byref(out)),
              "GetDecomposedTempStorageBytes")
        return out.value

    @staticmethod
    def GetSortKeysTempStorageBytes(key_dtype: int, num_items: int) -> int:
        out = ctypes.c_size_t()
        check(lib().lcpp_radix_sort_keys_temp_bytes(key_dtype, num_items, ctypes.byref(out)),
              "GetSortKeysTempStorageBytes")
        return out.value

    @staticmethod
    def GetSortPairsTempStorageBytes(key_dtype: int, value_dtype: int, num_items: int) -> int:
        out = ctypes.c_size_t()
        check(lib().lcpp_radix_sort_pairs_temp_bytes(key_dtype, value_dtype, num_items,
                                                     ctypes.byref(out)),
              "GetSortPairsTempStorageBytes")
        return out.value

    def _keys(self, temp, kin, kout, n, begin, end, desc, stream):
        kd = dtype_code(kin)
        end = kin.element_size() * 8 if end is None else end
        check(lib().lcpp_radix_sort_keys(_ptr(temp), temp.numel() if temp is not None else 0,
                                         _ptr(kin), _ptr(kout), n, begin, end, int(desc), kd,
                                         _stream(stream)), "SortKeys")

    def _pairs(self, temp, kin, kout, vin, vout, n, begin, end, desc, stream):
        kd, vd = dtype_code(kin), dtype_code(vin)
        end = kin.element_size() * 8 if end is None else end
        check(lib().lcpp_radix_sort_pairs(_ptr(temp), temp.numel() if temp is not None else 0,
                                          _ptr(kin), _ptr(kout), _ptr(vin), _ptr(vout), n, begin,
                                          end, int(desc), kd, vd, _stream(stream)), "SortPairs")

    # Overloads as in the reference: copy form (temp, keys_in, keys_out, n, begin, end) and
    # DoubleBuffer form (temp, keys_db, n, begin, end) (device_radix_sort.h:369-555).
    def SortKeys(self, temp, *args, stream=None):
        self._dispatch_keys(temp, args, False, stream)

    def SortKeysDescending(self, temp, *args, stream=None):
        self._dispatch_keys(temp, args, True, stream)

    # Copy form (temp, keys_in, keys_out, values_in, values_out, n, begin, end) and
    # DoubleBuffer form (temp, keys_db, values_db, n, begin, end).
    def SortPairs(self, temp, *args, stream=None):
        self._dispatch_pairs(temp, args, False, stream)

    def SortPairsDescending(self, temp, *args, stream=None):
        self._dispatch_pairs(temp, args, True, stream)

    def _decomposed(self, temp, args, desc, stream, pairs):
        tb = temp.numel() if temp is not None else 0
        st = _stream(stream)
        if isinstance(args[0], DoubleBuffer):
            if pairs:
                kdb, vdb, n, dec, *rest = args
                if kdb.selector != vdb.selector:
                    raise LcppError(ERR_INVALID_ARG, "key and value DoubleBuffer selectors must match")
            else:
                kdb, n, dec, *rest = args
            begin, end = _bit_range(rest)
            end = dec.bits if end is None else end
            kb = (ctypes.c_void_p * 2)(kdb.d_buffers[0].data_ptr(), kdb.d_buffers[1].data_ptr())
            sel = ctypes.c_int(kdb.selector)
            if pairs:
                vb = (ctypes.c_void_p * 2)(vdb.d_buffers[0].data_ptr(), vdb.d_buffers[1].data_ptr())
                check(lib().lcpp_radix_sort_decomposed_pairs_double_buffer(
                    _ptr(temp), tb, kb, vb, ctypes.byref(sel), n, dec.key_bytes, dec._arr, len(dec.members), begin,
                    end, int(desc), dtype_code(vdb.d_buffers[0]), st), "SortPairs(decomposed, DoubleBuffer)")
                vdb.selector = sel.value
            else:
                check(lib().lcpp_radix_sort_decomposed_keys_double_buffer(
                    _ptr(temp), tb, kb, ctypes.byref(sel), n, dec.key_bytes, dec._arr, len(dec.members), begin, end,
                    int(desc), st), "SortKeys(decomposed, DoubleBuffer)")
            kdb.selector = sel.value
            return
        if pairs:
            kin, kout, vin, vout, n, dec, *rest = args
        else:
            kin, kout, n, dec, *rest = args
        begin, end = _bit_range(rest)
        end = dec.bits if end is None else end
        if pairs:
            check(lib().lcpp_radix_sort_decomposed_pairs(
                _ptr(temp), tb, _ptr(kin), _ptr(kout), _ptr(vin), _ptr(vout), n, dec.key_bytes, dec._arr,
                len(dec.members), begin, end, int(desc), dtype_code(vin), st), "SortPairs(decomposed)")
        else:
            check(lib().lcpp_radix_sort_decomposed_keys(
                _ptr(temp), tb, _ptr(kin), _ptr(kout), n, dec.key_bytes, dec._arr, len(dec.members), begin, end,
                int(desc), st), "SortKeys(decomposed)")

    def _dispatch_keys(self, temp, args, desc, stream):
        if any(isinstance(a, Decomposer) for a in args):
            return self._decomposed(temp, args, desc, stream, False)
        if isinstance(args[0], DoubleBuffer):
            db, n, *rest = args
            begin, end = _bit_range(rest)
            return self._keys_db(temp, db, n, begin, end, desc, stream)
        kin, kout, n, *rest = args
        begin, end = _bit_range(rest)
        self._keys(temp, kin, kout, n, begin, end, desc, stream)

    def _dispatch_pairs(self, temp, args, desc, stream):
        if any(isinstance(a, Decomposer) for a in args):
            return self._decomposed(temp, args, desc, stream, True)
        if isinstance(args[0], DoubleBuffer):
            kdb, vdb, n, *rest = args
            begin, end = _bit_range(rest)
            return self._pairs_db(temp, kdb, vdb, n, begin, end, desc, stream)
        kin, kout, vin, vout, n, *rest = args
        begin, end = _bit_range(rest)
        self._pairs(temp, kin, kout, vin, vout, n, begin, end, desc, stream)

    # DoubleBuffer forms: SortKeys(temp, db, n, begin, end)
    def _keys_db(self, temp, db, n, begin, end, desc, stream):
        kd = dtype_code(db.d_buffers[0])
        end = db.d_buffers[0].element_size() * 8 if end is None else end
        bufs = (ctypes.c_void_p * 2)(db.d_buffers[0].data_ptr(), db.d_buffers[1].data_ptr())
        sel = ctypes.c_int(db.selector)
        check(lib().lcpp_radix_sort_keys_double_buffer(
            _ptr(temp), temp.numel() if temp is not None else 0, bufs, ctypes.byref(sel), n,
            begin, end, int(desc), kd, _stream(stream)), "SortKeys(DoubleBuffer)")
        db.selector = sel.value

    def _pairs_db(self, temp, kdb, vdb, n, begin, end, desc, stream):
        if kdb.selector != vdb.selector:
            raise LcppError(ERR_INVALID_ARG, "key and value DoubleBuffer selectors must match")
        kd, vd = dtype_code(kdb.d_buffers[0]), dtype_code(vdb.d_buffers[0])
        end = kdb.d_buffers[0].element_size() * 8 if end is None else end
        kb = (ctypes.c_void_p * 2)(kdb.d_buffers[0].data_ptr(), kdb.d_buffers[1].data_ptr())
        vb = (ctypes.c_void_p * 2)(vdb.d_buffers[0].data_ptr(), vdb.d_buffers[1].data_ptr())
        sel = ctypes.c_int(kdb.selector)
        check(lib().lcpp_radix_sort_pairs_double_buffer(
            _ptr(temp), temp.numel() if temp is not None else 0, kb, vb, ctypes.byref(sel), n,
            begin, end, int(desc), kd, vd, _stream(stream)), "SortPairs(DoubleBuffer)")
        kdb.selector = vdb.selector = sel.value


class DeviceSegmentedRadixSort:
    """Mirror of lcpp::DeviceSegmentedRadixSort
    (src/lcpp/device/device_segmented_radix_sort.h:16-246): copy form
    (temp, keys_in, keys_out, n, num_segments, begin_offsets, end_offsets,
    begin_bit, end_bit) and DoubleBuffer form (temp, keys_db, n, num_segments,
    begin_offsets, end_offsets, begin_bit, end_bit); offsets are uint32 device
    tensors."""

    @staticmethod
    def GetSortKeysTempStorageBytes(key_dtype: int, num_items: int) -> int:
        out = ctypes.c_size_t()
        check(lib().lcpp_segmented_radix_sort_keys_temp_bytes(key_dtype, num_items, ctypes.byref(out)),
              "GetSortKeysTempStorageBytes")
        return out.value

    @staticmethod
    def GetSortPairsTempStorageBytes(key_dtype: int, value_dtype: int, num_items: int) -> int:
        out = ctypes.c_size_t()
        check(lib().lcpp_segmented_radix_sort_pairs_temp_bytes(key_dtype, value_dtype, num_items,
                                                               ctypes.byref(out)), "GetSortPairsTempStorageBytes")
        return out.value

    def SortKeys(self, temp, *args, stream=None):
        self._keys(temp, args, False, stream)

    def SortKeysDescending(self, temp, *args, stream=None):
        self._keys(temp, args, True, stream)

    def SortPairs(self, temp, *args, stream=None):
        self._pairs(temp, args, False, stream)

    def SortPairsDescending(self, temp, *args, stream=None):
        self._pairs(temp, args, True, stream)

    def _keys(self, temp, args, desc, stream):
        tb = temp.numel() if temp is not None else 0
        if isinstance(args[0], DoubleBuffer):
            db, n, nseg, bo, eo, *rest = args
            begin, end = _bit_range(rest)
            k0 = db.d_buffers[0]
            end = k0.element_size() * 8 if end is None else end
            bufs = (ctypes.c_void_p * 2)(db.d_buffers[0].data_ptr(), db.d_buffers[1].data_ptr())
            sel = ctypes.c_int(db.selector)
            check(lib().lcpp_segmented_radix_sort_keys_double_buffer(
                _ptr(temp), tb, bufs, ctypes.byref(sel), n, nseg, _ptr(bo), _ptr(eo), begin, end, int(desc),
                dtype_code(k0), _stream(stream)), "SortKeys(DoubleBuffer)")
            db.selector = sel.value
            return
        kin, kout, n, nseg, bo, eo, *rest = args
        begin, end = _bit_range(rest)
        end = kin.element_size() * 8 if end is None else end
        check(lib().lcpp_segmented_radix_sort_keys(_ptr(temp), tb, _ptr(kin), _ptr(kout), n, nseg, _ptr(bo),
                                                   _ptr(eo), begin, end, int(desc), dtype_code(kin),
                                                   _stream(stream)), "SortKeys")

    def _pairs(self, temp, args, desc, stream):
        tb = temp.numel() if temp is not None else 0
        if isinstance(args[0], DoubleBuffer):
            kdb, vdb, n, nseg, bo, eo, *rest = args
            if kdb.selector != vdb.selector:
                raise LcppError(ERR_INVALID_ARG, "key and value DoubleBuffer selectors must match")
            begin, end = _bit_range(rest)
            k0, v0 = kdb.d_buffers[0], vdb.d_buffers[0]
            end = k0.element_size() * 8 if end is None else end
            kb = (ctypes.c_void_p * 2)(kdb.d_buffers[0].data_ptr(), kdb.d_buffers[1].data_ptr())
            vb = (ctypes.c_void_p * 2)(vdb.d_buffers[0].data_ptr(), vdb.d_buffers[1].data_ptr())
            sel = ctypes.c_int(kdb.selector)
            check(lib().lcpp_segmented_radix_sort_pairs_double_buffer(
                _ptr(temp), tb, kb, vb, ctypes.byref(sel), n, nseg, _ptr(bo), _ptr(eo), begin, end, int(desc),
                dtype_code(k0), dtype_code(v0), _stream(stream)), "SortPairs(DoubleBuffer)")
            kdb.selector = vdb.selector = sel.value
            return
        kin, kout, vin, vout, n, nseg, bo, eo, *rest = args
        begin, end = _bit_range(rest)
        end = kin.element_size() * 8 if end is None else end
        check(lib().lcpp_segmented_radix_sort_pairs(_ptr(temp), tb, _ptr(kin), _ptr(kout), _ptr(vin), _ptr(vout),
                                                    n, nseg, _ptr(bo), _ptr(eo), begin, end, int(desc),
                                                    dtype_code(kin), dtype_code(vin), _stream(stream)), "SortPairs")


class DeviceScan:
    """Mirror of lcpp::DeviceScan (src/lcpp/device/device_scan.h:40-1560)."""

    @staticmethod
    def GetTempStorageBytes(dtype: int, num_items: int) -> int:
        out = ctypes.c_size_t()
        check(lib().lcpp_scan_temp_bytes(dtype, num_items, ctypes.byref(out)), "GetTempStorageBytes")
        return out.value

    def ExclusiveSum(self, temp, d_in, d_out, num_items, stream=None):
        check(lib().lcpp_scan_exclusive_sum(_ptr(temp), temp.numel() if temp is not None else 0,
                                            _ptr(d_in), _ptr(d_out), num_items, dtype_code(d_in),
                                            _stream(stream)), "ExclusiveSum")

    def InclusiveSum(self, temp, d_in, d_out, num_items, stream=None):
        check(lib().lcpp_scan_inclusive_sum(_ptr(temp), temp.numel() if temp is not None else 0,
                                            _ptr(d_in), _ptr(d_out), num_items, dtype_code(d_in),
                                            _stream(stream)), "InclusiveSum")

    def ExclusiveScan(self, temp, d_in, d_out, num_items, op, initial_value, stream=None):
        code = dtype_code(d_in)
        keep, init = _host_scalar(initial_value, code)
        check(lib().lcpp_scan_exclusive(_ptr(temp), temp.numel() if temp is not None else 0,
                                        _ptr(d_in), _ptr(d_out), num_items, op, init, code,
                                        _stream(stream)), "ExclusiveScan")
        del keep

    def InclusiveScan(self, temp, d_in, d_out, num_items, op, initial_value=None, stream=None):
        code = dtype_code(d_in)
        if initial_value is None:
            check(lib().lcpp_scan_inclusive(_ptr(temp), temp.numel() if temp is not None else 0,
                                            _ptr(d_in), _ptr(d_out), num_items, op, code,
                                            _stream(stream)), "InclusiveScan")
        else:
            self.InclusiveScanInit(temp, d_in, d_out, num_items, op, initial_value, stream)

    def InclusiveScanInit(self, temp, d_in, d_out, num_items, op, initial_value, stream=None):
        code = dtype_code(d_in)
        keep, init = _host_scalar(initial_value, code)
        check(lib().lcpp_scan_inclusive_init(_ptr(temp), temp.numel() if temp is not None else 0,
                                             _ptr(d_in), _ptr(d_out), num_items, op, init, code,
                                             _stream(stream)), "InclusiveScanInit")
        del keep

    # ---- counting scans (device_scan.h:387-406)
    @staticmethod
    def GetTransformTempStorageBytes(num_items: int) -> int:
        out = ctypes.c_size_t()
        check(lib().lcpp_scan_transform_temp_bytes(num_items, ctypes.byref(out)), "GetTransformTempStorageBytes")
        return out.value

    def ExclusiveSumTransform(self, temp, d_in, d_out, num_items, pred, stream=None):
        """d_out[i] (4-byte tensor) = how many of d_in[0..i) satisfy pred (a Pred)."""
        code = dtype_code(d_in)
        arr, n = pred.encode(code)
        check(lib().lcpp_scan_exclusive_sum_transform(_ptr(temp), temp.numel() if temp is not None else 0,
                                                      _ptr(d_in), _ptr(d_out), num_items, code, arr, n,
                                                      _stream(stream)), "ExclusiveSumTransform")

    def ExclusiveSumAdjacent(self, temp, d_in, d_out, num_items, stream=None):
        """d_out[i] = how many runs of equal items start before i."""
        check(lib().lcpp_scan_exclusive_sum_adjacent(_ptr(temp), temp.numel() if temp is not None else 0,
                                                     _ptr(d_in), _ptr(d_out), num_items, dtype_code(d_in),
                                                     _stream(stream)), "ExclusiveSumAdjacent")

    # ---- by key (device_scan.h:310-597): argument order as the reference's
    @staticmethod
    def GetScanByKeyTempStorageBytes(key_dtype: int, value_dtype: int, num_items: int) -> int:
        out = ctypes.c_size_t()
        check(lib().lcpp_scan_by_key_temp_bytes(key_dtype, value_dtype, num_items, ctypes.byref(out)),
              "GetScanByKeyTempStorageBytes")
        return out.value

    def ExclusiveScanByKey(self, temp, d_keys_in, d_values_in, d_values_out, scan_op, num_items, initial_value,
                           stream=None):
        vc = dtype_code(d_values_in)
        keep, init = _host_scalar(initial_value, vc)
        check(lib().lcpp_scan_exclusive_by_key(_ptr(temp), temp.numel() if temp is not None else 0,
                                               _ptr(d_keys_in), _ptr(d_values_in), _ptr(d_values_out), num_items,
                                               scan_op, init, dtype_code(d_keys_in), vc, _stream(stream)),
              "ExclusiveScanByKey")
        del keep

    def InclusiveScanByKey(self, temp, d_keys_in, d_values_in, d_values_out, scan_op, num_items,
                           initial_value=None, stream=None):
        vc = dtype_code(d_values_in)
        t = (_ptr(temp), temp.numel() if temp is not None else 0, _ptr(d_keys_in), _ptr(d_values_in),
             _ptr(d_values_out), num_items, scan_op)
        if initial_value is None:
            check(lib().lcpp_scan_inclusive_by_key(*t, dtype_code(d_keys_in), vc, _stream(stream)),
                  "InclusiveScanByKey")
        else:
            keep, init = _host_scalar(initial_value, vc)
            check(lib().lcpp_scan_inclusive_by_key_init(*t, init, dtype_code(d_keys_in), vc, _stream(stream)),
                  "InclusiveScanByKey")
            del keep

    def ExclusiveSumByKey(self, temp, d_keys_in, d_values_in, d_values_out, num_items, stream=None):
        check(lib().lcpp_scan_exclusive_sum_by_key(_ptr(temp), temp.numel() if temp is not None else 0,
                                                   _ptr(d_keys_in), _ptr(d_values_in), _ptr(d_values_out),
                                                   num_items, dtype_code(d_keys_in), dtype_code(d_values_in),
                                                   _stream(stream)), "ExclusiveSumByKey")

    def InclusiveSumByKey(self, temp, d_keys_in, d_values_in, d_values_out, num_items, stream=None):
        check(lib().lcpp_scan_inclusive_sum_by_key(_ptr(temp), temp.numel() if temp is not None else 0,
                                                   _ptr(d_keys_in), _ptr(d_values_in), _ptr(d_values_out),
                                                   num_items, dtype_code(d_keys_in), dtype_code(d_values_in),
                                                   _stream(stream)), "InclusiveSumByKey")


class DeviceReduce:
    """Mirror of lcpp::DeviceReduce (src/lcpp/device/device_reduce.h:102-1187)."""

    @staticmethod
    def GetTempStorageBytes(dtype: int, num_items: int) -> int:
        out = ctypes.c_size_t()
        check(lib().lcpp_reduce_temp_bytes(dtype, num_items, ctypes.byref(out)), "GetTempStorageBytes")
        return out.value

    def Reduce(self, temp, d_in, d_out, num_items, op, initial_value, stream=None):
        code = dtype_code(d_in)
        keep, init = _host_scalar(initial_value, code)
        check(lib().lcpp_reduce(_ptr(temp), temp.numel() if temp is not None else 0, _ptr(d_in),
                                _ptr(d_out), num_items, op, init, code, _stream(stream)), "Reduce")
        del keep

    def _named(self, fn, temp, d_in, d_out, num_items, stream, what):
        check(fn(_ptr(temp), temp.numel() if temp is not None else 0, _ptr(d_in), _ptr(d_out),
                 num_items, dtype_code(d_out), _stream(stream)), what)

    @staticmethod
    def GetReduceByKeyTempStorageBytes(key_dtype: int, value_dtype: int, num_items: int) -> int:
        out = ctypes.c_size_t()
        check(lib().lcpp_reduce_by_key_temp_bytes(key_dtype, value_dtype, num_items, ctypes.byref(out)),
              "GetReduceByKeyTempStorageBytes")
        return out.value

    def ReduceByKey(self, temp, d_keys_in, d_values_in, d_unique_out, d_aggregates_out, d_num_runs_out,
                    reduce_op, num_elements, stream=None):
        """device_reduce.h:437-491 (argument order as the reference's);
        d_num_runs_out: a one-element 4-byte tensor (uint32 run count)."""
        check(lib().lcpp_reduce_by_key(_ptr(temp), temp.numel() if temp is not None else 0, _ptr(d_keys_in),
                                       _ptr(d_values_in), _ptr(d_unique_out), _ptr(d_aggregates_out),
                                       _ptr(d_num_runs_out), num_elements, reduce_op, dtype_code(d_keys_in),
                                       dtype_code(d_values_in), _stream(stream)), "ReduceByKey")

    @staticmethod
    def GetArgTempStorageBytes(dtype: int, num_items: int) -> int:
        out = ctypes.c_size_t()
        check(lib().lcpp_reduce_arg_temp_bytes(dtype, num_items, ctypes.byref(out)), "GetArgTempStorageBytes")
        return out.value

    def ArgMin(self, temp, d_in, d_out, d_index_out, num_items, stream=None):
        """d_out[0] = min value, d_index_out[0] = its first index (uint32 / int32 tensor)."""
        check(lib().lcpp_reduce_argmin(_ptr(temp), temp.numel() if temp is not None else 0, _ptr(d_in), _ptr(d_out),
                                       _ptr(d_index_out), num_items, dtype_code(d_out), _stream(stream)), "ArgMin")

    def ArgMax(self, temp, d_in, d_out, d_index_out, num_items, stream=None):
        check(lib().lcpp_reduce_argmax(_ptr(temp), temp.numel() if temp is not None else 0, _ptr(d_in), _ptr(d_out),
                                       _ptr(d_index_out), num_items, dtype_code(d_out), _stream(stream)), "ArgMax")

    def Sum(self, temp, d_in, d_out, num_items, stream=None):
        self._named(lib().lcpp_reduce_sum, temp, d_in, d_out, num_items, stream, "Sum")

    def Min(self, temp, d_in, d_out, num_items, stream=None):
        self._named(lib().lcpp_reduce_min, temp, d_in, d_out, num_items, stream, "Min")

    def Max(self, temp, d_in, d_out, num_items, stream=None):
        self._named(lib().lcpp_reduce_max, temp, d_in, d_out, num_items, stream, "Max")


def device_status(temp, stream=None) -> int:
    """Synchronise and read the device error word of the call that used `temp`."""
    return lib().lcpp_device_status(_ptr(temp), _stream(stream))


def testgen_fill(dst, dist: int, seed: int, offset: int = 0, stream=None) -> None:
    check(lib().lcpp_testgen_fill(_ptr(dst), dst.numel(), offset, seed, dist, _stream(stream)),
          "testgen_fill")


def diag_timing_enable(enable: bool) -> None:
    """Record CUDA events around every library kernel launch (lcpp_b200_diag.h)."""
    check(lib().lcpp_diag_timing_enable(int(enable)), "diag_timing_enable")


def diag_timing_read() -> list[tuple[int, float, int]]:
    """(kind, ms, items) of every launch recorded since timing was enabled."""
    count = ctypes.c_int()
    check(lib().lcpp_diag_timing_read(None, 0, ctypes.byref(count)), "diag_timing_read")
    buf = (KernelTime * max(count.value, 1))()
    check(lib().lcpp_diag_timing_read(buf, count.value, ctypes.byref(count)), "diag_timing_read")
    return [(buf[i].kind, buf[i].ms, buf[i].items) for i in range(count.value)]


def _tb(temp):
    return temp.numel() if temp is not None else 0


class DeviceSelect:
    """Mirror of lcpp::DeviceSelect (src/lcpp/device/device_select.h); the
    predicate arguments are Pred objects.  Passing d_out = d_in (or omitting
    it in the in-place helpers) compacts in place."""

    @staticmethod
    def GetTempStorageBytes(num_items: int) -> int:
        out = ctypes.c_size_t()
        check(lib().lcpp_select_temp_bytes(num_items, ctypes.byref(out)), "GetTempStorageBytes")
        return out.value

    def Flagged(self, temp, d_in, d_flags, d_out, d_num_selected_out, num_items, stream=None):
        check(lib().lcpp_select_flagged(_ptr(temp), _tb(temp), _ptr(d_in), _ptr(d_flags), _ptr(d_out),
                                        _ptr(d_num_selected_out), num_items, dtype_code(d_in), flag_code(d_flags),
                                        _stream(stream)), "Flagged")

    def FlaggedIf(self, temp, d_in, d_flags, d_out, d_num_selected_out, num_items, pred: Pred, stream=None):
        fc = flag_code(d_flags)
        arr, n = pred.encode(fc)
        check(lib().lcpp_select_flagged_if(_ptr(temp), _tb(temp), _ptr(d_in), _ptr(d_flags), _ptr(d_out),
                                           _ptr(d_num_selected_out), num_items, dtype_code(d_in), fc, arr, n,
                                           _stream(stream)), "FlaggedIf")

    def If(self, temp, d_in, d_out, d_num_selected_out, num_items, pred: Pred, stream=None):
        code = dtype_code(d_in)
        arr, n = pred.encode(code)
        check(lib().lcpp_select_if(_ptr(temp), _tb(temp), _ptr(d_in), _ptr(d_out), _ptr(d_num_selected_out),
                                   num_items, code, arr, n, _stream(stream)), "If")

    def Unique(self, temp, d_in, d_out, d_num_selected_out, num_items, stream=None):
        check(lib().lcpp_select_unique(_ptr(temp), _tb(temp), _ptr(d_in), _ptr(d_out), _ptr(d_num_selected_out),
                                       num_items, dtype_code(d_in), _stream(stream)), "Unique")

    def UniqueByKey(self, temp, d_keys_in, d_values_in, d_keys_out, d_values_out, d_num_selected_out, num_items,
                    stream=None):
        check(lib().lcpp_select_unique_by_key(_ptr(temp), _tb(temp), _ptr(d_keys_in), _ptr(d_values_in),
                                              _ptr(d_keys_out), _ptr(d_values_out), _ptr(d_num_selected_out),
                                              num_items, dtype_code(d_keys_in), dtype_code(d_values_in),
                                              _stream(stream)), "UniqueByKey")


class DevicePartition:
    """Mirror of lcpp::DevicePartition (src/lcpp/device/device_partition.h):
    selected items in order from the front, rejected ones in reverse order
    from the back."""

    @staticmethod
    def GetTempStorageBytes(num_items: int) -> int:
        out = ctypes.c_size_t()
        check(lib().lcpp_partition_temp_bytes(num_items, ctypes.byref(out)), "GetTempStorageBytes")
        return out.value

    @staticmethod
    def GetThreeWayTempStorageBytes(num_items: int) -> int:
        out = ctypes.c_size_t()
        check(lib().lcpp_partition_three_way_temp_bytes(num_items, ctypes.byref(out)),
              "GetThreeWayTempStorageBytes")
        return out.value

    def Flagged(self, temp, d_in, d_flags, d_out, d_num_selected_out, num_items, stream=None):
        check(lib().lcpp_partition_flagged(_ptr(temp), _tb(temp), _ptr(d_in), _ptr(d_flags), _ptr(d_out),
                                           _ptr(d_num_selected_out), num_items, dtype_code(d_in),
                                           flag_code(d_flags), _stream(stream)), "Flagged")

    def If(self, temp, d_in, d_out, d_num_selected_out, num_items, pred: Pred, stream=None):
        code = dtype_code(d_in)
        arr, n = pred.encode(code)
        check(lib().lcpp_partition_if(_ptr(temp), _tb(temp), _ptr(d_in), _ptr(d_out), _ptr(d_num_selected_out),
                                      num_items, code, arr, n, _stream(stream)), "If")

    def IfThreeWay(self, temp, d_in, d_first_out, d_second_out, d_unselected_out, d_num_selected_out, num_items,
                   select_first: Pred, select_second: Pred, stream=None):
        """The reference's three-way If overload (device_partition.h:157-227);
        d_num_selected_out holds two counts."""
        code = dtype_code(d_in)
        a1, n1 = select_first.encode(code)
        a2, n2 = select_second.encode(code)
        check(lib().lcpp_partition_if_three_way(_ptr(temp), _tb(temp), _ptr(d_in), _ptr(d_first_out),
                                                _ptr(d_second_out), _ptr(d_unselected_out),
                                                _ptr(d_num_selected_out), num_items, code, a1, n1, a2, n2,
                                                _stream(stream)), "IfThreeWay")


# ---------------------------------------------------------------------------
# Operators of one language-model step (include/lcpp_b200_model.h)
# ---------------------------------------------------------------------------
_ROW_CODES = None


def _row_code(t) -> int:
    """dtype code of logits or token rows."""
    global _ROW_CODES
    if _ROW_CODES is None:
        torch = _torch()
        _ROW_CODES = {torch.float32: F32, torch.float16: F16, torch.bfloat16: BF16}
    code = _ROW_CODES.get(t.dtype)
    if code is None:
        raise TypeError(f"unsupported dtype {t.dtype}")
    return code


def _flat(t, dtype, count, name):
    """Pointer of a contiguous tensor of `dtype` with at least `count` elements (None stays None)."""
    if t is None:
        return None
    if t.dtype != dtype or not t.is_contiguous() or t.numel() < count:
        raise LcppError(ERR_INVALID_ARG, f"{name}: contiguous {dtype} with at least {count} elements")
    if not t.is_cuda:
        raise LcppError(ERR_INVALID_ARG, f"{name}: a CUDA tensor")
    return t.data_ptr()


def _rows(t, rows, columns, code, name):
    """(pointer, row stride) of a 2-D tensor of at least rows x columns with unit column stride."""
    shape = t.shape
    if _row_code(t) != code or len(shape) != 2 or shape[0] < rows or shape[1] < columns:
        raise LcppError(ERR_INVALID_ARG, f"{name}: rows of one dtype, at least {rows} x {columns}")
    stride = t.stride()
    if stride[1] != 1 and shape[1] > 1 and shape[0]:
        raise LcppError(ERR_INVALID_ARG, f"{name}: a row's columns have to be adjacent")
    if not t.is_cuda:
        raise LcppError(ERR_INVALID_ARG, f"{name}: a CUDA tensor")
    return t.data_ptr(), (stride[0] if shape[0] > 1 else max(stride[0], columns))


_raw_stream = None


def _queue(stream, device=None):
    """Handle of the stream to enqueue on: the one given, else torch's current one."""
    global _raw_stream
    if stream is not None:
        return stream.cuda_stream
    if _raw_stream is None:
        torch = _torch()
        # the handle without a Stream object around it, where torch offers it
        _raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream",
                              lambda device: torch.cuda.current_stream(device).cuda_stream)
    return _raw_stream(_torch().cuda.current_device() if device is None else device)


_FORMATS = {ctypes.c_void_p: "Q", ctypes.c_uint64: "Q", ctypes.c_uint32: "I", ctypes.c_int: "i", ctypes.c_float: "f"}


def _packer(structure):
    """struct.Struct.pack for a ctypes structure's fields, those of nested ones in their place: a call's arguments
    are put together several times faster than by the structure itself."""
    import struct

    def fields(kind, at):
        for name, field in kind._fields_:
            offset = at + getattr(kind, name).offset
            if issubclass(field, ctypes.Structure):
                yield from fields(field, offset)
            else:
                yield offset, ctypes.sizeof(field), _FORMATS[field]

    text, end = "=", 0
    for offset, size, code in fields(structure, 0):
        text += f"{offset - end}x{code}"
        end = offset + size
    pack = struct.Struct(text + f"{ctypes.sizeof(structure) - end}x").pack

    def packed(*values):
        try:
            return pack(*values)
        except (struct.error, OverflowError) as error:  # a number that its field does not hold
            raise LcppError(ERR_INVALID_ARG, str(error)) from None

    return packed


_pack_rotary, _pack_append = _packer(RotaryArgs), _packer(CacheAppendArgs)
_pack_attention, _pack_evict, _pack_cache = _packer(PagedAttentionArgs), _packer(CacheEvictArgs), _packer(KVCache)


_current_device = None


def _device():
    """The current device, whose memory alone the kernels use (-2 without one, where no tensor is)."""
    global _current_device
    if _current_device is None:
        torch = _torch()
        if not torch.cuda.is_available():
            return -2
        torch.cuda.current_device()  # starts CUDA
        # the number without the checks around it, where torch offers it
        _current_device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)
    return _current_device()


def _array(t, dtype, count, name, device):
    """Pointer of a contiguous tensor of `dtype` with at least `count` elements on the device (None: 0)."""
    if t is None:
        return 0
    if t.dtype is not dtype or t.numel() < count or not t.is_contiguous():
        raise LcppError(ERR_INVALID_ARG, f"{name}: contiguous {dtype} with at least {count} elements")
    if t.get_device() != device:
        raise LcppError(ERR_INVALID_ARG, f"{name}: a CUDA tensor of the current device")
    return t.data_ptr()


def _heads(t, tokens, heads, dim, dtype, name, device):
    """(pointer, token stride, head stride) of a [tokens, heads, dim] tensor whose columns are adjacent."""
    shape, stride = t.shape, t.stride()
    if t.dtype is not dtype or len(shape) != 3 or shape[0] < tokens or shape[1] != heads or shape[2] != dim:
        raise LcppError(ERR_INVALID_ARG, f"{name}: {dtype}, at least {tokens} x {heads} x {dim}")
    if stride[2] != 1 and dim > 1 and tokens:
        raise LcppError(ERR_INVALID_ARG, f"{name}: a head's columns have to be adjacent")
    if t.get_device() != device:
        raise LcppError(ERR_INVALID_ARG, f"{name}: a CUDA tensor of the current device")
    return t.data_ptr(), stride[0], stride[1]


def _kv_cache(k, v, device):
    """The lcpp_kv_cache's fields of two [pages, block_size, heads, dim] tensors of equal strides (those along a single
    entry do not matter)."""
    shape, stride, dtype = k.shape, k.stride(), k.dtype
    if len(shape) != 4 or v.shape != shape or v.dtype is not dtype or \
            (v.stride() != stride and any(a != b and n > 1 for a, b, n in zip(stride, v.stride(), shape))):
        raise LcppError(ERR_INVALID_ARG, "keys and values: [pages, block_size, heads, dim] of one dtype, shape and layout")
    if stride[3] != 1 and shape[3] > 1:
        raise LcppError(ERR_INVALID_ARG, "keys and values: a head's columns have to be adjacent")
    if k.get_device() != device or v.get_device() != device:
        raise LcppError(ERR_INVALID_ARG, "keys and values: CUDA tensors of the current device")
    return k.data_ptr(), v.data_ptr(), stride[0], stride[1], stride[2], *shape, _row_code(k)


def _table(t, rows, device):
    """(pointer, row stride, width) of an int32 block table of at least `rows` rows."""
    shape, stride = t.shape, t.stride()
    if t.dtype is not _torch().int32 or len(shape) != 2 or shape[0] < rows or (stride[1] != 1 and shape[1] > 1 and rows):
        raise LcppError(ERR_INVALID_ARG, "d_block_table: int32 [num_requests, width], columns adjacent")
    if t.get_device() != device:
        raise LcppError(ERR_INVALID_ARG, "d_block_table: a CUDA tensor of the current device")
    return t.data_ptr(), (stride[0] if rows > 1 else max(stride[0], shape[1])), shape[1]


def _moves(t, requests, name, device):
    """(pointer, pairs from request to request, pairs of a request) of an int64 [requests, moves, 2] tensor."""
    shape, stride = t.shape, t.stride()
    if t.dtype is not _torch().int64 or len(shape) != 3 or shape[2] != 2 or shape[0] < requests or stride[2] != 1 or \
            (stride[1] != 2 and shape[1] > 1) or (stride[0] % 2 and shape[0] > 1):
        raise LcppError(ERR_INVALID_ARG, f"{name}: int64 [num_requests, max_moves, 2], pairs adjacent")
    if t.get_device() != device:
        raise LcppError(ERR_INVALID_ARG, f"{name}: a CUDA tensor of the current device")
    return t.data_ptr(), (stride[0] // 2 if requests > 1 else max(stride[0] // 2, shape[1])), shape[1]


def _scratch(temp):
    """(pointer, bytes) of temp storage."""
    return (None, 0) if temp is None else (temp.data_ptr(), temp.numel() * temp.element_size())


_router_configs = {}


def _router_config(*fields):
    """The lcpp_router_config of these settings; a program uses few, so they are kept."""
    config = _router_configs.get(fields)
    if config is None:
        if len(_router_configs) >= 256:
            _router_configs.clear()
        config = _router_configs[fields] = RouterConfig(*fields)
    return config


class DeviceBlockTable:
    """Block tables and slot maps of a paged cache, from request lengths."""

    @staticmethod
    def GetTempStorageBytes(num_requests: int, max_tokens: int) -> int:
        out = ctypes.c_size_t()
        check(lib().lcpp_block_table_temp_bytes(num_requests, max_tokens, ctypes.byref(out)), "GetTempStorageBytes")
        return out.value

    def Extend(self, temp, d_context_lens, d_new_lens, d_block_table, d_free_blocks, d_free_used, d_free_used_out,
               d_seq_lens_out, d_query_starts_out, d_slots_out, d_positions_out, d_token_request_out, num_requests,
               block_size, stream=None):
        """Gives the step's tokens their pages and slots (lcpp_block_table_extend).

        d_block_table [num_requests, width] is extended in place; d_new_lens None
        adds one token to each request; d_free_used, d_positions_out and
        d_token_request_out may be None.  All tensors int32, d_slots_out int64;
        its length is the number of tokens laid out, padding included."""
        torch = _torch()
        i32, n, tokens = torch.int32, num_requests, d_slots_out.numel()
        if d_block_table.dtype != i32 or d_block_table.dim() != 2 or d_block_table.shape[0] < n or \
                (d_block_table.stride(1) != 1 and d_block_table.shape[1] > 1 and n):
            raise LcppError(ERR_INVALID_ARG, "d_block_table: int32 [num_requests, width], columns adjacent")
        if not d_block_table.is_cuda:
            raise LcppError(ERR_INVALID_ARG, "d_block_table: a CUDA tensor")
        width = d_block_table.shape[1]
        # as it is, for the library to refuse rows that share memory; of one request only its row counts
        stride = d_block_table.stride(0) if n > 1 else max(d_block_table.stride(0), width)
        args = BlockTableArgs(
            _flat(d_context_lens, i32, n, "d_context_lens"), _flat(d_new_lens, i32, n, "d_new_lens"),
            d_block_table.data_ptr(), stride, width, n, block_size,
            d_free_blocks.numel(), _flat(d_free_blocks, i32, 0, "d_free_blocks"),
            _flat(d_free_used, i32, 1, "d_free_used"), _flat(d_free_used_out, i32, 1, "d_free_used_out"),
            _flat(d_seq_lens_out, i32, n, "d_seq_lens_out"),
            _flat(d_query_starts_out, i32, n + 1, "d_query_starts_out"),
            _flat(d_slots_out, torch.int64, tokens, "d_slots_out"),
            _flat(d_positions_out, i32, tokens, "d_positions_out"),
            _flat(d_token_request_out, i32, tokens, "d_token_request_out"), tokens)
        check(lib().lcpp_block_table_extend(*_scratch(temp), args, _queue(stream)), "Extend")


class DeviceRouter:
    """Experts of each token, their weights, per-expert counts and the balance loss, with the gradient."""

    @staticmethod
    def GetTempStorageBytes(num_tokens: int, num_experts: int) -> int:
        out = ctypes.c_size_t()
        check(lib().lcpp_router_temp_bytes(num_tokens, num_experts, ctypes.byref(out)), "GetTempStorageBytes")
        return out.value

    def Forward(self, temp, d_logits, d_weights_out, d_experts_out, d_counts_out, d_num_routed_out, d_loss_out,
                num_tokens, num_experts, top_k, score=SCORE_SOFTMAX, renormalize=True, weight_scale=1.0,
                loss_coef=1.0, d_bias=None, d_token_request=None, stream=None):
        """lcpp_router_forward: d_logits [num_tokens, num_experts] float32, float16 or bfloat16;
        weights float32 and experts int32 [num_tokens, top_k], counts int32 [num_experts].
        d_bias [num_experts] float32 joins the logits in the choice, or the scores with
        score=SCORE_SIGMOID + BIAS_ON_SCORE (or SCORE_SOFTMAX + BIAS_ON_SCORE)."""
        torch = _torch()
        i32, f32, pairs, code = torch.int32, torch.float32, num_tokens * top_k, _row_code(d_logits)
        logits, stride = _rows(d_logits, num_tokens, num_experts, code, "d_logits")
        check(lib().lcpp_router_forward(
            *_scratch(temp), logits, stride, code, _flat(d_bias, f32, num_experts, "d_bias"),
            _flat(d_token_request, i32, num_tokens, "d_token_request"),
            _flat(d_weights_out, f32, pairs, "d_weights_out"), _flat(d_experts_out, i32, pairs, "d_experts_out"),
            _flat(d_counts_out, i32, num_experts, "d_counts_out"),
            _flat(d_num_routed_out, i32, 1, "d_num_routed_out"), _flat(d_loss_out, f32, 1, "d_loss_out"), num_tokens,
            _router_config(num_experts, top_k, score, int(renormalize), weight_scale, loss_coef), _queue(stream)),
            "Forward")

    def Backward(self, d_logits, d_experts, d_counts, d_num_routed, d_grad_weights, d_grad_loss, d_grad_logits_out,
                 num_tokens, num_experts, top_k, score=SCORE_SOFTMAX, renormalize=True, weight_scale=1.0,
                 loss_coef=1.0, stream=None):
        """lcpp_router_backward: experts, counts and num_routed as Forward wrote them;
        d_grad_weights and d_grad_loss may be None."""
        torch = _torch()
        i32, f32, pairs, code = torch.int32, torch.float32, num_tokens * top_k, _row_code(d_logits)
        logits, stride = _rows(d_logits, num_tokens, num_experts, code, "d_logits")
        grad, grad_stride = _rows(d_grad_logits_out, num_tokens, num_experts, code, "d_grad_logits_out")
        check(lib().lcpp_router_backward(
            logits, stride, code, _flat(d_experts, i32, pairs, "d_experts"),
            _flat(d_counts, i32, num_experts, "d_counts"), _flat(d_num_routed, i32, 1, "d_num_routed"),
            _flat(d_grad_weights, f32, pairs, "d_grad_weights"), _flat(d_grad_loss, f32, 1, "d_grad_loss"), grad,
            grad_stride, num_tokens,
            _router_config(num_experts, top_k, score, int(renormalize), weight_scale, loss_coef), _queue(stream)),
            "Backward")


class DeviceDispatch:
    """Token rows grouped by expert and summed back, with the gradients."""

    @staticmethod
    def GetTempStorageBytes(num_tokens: int, top_k: int, num_experts: int) -> int:
        out = ctypes.c_size_t()
        check(lib().lcpp_dispatch_temp_bytes(num_tokens, top_k, num_experts, ctypes.byref(out)),
              "GetTempStorageBytes")
        return out.value

    @staticmethod
    def MaxRows(num_tokens: int, top_k: int, num_experts: int, row_align: int = 1) -> int:
        """Rows that hold any choice when segments start at multiples of row_align."""
        out = ctypes.c_uint64()
        check(lib().lcpp_dispatch_max_rows(num_tokens, top_k, num_experts, row_align, ctypes.byref(out)), "MaxRows")
        return out.value

    def Plan(self, temp, d_experts, d_expert_starts_out, d_row_of_out, d_pair_of_out, num_tokens, top_k, num_experts,
             row_align=1, stream=None):
        """Groups the pairs by expert (lcpp_dispatch_plan); d_pair_of_out's length is max_rows.  All int32."""
        i32, pairs = _torch().int32, num_tokens * top_k
        check(lib().lcpp_dispatch_plan(
            *_scratch(temp), _flat(d_experts, i32, pairs, "d_experts"),
            _flat(d_expert_starts_out, i32, num_experts + 1, "d_expert_starts_out"),
            _flat(d_row_of_out, i32, pairs, "d_row_of_out"), _flat(d_pair_of_out, i32, 0, "d_pair_of_out"),
            num_tokens, top_k, num_experts, row_align, d_pair_of_out.numel(), _queue(stream)), "Plan")

    def Gather(self, d_x, d_row_of, d_pair_of, d_expert_starts, d_rows_out, num_tokens, top_k, num_experts,
               stream=None):
        """Token rows to their experts' rows (lcpp_dispatch_gather); d_rows_out has a row per entry of d_pair_of."""
        i32, code, hidden, rows = _torch().int32, _row_code(d_x), d_x.shape[1], d_pair_of.numel()
        x, x_stride = _rows(d_x, num_tokens, hidden, code, "d_x")
        out, out_stride = _rows(d_rows_out, rows, hidden, code, "d_rows_out")
        check(lib().lcpp_dispatch_gather(
            x, x_stride, _flat(d_row_of, i32, num_tokens * top_k, "d_row_of"), _flat(d_pair_of, i32, 0, "d_pair_of"),
            _flat(d_expert_starts, i32, num_experts + 1, "d_expert_starts"), out, out_stride, num_tokens, top_k,
            num_experts, rows, hidden, code, _queue(stream)), "Gather")

    def Combine(self, d_rows, d_row_of, d_weights, d_out, num_tokens, top_k, stream=None):
        """Sums of the tokens' rows, weighted unless d_weights is None (lcpp_dispatch_combine)."""
        torch = _torch()
        code, hidden, pairs = _row_code(d_rows), d_out.shape[1], num_tokens * top_k
        rows, rows_stride = _rows(d_rows, 0, hidden, code, "d_rows")
        out, out_stride = _rows(d_out, num_tokens, hidden, code, "d_out")
        check(lib().lcpp_dispatch_combine(
            rows, rows_stride, _flat(d_row_of, torch.int32, pairs, "d_row_of"),
            _flat(d_weights, torch.float32, pairs, "d_weights"), out, out_stride, num_tokens, top_k,
            d_rows.shape[0], hidden, code, _queue(stream)), "Combine")

    def CombineBackward(self, d_grad_out, d_rows, d_row_of, d_pair_of, d_expert_starts, d_weights, d_grad_rows_out,
                        d_grad_weights_out, num_tokens, top_k, num_experts, stream=None):
        """Gradients of Combine with weights (lcpp_dispatch_combine_backward)."""
        torch = _torch()
        i32, f32, pairs, max_rows = torch.int32, torch.float32, num_tokens * top_k, d_pair_of.numel()
        code, hidden = _row_code(d_grad_out), d_grad_out.shape[1]
        grad, grad_stride = _rows(d_grad_out, num_tokens, hidden, code, "d_grad_out")
        rows, rows_stride = _rows(d_rows, max_rows, hidden, code, "d_rows")
        out, out_stride = _rows(d_grad_rows_out, max_rows, hidden, code, "d_grad_rows_out")
        check(lib().lcpp_dispatch_combine_backward(
            grad, grad_stride, rows, rows_stride, _flat(d_row_of, i32, pairs, "d_row_of"),
            _flat(d_pair_of, i32, 0, "d_pair_of"), _flat(d_expert_starts, i32, num_experts + 1, "d_expert_starts"),
            _flat(d_weights, f32, pairs, "d_weights"), out, out_stride,
            _flat(d_grad_weights_out, f32, pairs, "d_grad_weights_out"), num_tokens, top_k, num_experts, max_rows,
            hidden, code, _queue(stream)), "CombineBackward")


class DeviceRotary:
    """Rotary positions of queries and keys, with the gradient and the write of keys and values into a paged cache."""

    @staticmethod
    def Frequencies(rotary_dim: int, base: float = 10000.0, scaling: int = ROTARY_PLAIN, factor: float = 1.0,
                    original_context: float = 0.0, low: float = 1.0, high: float = 4.0, device=None):
        """lcpp_rotary_frequencies as a CUDA tensor: float64 [rotary_dim / 2], radians per position."""
        torch = _torch()
        out = (ctypes.c_double * max(1, rotary_dim // 2))()
        check(lib().lcpp_rotary_frequencies(out, rotary_dim, base, scaling, factor, original_context, low, high),
              "Frequencies")
        return torch.tensor(list(out)[:rotary_dim // 2], dtype=torch.float64, device=device or "cuda")

    @staticmethod
    def _args(device, q, k, q_out, k_out, positions, frequencies, tokens, layout, scale, token_request,
              position_offset, append=False):
        """The fields of lcpp_rotary_args."""
        torch = _torch()
        some = k if q is None else q
        if some is None or some.dim() != 3:
            raise LcppError(ERR_INVALID_ARG, "d_q, d_k: [tokens, heads, dim]")
        dtype, code, dim = some.dtype, _row_code(some), some.shape[2]
        fields = []
        for x, out, name in ((q, q_out, "d_q"), (k, k_out, "d_k")):
            if x is None:
                fields += (0, 0, 0, 0, 0, 0, 0)
                continue
            heads = x.shape[1] if x.dim() == 3 else 0
            at, a, b = _heads(x, tokens, heads, dim, dtype, name, device)
            to, c, d = (0, 0, 0) if append and name == "d_k" else _heads(out, tokens, heads, dim, dtype, name + "_out", device)
            fields += (at, to, a, b, c, d, heads)
        requests = 0 if token_request is None else 0x7fffffff if position_offset is None else position_offset.numel()
        turned = frequencies.numel()
        return (*fields, _array(positions, torch.int32, tokens, "d_positions", device),
                _array(token_request, torch.int32, tokens, "d_token_request", device),
                _array(position_offset, torch.int32, 0, "d_position_offset", device),
                _array(frequencies, torch.float64, 0, "d_frequencies", device), tokens, requests, dim, 2 * turned,
                layout, scale, code)

    def Forward(self, d_q, d_k, d_q_out, d_k_out, d_positions, d_frequencies, num_tokens, layout=ROTARY_HALF, scale=1.0,
                d_token_request=None, d_position_offset=None, stream=None):
        """Turns q and k (either may be None) by their positions (lcpp_rotary_forward): [tokens, heads, dim] tensors
        with any strides of tokens and heads, in place where the output is the input; positions int32; as many
        columns as twice the frequencies (float64) are turned.  Tokens whose request (int32) is negative are left
        out; a request's offset (int32) is added to its tokens' positions."""
        device = _device()
        args = self._args(device, d_q, d_k, d_q_out, d_k_out, d_positions, d_frequencies, num_tokens, layout, scale,
                          d_token_request, d_position_offset)
        check(lib().lcpp_rotary_forward(_pack_rotary(*args), _queue(stream, device)), "Forward")

    def Backward(self, d_grad_q, d_grad_k, d_grad_q_out, d_grad_k_out, d_positions, d_frequencies, num_tokens,
                 layout=ROTARY_HALF, scale=1.0, d_token_request=None, d_position_offset=None, stream=None):
        """Gradients of Forward's inputs from those of its outputs (lcpp_rotary_backward)."""
        device = _device()
        args = self._args(device, d_grad_q, d_grad_k, d_grad_q_out, d_grad_k_out, d_positions, d_frequencies,
                          num_tokens, layout, scale, d_token_request, d_position_offset)
        check(lib().lcpp_rotary_backward(_pack_rotary(*args), _queue(stream, device)), "Backward")

    def Append(self, d_q, d_k, d_v, d_q_out, d_k_cache, d_v_cache, d_slots, d_positions, d_frequencies, num_tokens,
               layout=ROTARY_HALF, scale=1.0, d_token_request=None, d_position_offset=None, d_slot_positions=None,
               d_slot_scores=None, stream=None):
        """Forward for q (None: no queries), with keys and values going to their slots of the cache
        (lcpp_rotary_append): caches [pages, block_size, heads, dim] with any strides, slots int64 as
        DeviceBlockTable.Extend gives them.  d_slot_positions (int32, one per slot) gets the tokens' positions,
        d_slot_scores (float32) zeros."""
        torch, device = _torch(), _device()
        args = self._args(device, d_q, d_k, d_q_out, None, d_positions, d_frequencies, num_tokens, layout, scale,
                          d_token_request, d_position_offset, append=True)
        cache = _kv_cache(d_k_cache, d_v_cache, device)
        pages, block, heads, dim = cache[5:9]
        append = _pack_append(
            *cache, *_heads(d_v, num_tokens, heads, dim, d_k_cache.dtype, "d_v", device),
            _array(d_slots, torch.int64, num_tokens, "d_slots", device),
            _array(d_slot_positions, torch.int32, pages * block, "d_slot_positions", device),
            _array(d_slot_scores, torch.float32, pages * block, "d_slot_scores", device))
        check(lib().lcpp_rotary_append(_pack_rotary(*args), append, _queue(stream, device)), "Append")


class DevicePagedAttention:
    """Attention of one new token of each request over a paged cache."""

    @staticmethod
    def GetTempStorageBytes(num_requests: int, num_heads: int, num_kv_heads: int, head_dim: int,
                            score_slots: int = 0) -> int:
        """score_slots: pages * block_size when scores are wanted."""
        out = ctypes.c_size_t()
        check(lib().lcpp_paged_attention_temp_bytes(num_requests, num_heads, num_kv_heads, head_dim, score_slots,
                                                    ctypes.byref(out)), "GetTempStorageBytes")
        return out.value

    def Decode(self, temp, d_q, d_k_cache, d_v_cache, d_block_table, d_seq_lens, d_out, num_requests, scale=None,
               window=0, softcap=0.0, d_lse_out=None, d_scores=None, d_scores_out=None, score_decay=1.0, stream=None):
        """lcpp_paged_attention_decode: q and out [requests, heads, dim], caches [pages, block_size, kv_heads, dim]
        with any strides, block table and lengths int32 as DeviceBlockTable.Extend leaves them.  scale None:
        dim ** -0.5.  d_lse_out float32 [requests, heads]; scores float32, one per slot: the outputs are
        score_decay * d_scores (None: zeros) plus each token's attention weight, summed over the heads."""
        device, n, f32 = _device(), num_requests, _torch().float32
        cache = _kv_cache(d_k_cache, d_v_cache, device)
        slots, dim, dtype, heads = cache[5] * cache[6], cache[8], d_k_cache.dtype, d_q.shape[1] if d_q.dim() == 3 else 0
        table, table_stride, width = _table(d_block_table, n, device)
        args = _pack_attention(
            *cache, *_heads(d_q, n, heads, dim, dtype, "d_q", device), *_heads(d_out, n, heads, dim, dtype, "d_out", device),
            table, table_stride, width, n, _array(d_seq_lens, _torch().int32, n, "d_seq_lens", device), heads, window,
            dim ** -0.5 if scale is None else scale, softcap, _array(d_lse_out, f32, n * heads, "d_lse_out", device),
            _array(d_scores, f32, slots, "d_scores", device), _array(d_scores_out, f32, slots, "d_scores_out", device),
            score_decay)
        if temp is not None and (temp.get_device() != device or not temp.is_contiguous()):
            raise LcppError(ERR_INVALID_ARG, "temp: contiguous, a CUDA tensor of the current device")
        check(lib().lcpp_paged_attention_decode(*_scratch(temp), args, _queue(stream, device)), "Decode")


class DeviceCacheEviction:
    """Requests of a paged cache cut down to their heaviest tokens."""

    def Plan(self, d_seq_lens, d_block_table, d_scores, d_seq_lens_out, d_move_counts_out, d_moves_out, num_requests,
             block_size, budget, trigger=None, keep_first=0, keep_recent=0, d_positions=None, d_evicted=None,
             d_evicted_out=None, d_free_blocks=None, d_free_used=None, d_free_used_out=None, stream=None):
        """Chooses the tokens that stay (lcpp_cache_evict_plan): requests longer than trigger (None: budget) keep
        budget tokens, by d_scores (float32, one per slot).  d_moves_out int64 [requests, max_moves, 2]; the lengths
        and counts int32.  With the free list that DeviceBlockTable.Extend takes pages from, pages that are not
        needed any more go back to it."""
        torch, device, n = _torch(), _device(), num_requests
        i32 = torch.int32
        table, table_stride, width = _table(d_block_table, n, device)
        moves, moves_stride, max_moves = _moves(d_moves_out, n, "d_moves_out", device)
        if block_size < 1:
            raise LcppError(ERR_INVALID_ARG, "block_size: at least 1")
        pages = d_scores.numel() // block_size
        args = _pack_evict(
            _array(d_seq_lens, i32, n, "d_seq_lens", device), table, table_stride, width, n, pages, block_size,
            _array(d_scores, torch.float32, 0, "d_scores", device),
            _array(d_positions, i32, pages * block_size, "d_positions", device),
            _array(d_evicted, i32, n, "d_evicted", device), budget, budget if trigger is None else trigger, keep_first,
            keep_recent, max_moves, _array(d_seq_lens_out, i32, n, "d_seq_lens_out", device),
            _array(d_evicted_out, i32, n, "d_evicted_out", device),
            _array(d_move_counts_out, i32, n, "d_move_counts_out", device), moves, moves_stride,
            _array(d_free_blocks, i32, 0, "d_free_blocks", device), _array(d_free_used, i32, 1, "d_free_used", device),
            _array(d_free_used_out, i32, 1, "d_free_used_out", device),
            0 if d_free_blocks is None else d_free_blocks.numel())
        check(lib().lcpp_cache_evict_plan(args, _queue(stream, device)), "Plan")

    def Move(self, d_moves, d_move_counts, d_k_cache, d_v_cache, num_requests, d_scores=None, d_positions=None,
             stream=None):
        """Moves a layer's keys and values as a plan says (lcpp_cache_evict_move), and where given the scores and
        positions, which belong in one call only."""
        torch, device, n = _torch(), _device(), num_requests
        cache = _kv_cache(d_k_cache, d_v_cache, device)
        slots = cache[5] * cache[6]
        moves, moves_stride, max_moves = _moves(d_moves, n, "d_moves", device)
        check(lib().lcpp_cache_evict_move(
            _pack_cache(*cache), moves, moves_stride, max_moves,
            _array(d_move_counts, torch.int32, n, "d_move_counts", device), n,
            _array(d_scores, torch.float32, slots, "d_scores", device),
            _array(d_positions, torch.int32, slots, "d_positions", device), _queue(stream, device)), "Move")
