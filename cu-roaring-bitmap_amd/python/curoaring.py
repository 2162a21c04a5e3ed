"""ctypes binding of libcuroaring_amd.so (the C-ABI in include/cu_roaring_abi.h).

Used by the tests and bench.py.  Every call goes through the C-ABI into the HIP
library; there is no CPU fallback: load() raises when the built library is
missing.  Device buffers come from torch (plumbing only).
"""
from __future__ import annotations

import ctypes as C
import os
import struct
from types import SimpleNamespace
from typing import Optional, Sequence

import numpy as np

_HERE = os.path.dirname(os.path.abspath(__file__))
PKG_DIR = os.path.dirname(_HERE)
LIB_PATH = os.path.join(PKG_DIR, "lib", "libcuroaring_amd.so")

CR_OK = 0
CR_ERR_HIP, CR_ERR_INVALID, CR_ERR_ALLOC, CR_ERR_UNSUPPORTED, CR_ERR_RANGE = 1, 2, 3, 4, 5
ARRAY, BITMAP, RUN = 0, 1, 2
AND, OR, ANDNOT, XOR = 0, 1, 2, 3
PROMOTE_KEEP_DEFAULT = 4096
PROMOTE_ALL = 0
PROMOTE_AUTO = 0xFFFFFFFF
TC_BITSET, TC_ARRAY, TC_RUN = 1, 2, 3
QUERY_CONTAINS, QUERY_WAVEFRONT, QUERY_WAVEFRONT_API, QUERY_CONTAINS_API, QUERY_PARTITIONED = 0, 1, 2, 3, 4

EXPORTS = [
    "cr_last_error", "cr_upload_from_ids", "cr_upload_from_device_ids", "cr_upload_from_bitset",
    "cr_upload_from_device_bitset", "cr_upload_containers", "cr_get_meta", "cr_set_operation", "cr_multi_and",
    "cr_free", "cr_free_async", "cr_resolve_auto_threshold", "cr_make_view", "cr_contains_batch",
    "cr_topk_filtered", "cr_topk_set_small_limit", "cr_device_l2_bytes", "cr_device_malloc", "cr_device_free", "cr_memcpy_h2d",
    "cr_memcpy_d2h", "cr_stream_synchronize", "cr_timing_enable", "cr_timing_report", "cr_mempool_trim",
    "cr_decompress_to_bitset", "cr_decompress_to_bitset_alloc", "cr_enumerate_ids", "cr_enumerate_ids_alloc",
    "cr_enumerate_ids_noalloc", "cr_cardinality",
    "cr_promote_to_bitmap", "cr_promote_auto", "cr_deep_copy",
    "cr_portable_size_in_bytes", "cr_portable_serialize", "cr_portable_deserialize",
    "cr_upload_batch", "cr_free_batch", "cr_promote_batch", "cr_batch_make_view", "cr_batch_multi_and",
    "cr_batch_decompress", "cr_batch_contains", "cr_batch_view_contains", "cr_debug_fail_device_allocs",
    "cr_paged_plan", "cr_paged_append", "cr_paged_select", "cr_paged_attention", "cr_paged_rotary", "cr_paged_weights", "cr_paged_evict", "cr_paged_move",
    "cr_draft_verify", "cr_beam_select", "cr_beam_reorder",
]


class GpuRoaring(C.Structure):
    """cr_gpu_roaring == cu_roaring::GpuRoaring (include/cu_roaring/types.cuh:15-54)."""
    _fields_ = [
        ("keys", C.c_void_p),
        ("types", C.c_void_p),
        ("offsets", C.c_void_p),
        ("cardinalities", C.c_void_p),
        ("n_containers", C.c_uint32),
        ("universe_size", C.c_uint32),
        ("total_cardinality", C.c_uint64),
        ("bitmap_data", C.c_void_p),
        ("n_bitmap_containers", C.c_uint32),
        ("array_data", C.c_void_p),
        ("n_array_containers", C.c_uint32),
        ("array_pool_bytes", C.c_uint32),
        ("run_data", C.c_void_p),
        ("n_run_containers", C.c_uint32),
        ("run_pool_bytes", C.c_uint32),
        ("key_index", C.c_void_p),
        ("max_key", C.c_uint32),
        ("negated", C.c_bool),
        ("_alloc_base", C.c_void_p),
    ]


class GpuRoaringView(C.Structure):
    _fields_ = [
        ("keys", C.c_void_p),
        ("types", C.c_void_p),
        ("offsets", C.c_void_p),
        ("cardinalities", C.c_void_p),
        ("n_containers", C.c_uint32),
        ("bitmap_data", C.c_void_p),
        ("array_data", C.c_void_p),
        ("run_data", C.c_void_p),
        ("key_index", C.c_void_p),
        ("max_key", C.c_uint32),
        ("all_bitmap", C.c_bool),
        ("negated", C.c_bool),
    ]


class RoaringBatch(C.Structure):
    """cr_roaring_batch == cu_roaring::v2::GpuRoaringBatch (v2/include/cu_roaring_v2/types.cuh:37-86)."""
    _fields_ = [
        ("n_bitmaps", C.c_uint32), ("total_containers", C.c_uint32), ("n_bitmap_containers_total", C.c_uint32),
        ("array_pool_bytes", C.c_uint32), ("run_pool_bytes", C.c_uint32),
        ("container_starts", C.c_void_p), ("key_index_starts", C.c_void_p),
        ("keys", C.c_void_p), ("types", C.c_void_p), ("offsets", C.c_void_p), ("cardinalities", C.c_void_p),
        ("key_indices", C.c_void_p), ("bitmap_data", C.c_void_p), ("array_data", C.c_void_p),
        ("run_data", C.c_void_p),
        ("host_total_cardinalities", C.POINTER(C.c_uint64)), ("host_universe_sizes", C.POINTER(C.c_uint32)),
        ("host_container_starts", C.POINTER(C.c_uint32)), ("host_key_index_starts", C.POINTER(C.c_uint32)),
        ("host_n_bitmap_containers", C.POINTER(C.c_uint32)),
        ("_alloc_base", C.c_void_p), ("_host_meta_base", C.c_void_p),
    ]


class BatchView(C.Structure):
    """cr_batch_view == cu_roaring::v2::GpuRoaringView (v2/include/cu_roaring_v2/types.cuh:95-107)."""
    _fields_ = [
        ("n_containers", C.c_uint32), ("max_key", C.c_uint32),
        ("keys", C.c_void_p), ("types", C.c_void_p), ("offsets", C.c_void_p), ("cardinalities", C.c_void_p),
        ("key_index", C.c_void_p), ("bitmap_data", C.c_void_p), ("array_data", C.c_void_p), ("run_data", C.c_void_p),
    ]


class HostContainer(C.Structure):
    _fields_ = [("key", C.c_uint16), ("typecode", C.c_uint8), ("cardinality", C.c_int32), ("data", C.c_void_p)]


class Meta(C.Structure):
    _fields_ = [("n_containers", C.c_uint32), ("n_bitmap_containers", C.c_uint32),
                ("n_array_containers", C.c_uint32), ("n_run_containers", C.c_uint32),
                ("universe_size", C.c_uint32), ("total_bytes", C.c_size_t)]


class PagedCache(C.Structure):
    """cr_paged_cache (include/cu_roaring_abi.h)."""
    _fields_ = [("k", C.c_void_p), ("v", C.c_void_p)] + [
        (x, C.c_uint64) for x in ("k_page_stride", "k_slot_stride", "k_head_stride", "v_page_stride", "v_slot_stride",
                                  "v_head_stride")] + [
        (x, C.c_uint32) for x in ("n_pages", "page_size", "n_heads", "head_dim", "dtype")]


class PagedAttentionArgs(C.Structure):
    """cr_paged_attention_args (include/cu_roaring_abi.h)."""
    _fields_ = [("q", C.c_void_p), ("q_token_stride", C.c_uint64), ("q_head_stride", C.c_uint64),
                ("out", C.c_void_p), ("out_token_stride", C.c_uint64), ("out_head_stride", C.c_uint64),
                ("lse", C.c_void_p), ("n_tokens", C.c_uint32), ("n_heads", C.c_uint32), ("n_requests", C.c_uint32),
                ("d_starts", C.c_void_p), ("d_kv_len", C.c_void_p), ("d_table", C.c_void_p),
                ("table_cols", C.c_uint32), ("table_stride", C.c_uint64), ("d_sel", C.c_void_p),
                ("sel_stride", C.c_uint64), ("d_sel_len", C.c_void_p), ("d_limits", C.c_void_p),
                ("scale", C.c_float), ("causal", C.c_uint32), ("max_new", C.c_uint32), ("max_kv", C.c_uint32)]


class PagedRotaryArgs(C.Structure):
    """cr_paged_rotary_args (include/cu_roaring_abi.h)."""
    _fields_ = [("q", C.c_void_p), ("q_token_stride", C.c_uint64), ("q_head_stride", C.c_uint64),
                ("q_out", C.c_void_p), ("out_token_stride", C.c_uint64), ("out_head_stride", C.c_uint64),
                ("k", C.c_void_p), ("k_token_stride", C.c_uint64), ("k_head_stride", C.c_uint64),
                ("v", C.c_void_p), ("v_token_stride", C.c_uint64), ("v_head_stride", C.c_uint64),
                ("d_positions", C.c_void_p), ("d_freqs", C.c_void_p), ("d_slots", C.c_void_p),
                ("n_tokens", C.c_uint32), ("n_heads", C.c_uint32), ("rotated", C.c_uint32),
                ("interleaved", C.c_uint32), ("magnitude", C.c_float)]


class PagedWeightsArgs(C.Structure):
    """cr_paged_weights_args (include/cu_roaring_abi.h)."""
    _fields_ = [("q", C.c_void_p), ("q_token_stride", C.c_uint64), ("q_head_stride", C.c_uint64), ("lse", C.c_void_p),
                ("n_tokens", C.c_uint32), ("n_heads", C.c_uint32), ("n_requests", C.c_uint32),
                ("d_starts", C.c_void_p), ("d_new", C.c_void_p), ("d_kv_len", C.c_void_p), ("d_table", C.c_void_p),
                ("table_cols", C.c_uint32), ("table_stride", C.c_uint64), ("visible", C.c_void_p),
                ("d_past", C.c_void_p), ("past_stride", C.c_uint64), ("d_out", C.c_void_p), ("out_stride", C.c_uint64),
                ("scale", C.c_float), ("decay", C.c_float), ("causal", C.c_uint32), ("continued", C.c_uint32),
                ("max_new", C.c_uint32), ("max_kv", C.c_uint32)]


class PagedEvictArgs(C.Structure):
    """cr_paged_evict_args (include/cu_roaring_abi.h)."""
    _fields_ = [("d_weights", C.c_void_p), ("weights_stride", C.c_uint64), ("d_positions", C.c_void_p),
                ("positions_stride", C.c_uint64), ("d_kept", C.c_void_p), ("d_seen", C.c_void_p),
                ("d_kv_len", C.c_void_p), ("d_keep", C.c_void_p), ("d_table", C.c_void_p), ("table_cols", C.c_uint32),
                ("table_stride", C.c_uint64), ("page_size", C.c_uint32), ("n_pages", C.c_uint32),
                ("n_requests", C.c_uint32), ("sinks", C.c_uint32), ("recent", C.c_uint32), ("pinned", C.c_void_p),
                ("d_weights_out", C.c_void_p), ("weights_out_stride", C.c_uint64), ("d_positions_out", C.c_void_p),
                ("positions_out_stride", C.c_uint64), ("d_len", C.c_void_p), ("d_moves", C.c_void_p),
                ("moves_cap", C.c_uint32), ("moves_stride", C.c_uint64), ("d_n_moves", C.c_void_p),
                ("d_freed", C.c_void_p), ("freed_cap", C.c_uint32), ("d_counts", C.c_void_p)]


class DraftVerifyArgs(C.Structure):
    """cr_draft_verify_args (include/cu_roaring_abi.h)."""
    _fields_ = [("d_scores", C.c_void_p), ("row_stride", C.c_uint64), ("d_draft", C.c_void_p),
                ("draft_row_stride", C.c_uint64), ("dtype", C.c_uint32), ("n_rows", C.c_uint32),
                ("n_requests", C.c_uint32), ("vocab", C.c_uint32), ("d_tokens", C.c_void_p), ("d_starts", C.c_void_p),
                ("d_uniform", C.c_void_p), ("allowed", C.c_void_p), ("d_allowed_bits", C.c_void_p),
                ("bits_stride", C.c_uint64), ("temperature", C.c_float), ("d_accepted", C.c_void_p),
                ("d_out", C.c_void_p), ("out_cols", C.c_uint32), ("out_stride", C.c_uint64)]


assert C.sizeof(GpuRoaring) == 120 and C.sizeof(GpuRoaringView) == 80

_lib = None


class CrError(RuntimeError):
    def __init__(self, code: int, msg: str):
        super().__init__(f"[{code}] {msg}")
        self.code = code


def load(path: Optional[str] = None):
    """Load the HIP library; raises if it has not been built."""
    global _lib
    if _lib is not None:
        return _lib
    p = path or LIB_PATH
    if not os.path.exists(p):
        raise RuntimeError(f"libcuroaring_amd.so not built at {p}: run `make -C cu-roaring-bitmap_amd` "
                           f"(or __graft_entry__.build())")
    L = C.CDLL(p)
    P = C.POINTER
    L.cr_last_error.restype = C.c_char_p
    sigs = {
        "cr_upload_from_ids": [C.c_void_p, C.c_uint32, C.c_uint32, C.c_void_p, C.c_uint32, P(GpuRoaring)],
        "cr_upload_from_device_ids": [C.c_void_p, C.c_uint32, C.c_uint32, C.c_void_p, C.c_uint32, P(GpuRoaring)],
        "cr_upload_from_bitset": [C.c_void_p, C.c_uint32, C.c_uint32, C.c_void_p, P(GpuRoaring)],
        "cr_upload_from_device_bitset": [C.c_void_p, C.c_uint32, C.c_uint32, C.c_void_p, P(GpuRoaring)],
        "cr_upload_containers": [C.c_void_p, C.c_uint32, C.c_uint32, C.c_bool, C.c_uint64, C.c_void_p, C.c_uint32,
                                 P(GpuRoaring)],
        "cr_get_meta": [C.c_void_p, C.c_uint32, P(Meta)],
        "cr_set_operation": [P(GpuRoaring), P(GpuRoaring), C.c_uint32, C.c_void_p, P(GpuRoaring)],
        "cr_multi_and": [C.c_void_p, C.c_uint32, C.c_void_p, P(GpuRoaring)],
        "cr_free": [P(GpuRoaring)],
        "cr_free_async": [P(GpuRoaring), C.c_void_p],
        "cr_resolve_auto_threshold": [C.c_uint32, C.c_int, P(C.c_uint32)],
        "cr_make_view": [P(GpuRoaring), P(GpuRoaringView)],
        "cr_contains_batch": [P(GpuRoaringView), C.c_void_p, C.c_uint64, C.c_void_p, C.c_uint32, C.c_void_p],
        "cr_topk_set_small_limit": [C.c_uint32],
        "cr_topk_filtered": [C.c_void_p, C.c_uint64, C.c_void_p, C.c_uint32, C.c_uint32, P(GpuRoaring), C.c_uint32,
                             C.c_void_p, C.c_void_p, C.c_void_p],
        "cr_device_l2_bytes": [C.c_int, P(C.c_uint64)],
        "cr_device_malloc": [P(C.c_void_p), C.c_size_t],
        "cr_device_free": [C.c_void_p],
        "cr_memcpy_h2d": [C.c_void_p, C.c_void_p, C.c_size_t],
        "cr_memcpy_d2h": [C.c_void_p, C.c_void_p, C.c_size_t],
        "cr_stream_synchronize": [C.c_void_p],
        "cr_timing_enable": [C.c_int],
        "cr_mempool_trim": [C.c_int, C.c_size_t],
        "cr_timing_report": [C.c_char_p, C.c_size_t],
        "cr_decompress_to_bitset": [P(GpuRoaring), C.c_void_p, C.c_uint32, C.c_void_p],
        "cr_decompress_to_bitset_alloc": [P(GpuRoaring), C.c_void_p, P(C.c_void_p), P(C.c_uint32)],
        "cr_enumerate_ids": [P(GpuRoaring), C.c_void_p, C.c_uint64, C.c_void_p],
        "cr_enumerate_ids_alloc": [P(GpuRoaring), C.c_void_p, P(C.c_void_p), P(C.c_uint64)],
        "cr_enumerate_ids_noalloc": [P(GpuRoaring), C.c_void_p, C.c_uint64, C.c_void_p],
        "cr_cardinality": [P(GpuRoaring), C.c_void_p, P(C.c_uint64)],
        "cr_promote_to_bitmap": [P(GpuRoaring), C.c_void_p, P(GpuRoaring)],
        "cr_promote_auto": [P(GpuRoaring), C.c_void_p, C.c_int, P(GpuRoaring)],
        "cr_deep_copy": [P(GpuRoaring), C.c_void_p, P(GpuRoaring)],
        "cr_portable_size_in_bytes": [P(GpuRoaring), C.c_void_p, P(C.c_size_t)],
        "cr_portable_serialize": [P(GpuRoaring), C.c_void_p, C.c_void_p, C.c_size_t, P(C.c_size_t)],
        "cr_portable_deserialize": [C.c_void_p, C.c_size_t, C.c_uint32, C.c_void_p, C.c_uint32, P(GpuRoaring)],
        "cr_upload_batch": [C.c_void_p, C.c_void_p, C.c_uint32, C.c_void_p, P(RoaringBatch)],
        "cr_free_batch": [P(RoaringBatch)],
        "cr_promote_batch": [P(RoaringBatch), C.c_void_p, P(RoaringBatch)],
        "cr_batch_make_view": [P(RoaringBatch), C.c_uint32, P(BatchView)],
        "cr_batch_multi_and": [P(RoaringBatch), C.c_void_p, C.c_uint32, C.c_void_p, P(RoaringBatch)],
        "cr_batch_decompress": [P(RoaringBatch), C.c_void_p, C.c_uint64, C.c_void_p],
        "cr_batch_contains": [P(RoaringBatch), C.c_void_p, C.c_uint32, C.c_void_p, C.c_uint64, C.c_void_p, C.c_void_p],
        "cr_batch_view_contains": [P(BatchView), C.c_void_p, C.c_uint64, C.c_void_p, C.c_void_p],
        "cr_debug_fail_device_allocs": [C.c_uint32, C.c_uint32],
        "cr_paged_plan": [P(GpuRoaring), C.c_uint32, C.c_uint32, C.c_void_p, C.c_void_p, C.c_uint32, C.c_void_p,
                          C.c_uint32, C.c_uint64, C.c_void_p, C.c_uint32, C.c_void_p, C.c_void_p, C.c_void_p,
                          C.c_uint32, C.c_void_p, C.c_void_p],
        "cr_paged_append": [C.c_void_p, C.c_void_p, C.c_uint64, C.c_uint64, C.c_uint64, C.c_uint64, C.c_uint32,
                            C.c_void_p, C.c_void_p, C.c_void_p],
        "cr_paged_select": [P(GpuRoaring), C.c_uint32, C.c_uint32, C.c_void_p, C.c_uint32, C.c_uint64, C.c_void_p,
                            C.c_void_p, C.c_uint32, C.c_uint32, C.c_void_p, C.c_uint64, C.c_void_p, C.c_void_p,
                            C.c_void_p],
        "cr_paged_attention": [C.c_void_p, C.c_void_p, C.c_void_p],
        "cr_paged_rotary": [C.c_void_p, C.c_void_p, C.c_void_p],
        "cr_paged_weights": [C.c_void_p, C.c_void_p, C.c_void_p],
        "cr_paged_evict": [C.c_void_p, C.c_void_p],
        "cr_paged_move": [C.c_void_p, C.c_uint32, C.c_uint64, C.c_void_p, C.c_uint32, C.c_void_p, C.c_void_p],
        "cr_draft_verify": [C.c_void_p, C.c_void_p],
        "cr_beam_select": [C.c_void_p, C.c_uint32, C.c_uint32, C.c_uint32, C.c_uint32, C.c_uint64, C.c_uint64,
                           C.c_void_p, C.c_void_p, P(GpuRoaring), C.c_void_p, C.c_uint64, C.c_uint32, C.c_void_p,
                           C.c_void_p, C.c_void_p, C.c_void_p],
        "cr_beam_reorder": [C.c_void_p, C.c_void_p, C.c_uint32, C.c_uint32, C.c_uint32, C.c_uint64, C.c_uint64,
                            C.c_uint64, C.c_void_p, C.c_uint64, C.c_void_p, C.c_void_p],
    }
    for name, args in sigs.items():
        f = getattr(L, name)
        f.argtypes = args
        f.restype = C.c_int
    L.cr_topk_set_small_limit.restype = C.c_uint32
    _lib = L
    return L


def _check(rc: int, what: str):
    if rc != CR_OK:
        raise CrError(rc, f"{what}: {_lib.cr_last_error().decode(errors='replace')}")


def _stream(stream) -> Optional[int]:
    if stream is None:
        return None
    if isinstance(stream, int):
        return stream
    return stream.cuda_stream  # torch.cuda.Stream


def _dptr(t) -> int:
    return t.data_ptr()


# ---- uploads ---------------------------------------------------------------
def upload_from_ids(ids, universe: int, threshold: int = PROMOTE_AUTO, stream=None) -> GpuRoaring:
    ids = np.ascontiguousarray(ids, dtype=np.uint32)
    out = GpuRoaring()
    _check(load().cr_upload_from_ids(ids.ctypes.data if ids.size else None, ids.size, universe, _stream(stream),
                                     threshold, C.byref(out)), "upload_from_ids")
    return out


def upload_from_device_ids(d_ids, universe: int, threshold: int = PROMOTE_AUTO, stream=None) -> GpuRoaring:
    """d_ids: a torch int32/uint32 CUDA tensor (read as uint32)."""
    out = GpuRoaring()
    n = d_ids.numel()
    _check(load().cr_upload_from_device_ids(_dptr(d_ids) if n else None, n, universe, _stream(stream), threshold,
                                            C.byref(out)), "upload_from_device_ids")
    return out


def upload_from_bitset(words, universe: int, stream=None) -> GpuRoaring:
    words = np.ascontiguousarray(words, dtype=np.uint32)
    out = GpuRoaring()
    _check(load().cr_upload_from_bitset(words.ctypes.data if words.size else None, words.size, universe,
                                        _stream(stream), C.byref(out)), "upload_from_bitset")
    return out


def upload_from_device_bitset(d_words, universe: int, stream=None) -> GpuRoaring:
    out = GpuRoaring()
    n = d_words.numel()
    _check(load().cr_upload_from_device_bitset(_dptr(d_words) if n else None, n, universe, _stream(stream),
                                               C.byref(out)), "upload_from_device_bitset")
    return out


def _container_array(containers):
    arr = (HostContainer * max(1, len(containers)))()
    keep = []
    for i, (key, tc, card, payload) in enumerate(containers):
        p = np.ascontiguousarray(payload)
        keep.append(p)
        arr[i] = HostContainer(key, tc, card, p.ctypes.data if p.size else None)
    return arr, keep


def upload_containers(containers, universe: int = 0, complemented: bool = False, logical_cardinality: int = 0,
                      threshold: int = PROMOTE_AUTO, stream=None) -> GpuRoaring:
    """containers: [(key, typecode, cardinality|n_runs, payload ndarray)] sorted by key."""
    arr, keep = _container_array(containers)
    out = GpuRoaring()
    _check(load().cr_upload_containers(arr, len(containers), universe, complemented, logical_cardinality,
                                       _stream(stream), threshold, C.byref(out)), "upload_containers")
    del keep
    return out


def get_meta(containers) -> Meta:
    arr, keep = _container_array(containers)
    m = Meta()
    _check(load().cr_get_meta(arr, len(containers), C.byref(m)), "get_meta")
    return m


# ---- set operations ----------------------------------------------------------
def set_operation(a: GpuRoaring, b: GpuRoaring, op: int, stream=None) -> GpuRoaring:
    out = GpuRoaring()
    _check(load().cr_set_operation(C.byref(a), C.byref(b), op, _stream(stream), C.byref(out)), "set_operation")
    return out


def multi_and(bitmaps: Sequence[GpuRoaring], stream=None) -> GpuRoaring:
    arr = (GpuRoaring * max(1, len(bitmaps)))()
    for i, b in enumerate(bitmaps):
        arr[i] = b
    out = GpuRoaring()
    _check(load().cr_multi_and(arr, len(bitmaps), _stream(stream), C.byref(out)), "multi_and")
    return out


def free(g: GpuRoaring):
    _check(load().cr_free(C.byref(g)), "free")


def free_async(g: GpuRoaring, stream=None):
    _check(load().cr_free_async(C.byref(g), _stream(stream)), "free_async")


def resolve_auto_threshold(universe: int, device: int = -1) -> int:
    t = C.c_uint32()
    _check(load().cr_resolve_auto_threshold(universe, device, C.byref(t)), "resolve_auto_threshold")
    return t.value


def device_l2_bytes(device: int = -1) -> int:
    v = C.c_uint64()
    _check(load().cr_device_l2_bytes(device, C.byref(v)), "device_l2_bytes")
    return v.value


def make_view(g: GpuRoaring) -> GpuRoaringView:
    v = GpuRoaringView()
    _check(load().cr_make_view(C.byref(g), C.byref(v)), "make_view")
    return v


def contains_batch(g: GpuRoaring, d_ids, d_out, mode: int = QUERY_CONTAINS, stream=None):
    """d_ids / d_out: CUDA tensors of n uint32 (int32 storage); asynchronous."""
    v = make_view(g)
    n = d_ids.numel()
    _check(load().cr_contains_batch(C.byref(v), _dptr(d_ids), n, _dptr(d_out), mode, _stream(stream)),
           "contains_batch")


def topk_set_small_limit(rows: int) -> int:
    """Rows at or below which the top-k may keep every estimate and select per
    query (it does so up to 65536 rows at most, so larger limits, recorded up to
    262144, are alike; 0 turns the estimates off: sorted lists answer).  Returns
    the previous limit."""
    return int(load().cr_topk_set_small_limit(rows))


def topk_filtered(d_base, d_queries, k: int, filt: Optional[GpuRoaring], d_dist, d_ids, stream=None):
    n_base, dim = d_base.shape
    nq = d_queries.shape[0]
    _check(load().cr_topk_filtered(_dptr(d_base), n_base, _dptr(d_queries), nq, dim,
                                   C.byref(filt) if filt is not None else None, k, _dptr(d_dist), _dptr(d_ids),
                                   _stream(stream)), "topk_filtered")


# ---- conversions (stream-ordered, no synchronisation) -------------------------
NO_BOUND = 0xFFFFFFFFFFFFFFFF


def decompress_to_bitset(g: GpuRoaring, d_out, n_words: Optional[int] = None, stream=None):
    """decompress_to_bitset into d_out (a CUDA tensor of >= n_words 32-bit words)."""
    if n_words is None:
        n_words = d_out.numel()
    _check(load().cr_decompress_to_bitset(C.byref(g), _dptr(d_out), n_words, _stream(stream)),
           "decompress_to_bitset")


def decompress_to_bitset_alloc(g: GpuRoaring, stream=None):
    """The allocating overload: (device pointer or None, n_words); free with device_free."""
    p, n = C.c_void_p(), C.c_uint32()
    _check(load().cr_decompress_to_bitset_alloc(C.byref(g), _stream(stream), C.byref(p), C.byref(n)),
           "decompress_to_bitset_alloc")
    return p.value, n.value


def enumerate_ids(g: GpuRoaring, d_out, capacity: int = NO_BOUND, stream=None):
    """enumerate_ids into d_out (a CUDA int64 tensor)."""
    _check(load().cr_enumerate_ids(C.byref(g), _dptr(d_out), capacity, _stream(stream)), "enumerate_ids")


def cardinality(g: GpuRoaring, stream=None) -> int:
    """The logical cardinality counted on the device (set-operation results included)."""
    n = C.c_uint64()
    _check(load().cr_cardinality(C.byref(g), _stream(stream), C.byref(n)), "cardinality")
    return n.value


def enumerate_ids_noalloc(g: GpuRoaring, d_out, capacity: int = NO_BOUND, stream=None):
    """enumerate_ids into d_out with no device allocation (the library's fixed per-device scratch)."""
    _check(load().cr_enumerate_ids_noalloc(C.byref(g), _dptr(d_out), capacity, _stream(stream)),
           "enumerate_ids_noalloc")


def enumerate_ids_alloc(g: GpuRoaring, stream=None):
    """The allocating overload: (device pointer or None, n_ids); free with device_free."""
    p, n = C.c_void_p(), C.c_uint64()
    _check(load().cr_enumerate_ids_alloc(C.byref(g), _stream(stream), C.byref(p), C.byref(n)), "enumerate_ids_alloc")
    return p.value, n.value


def promote_to_bitmap(g: GpuRoaring, stream=None) -> GpuRoaring:
    out = GpuRoaring()
    _check(load().cr_promote_to_bitmap(C.byref(g), _stream(stream), C.byref(out)), "promote_to_bitmap")
    return out


def promote_auto(g: GpuRoaring, stream=None, device: int = -1) -> GpuRoaring:
    out = GpuRoaring()
    _check(load().cr_promote_auto(C.byref(g), _stream(stream), device, C.byref(out)), "promote_auto")
    return out


def deep_copy(g: GpuRoaring, stream=None) -> GpuRoaring:
    out = GpuRoaring()
    _check(load().cr_deep_copy(C.byref(g), _stream(stream), C.byref(out)), "deep_copy")
    return out


# ---- Roaring portable format ------------------------------------------------------
def portable_size_in_bytes(g: GpuRoaring, stream=None) -> int:
    n = C.c_size_t()
    _check(load().cr_portable_size_in_bytes(C.byref(g), _stream(stream), C.byref(n)), "portable_size_in_bytes")
    return n.value


def portable_serialize(g: GpuRoaring, stream=None) -> bytes:
    """The logical set of g in the Roaring portable format."""
    n = portable_size_in_bytes(g, stream)
    buf = C.create_string_buffer(max(n, 1))
    w = C.c_size_t()
    _check(load().cr_portable_serialize(C.byref(g), _stream(stream), buf, n, C.byref(w)), "portable_serialize")
    return buf.raw[:w.value]


def portable_deserialize(data: bytes, universe: int = 0, threshold: int = PROMOTE_AUTO, stream=None) -> GpuRoaring:
    """upload() of a portable-format bitmap (universe 0: upload(bm); else upload(bm, U))."""
    out = GpuRoaring()
    buf = C.create_string_buffer(bytes(data), max(len(data), 1))
    _check(load().cr_portable_deserialize(buf, len(data), universe, _stream(stream), threshold, C.byref(out)),
           "portable_deserialize")
    return out


# ---- the batch API (the reference's v2) -------------------------------------------
def upload_batch(bitmaps, stream=None) -> RoaringBatch:
    """bitmaps: a list of container lists, each [(key, typecode, card, ndarray)]."""
    arrays = [_container_array(c) for c in bitmaps]
    ptrs = (C.c_void_p * max(1, len(bitmaps)))(*[C.addressof(a[0]) if len(a[0]) else None for a in arrays])
    counts = (C.c_uint32 * max(1, len(bitmaps)))(*[len(c) for c in bitmaps])
    out = RoaringBatch()
    _check(load().cr_upload_batch(ptrs, counts, len(bitmaps), _stream(stream), C.byref(out)), "upload_batch")
    return out


def free_batch(b: RoaringBatch):
    _check(load().cr_free_batch(C.byref(b)), "free_batch")


def promote_batch(b: RoaringBatch, stream=None) -> RoaringBatch:
    out = RoaringBatch()
    _check(load().cr_promote_batch(C.byref(b), _stream(stream), C.byref(out)), "promote_batch")
    return out


def batch_make_view(b: RoaringBatch, idx: int) -> BatchView:
    v = BatchView()
    _check(load().cr_batch_make_view(C.byref(b), idx, C.byref(v)), "make_view")
    return v


def batch_multi_and(b: RoaringBatch, indices, stream=None) -> RoaringBatch:
    idx = np.ascontiguousarray(indices, dtype=np.uint32)
    out = RoaringBatch()
    _check(load().cr_batch_multi_and(C.byref(b), idx.ctypes.data if idx.size else None, idx.size, _stream(stream),
                                     C.byref(out)), "multi_and")
    return out


def batch_decompress(b: RoaringBatch, d_bitsets, words_each: int, stream=None):
    _check(load().cr_batch_decompress(C.byref(b), _dptr(d_bitsets), words_each, _stream(stream)), "decompress_batch")


def batch_contains(b: RoaringBatch, d_ids, d_out, bitmap: int = 0, d_bitmap_idx=None, stream=None):
    """d_out[i] = bitmap (d_bitmap_idx[i] or `bitmap`) holds d_ids[i]; d_out is a uint8 CUDA tensor."""
    _check(load().cr_batch_contains(C.byref(b), _dptr(d_bitmap_idx) if d_bitmap_idx is not None else None, bitmap,
                                    _dptr(d_ids), d_ids.numel(), _dptr(d_out), _stream(stream)), "batch_contains")


def batch_view_contains(v: BatchView, d_ids, d_out, stream=None):
    _check(load().cr_batch_view_contains(C.byref(v), _dptr(d_ids), d_ids.numel(), _dptr(d_out), _stream(stream)),
           "batch_view_contains")


def download_batch(b: RoaringBatch) -> SimpleNamespace:
    """Host copy of a batch (same fields as the oracle's HostBatch); the
    metadata arrays hold the batch's live slices only."""
    n, T = b.n_bitmaps, b.total_containers
    h = lambda p, k: np.ctypeslib.as_array(p, shape=(k,)).copy() if (k and p) else np.zeros(0)
    hcs = h(b.host_container_starts, n + 1).astype(np.uint32) if n else np.zeros(0, np.uint32)
    hks = h(b.host_key_index_starts, n + 1).astype(np.uint32) if n else np.zeros(0, np.uint32)
    kidx = int(hks[-1]) if n else 0
    return SimpleNamespace(
        n_bitmaps=n, total_containers=T, n_bitmap_containers_total=b.n_bitmap_containers_total,
        array_pool_bytes=b.array_pool_bytes, run_pool_bytes=b.run_pool_bytes,
        container_starts=_d2h(b.container_starts, n + 1 if n else 0, np.uint32),
        key_index_starts=_d2h(b.key_index_starts, n + 1 if n else 0, np.uint32),
        keys=_d2h(b.keys, T, np.uint16), types=_d2h(b.types, T, np.uint8), offsets=_d2h(b.offsets, T, np.uint32),
        cards=_d2h(b.cardinalities, T, np.uint16), key_indices=_d2h(b.key_indices, kidx, np.uint16),
        bitmap_data=_d2h(b.bitmap_data, b.n_bitmap_containers_total * 1024, np.uint64),
        array_data=_d2h(b.array_data, b.array_pool_bytes // 2, np.uint16),
        run_data=_d2h(b.run_data, b.run_pool_bytes // 2, np.uint16),
        host_total_cardinalities=h(b.host_total_cardinalities, n).astype(np.uint64) if n else np.zeros(0, np.uint64),
        host_universe_sizes=h(b.host_universe_sizes, n).astype(np.uint32) if n else np.zeros(0, np.uint32),
        host_container_starts=hcs, host_key_index_starts=hks,
        host_n_bitmap_containers=h(b.host_n_bitmap_containers, n).astype(np.uint32) if n else np.zeros(0, np.uint32),
    )


# ---- serving language models (stream-ordered, no synchronisation) ---------------
# As in all calls here, stream=None is the null stream, also inside torch.cuda.stream(s), where the tensors' own
# producers run on s: pass stream=torch.cuda.current_stream() there.  Tensors lie on the current device.
F32, F16, BF16 = 0, 1, 2
_TYPES = {"float32": F32, "float16": F16, "bfloat16": BF16}
_names, _codes = {}, {}
# The structs as the calls pass them: packed bytes cost a third of a filled ctypes structure.
_CACHE = struct.Struct("@PPQQQQQQIIIII4x")
_ATTENTION = struct.Struct("@PQQPQQPIIIPPPIQPQPPfIII")
_ROTARY = struct.Struct("@PQQPQQPQQPQQPPPIIIIf4x")
_WEIGHTS = struct.Struct("@PQQPIIIPPPPIQPPQPQffIIII")
_EVICT = struct.Struct("@PQPQPPPPPIQIIIIIPPQPQPPIQPPIP")
_VERIFY = struct.Struct("@PQPQIIIIPPPPPQfPPIQ")
assert _CACHE.size == C.sizeof(PagedCache) and _ATTENTION.size == C.sizeof(PagedAttentionArgs)
assert _ROTARY.size == C.sizeof(PagedRotaryArgs) and _WEIGHTS.size == C.sizeof(PagedWeightsArgs)
assert _EVICT.size == C.sizeof(PagedEvictArgs) and _VERIFY.size == C.sizeof(DraftVerifyArgs)


_devices = None


def _device() -> int:
    """The number of the current device, on which the calls below run, and their tensors have to be: -2 without one."""
    global _devices
    if _devices is None or _devices > 1:
        import torch
        _devices = torch.cuda.device_count()
        if _devices > 1:
            return torch.cuda.current_device()
    return 0 if _devices else -2


def _type_name(t) -> str:
    name = _names.get(t.dtype)
    if name is None:
        name = _names[t.dtype] = str(t.dtype).split(".")[-1]
    return name


def _typed(t) -> int:
    """The library's code of a tensor's type."""
    code = _codes.get(t.dtype)
    if code is None:
        code = _TYPES.get(_type_name(t))
        if code is None:
            raise CrError(CR_ERR_INVALID, f"a tensor of {t.dtype} where one of {', '.join(_TYPES)} is taken")
        _codes[t.dtype] = code
    return code


def _array(t, name: str, dtype: str, shape, device: int) -> int:
    """The address of a contiguous tensor of this type and shape (0: one axis of any extent) on this device."""
    if (_names.get(t.dtype) or _type_name(t)) == dtype and t.get_device() == device and t.is_contiguous() and (
            t.dim() == 1 if shape == 0 else t.shape == shape):
        return t.data_ptr()
    raise CrError(CR_ERR_INVALID, f"{name}: a contiguous {dtype} tensor of shape "
                                  f"{'(any,)' if shape == 0 else tuple(shape)} on the current CUDA device is taken, not "
                                  f"{t.dtype} {tuple(t.shape)} on {t.device}")


def _table(t, n_requests: int, device: int):
    """(address, columns, row stride) of a block table, rows of which may lie apart."""
    if _type_name(t) == "int32" and t.get_device() == device and t.dim() == 2:
        (rows, cols), (stride, one) = t.shape, t.stride()
        if rows <= 1:  # whose stride may be any number
            stride = cols
        if rows == n_requests and (one == 1 or cols <= 1) and stride >= cols:
            return t.data_ptr(), cols, stride
    raise CrError(CR_ERR_INVALID, f"block table: an int32 tensor of {n_requests} rows on the current CUDA device is "
                                  f"taken, not {t.dtype} {tuple(t.shape)} on {t.device}")


def _matrix(t, name: str, dtype: str, n_rows: int, cols: int, device: int):
    """(address, row stride) of a tensor of n_rows rows of at least `cols` values, which may lie apart."""
    if (_names.get(t.dtype) or _type_name(t)) == dtype and t.get_device() == device and t.dim() == 2:
        (rows, held), (stride, one) = t.shape, t.stride()
        if rows <= 1:  # whose stride may be any number
            stride = held
        if rows == n_rows and held >= cols and (one == 1 or held <= 1) and stride >= held:
            return t.data_ptr(), stride
    raise CrError(CR_ERR_INVALID, f"{name}: a {dtype} tensor of {n_rows} rows of at least {cols} values on the current "
                                  f"CUDA device is taken, not {t.dtype} {tuple(t.shape)} on {t.device}")


def _rows(t, name: str, dtype, shape, device: int):
    """(address, token stride, head stride) of a [tokens, heads, dim] tensor of this type and shape."""
    if t.dtype == dtype and t.get_device() == device and t.shape == shape:
        token, head, one = t.stride()
        if one == 1 or shape[2] <= 1:
            return t.data_ptr(), token, head
    raise CrError(CR_ERR_INVALID, f"{name}: a {dtype} tensor of shape {tuple(shape)} with contiguous rows on the "
                                  f"current CUDA device is taken, not {t.dtype} {tuple(t.shape)} on {t.device}")


def _cache(d_k, d_v, device: int):
    """(cr_paged_cache, page size, heads, dim) of a cache's tensors."""
    shape = d_k.shape
    if len(shape) == 4 and d_v.shape == shape and d_k.dtype == d_v.dtype and d_k.get_device() == device == d_v.get_device():
        (kp, ks, kh, k1), (vp, vs, vh, v1) = d_k.stride(), d_v.stride()
        pages, size, heads, dim = shape
        if (k1 == 1 and v1 == 1) or dim <= 1:
            return _CACHE.pack(d_k.data_ptr(), d_v.data_ptr(), kp, ks, kh, vp, vs, vh, pages, size, heads, dim,
                               _typed(d_k)), size, heads, dim
    raise CrError(CR_ERR_INVALID, "cache: keys and values of one type and shape [pages, page size, heads, dim] with "
                                  "contiguous rows on the current CUDA device are taken")


def paged_cache(d_k, d_v) -> PagedCache:
    """A cache of [pages, page size, heads, dim] keys and values (any strides with contiguous rows)."""
    return PagedCache.from_buffer_copy(_cache(d_k, d_v, _device())[0])


def paged_plan(free_pages: GpuRoaring, n_pages: int, page_size: int, d_cached, d_new, d_table, d_slots, d_starts,
               d_kv_len, d_taken, d_counts, stream=None):
    """Block tables and slot maps from the requests' lengths (cr_paged_plan).

    d_cached, d_new: int32 [R], tokens in the cache and new ones.  d_table: int32 [R, cols], completed in place with
    pages from `free_pages`.  Written: d_slots int64 [at least the new tokens], d_starts int32 [R + 1], d_kv_len
    int32 [R], d_taken int32 [any], d_counts int32 [3]: new tokens, pages taken, pages missing.  stream: None is the
    null stream."""
    n, on = d_cached.numel(), _device()
    table, cols, stride = _table(d_table, n, on)
    _check(load().cr_paged_plan(C.byref(free_pages), n_pages, page_size, _array(d_cached, "cached", "int32", (n,), on),
                                _array(d_new, "new", "int32", (n,), on), n, table, cols, stride,
                                _array(d_slots, "slots", "int64", 0, on), d_slots.numel(),
                                _array(d_starts, "starts", "int32", (n + 1,), on),
                                _array(d_kv_len, "kv_len", "int32", (n,), on),
                                _array(d_taken, "taken", "int32", 0, on), d_taken.numel(),
                                _array(d_counts, "counts", "int32", (3,), on), _stream(stream)), "paged_plan")


def paged_append(d_k, d_v, d_slots, d_k_cache, d_v_cache, stream=None):
    """New keys and values [T, heads, dim] into slots int64 [T] of the cache; slots outside it (-1) are left out.

    stream: None is the null stream."""
    on = _device()
    cache, _, heads, dim = _cache(d_k_cache, d_v_cache, on)
    n, dtype = d_slots.numel(), d_k_cache.dtype
    shape = (n, heads, dim)
    k, k_token, k_head = _rows(d_k, "k", dtype, shape, on)
    v, v_token, v_head = _rows(d_v, "v", dtype, shape, on)
    _check(load().cr_paged_append(k, v, k_token, k_head, v_token, v_head, n,
                                  _array(d_slots, "slots", "int64", (n,), on), cache, _stream(stream)), "paged_append")


def paged_select(visible: GpuRoaring, d_table, d_starts, d_kv_len, page_size: int, d_sel, d_sel_len, d_limits,
                 n_pages: Optional[int] = None, stream=None):
    """The slots of each request that the bitmap `visible` holds, listed once for every layer's attention.

    Written: d_sel int32 [R, at least cols * page_size], d_sel_len int32 [R], d_limits int32 [T].  n_pages: the
    cache's (default: those that the bitmap's universe reaches into).  stream: None is the null stream."""
    n, on = d_kv_len.numel(), _device()
    table, cols, stride = _table(d_table, n, on)
    sel, room, sel_stride = _table(d_sel, n, on)
    if room < cols * page_size:
        raise CrError(CR_ERR_INVALID, f"paged_select: a row of sel holds cols * page_size = {cols * page_size} slots")
    if n_pages is None:
        n_pages = -(-visible.universe_size // page_size)
    _check(load().cr_paged_select(C.byref(visible), n_pages, page_size, table, cols, stride,
                                  _array(d_starts, "starts", "int32", (n + 1,), on),
                                  _array(d_kv_len, "kv_len", "int32", (n,), on), n, d_limits.numel(), sel, sel_stride,
                                  _array(d_sel_len, "sel_len", "int32", (n,), on),
                                  _array(d_limits, "limits", "int32", 0, on), _stream(stream)), "paged_select")


def paged_attention(d_q, d_k_cache, d_v_cache, d_table, d_starts, d_kv_len, d_out, scale: Optional[float] = None,
                    causal: bool = True, d_lse=None, selection=None, max_new: int = 0, max_kv: int = 0, stream=None):
    """Attention of the requests' new tokens q [T, heads, dim] over the paged cache into d_out (cr_paged_attention).

    Request r's tokens are [starts[r], starts[r + 1]), the last of its kv_len[r] positions.  scale: 1 / sqrt(dim) by
    default.  d_lse: float32 [T, heads] or None.  selection: paged_select's (sel, sel_len, limits) or None.  max_new
    and max_kv: the most new tokens and keys of a request if known; they choose how the work is split.  stream: None is
    the null stream."""
    on = _device()
    cache, page_size, _, dim = _cache(d_k_cache, d_v_cache, on)
    dtype, shape = d_k_cache.dtype, d_q.shape
    if len(shape) != 3 or d_q.dtype != dtype or shape[2] != dim:
        raise CrError(CR_ERR_INVALID, f"paged_attention: {dtype} queries [tokens, heads, {dim}] are taken, not "
                                      f"{d_q.dtype} {tuple(shape)}")
    n, (tokens, heads, _) = d_kv_len.numel(), shape
    q, q_token, q_head = _rows(d_q, "q", dtype, shape, on)
    out, out_token, out_head = _rows(d_out, "out", dtype, shape, on)
    table, cols, stride = _table(d_table, n, on)
    sel, room, sel_stride, sel_len, limits = 0, 0, 0, 0, 0
    if selection is not None:
        sel, room, sel_stride = _table(selection[0], n, on)
        if room < cols * page_size:
            raise CrError(CR_ERR_INVALID, "paged_attention: a row of sel holds cols * page_size slots")
        sel_len = _array(selection[1], "sel_len", "int32", (n,), on)
        limits = _array(selection[2], "limits", "int32", (tokens,), on)
    if not (0 <= max_new < 1 << 32 and 0 <= max_kv < 1 << 32):
        raise CrError(CR_ERR_INVALID, f"paged_attention: max_new {max_new}, max_kv {max_kv}")
    a = _ATTENTION.pack(q, q_token, q_head, out, out_token, out_head,
                        _array(d_lse, "lse", "float32", (tokens, heads), on) if d_lse is not None else 0,
                        tokens, heads, n, _array(d_starts, "starts", "int32", (n + 1,), on),
                        _array(d_kv_len, "kv_len", "int32", (n,), on), table, cols, stride, sel, sel_stride, sel_len,
                        limits, dim ** -0.5 if scale is None else scale, causal, max_new, max_kv)
    _check(load().cr_paged_attention(a, cache, _stream(stream)), "paged_attention")


def rotary_frequencies(rotated: int, base: float = 10000.0, scaling: Optional[str] = None, factor: float = 1.0,
                       original: int = 4096, fast: float = 32.0, slow: float = 1.0, device="cuda"):
    """(freqs, magnitude) of paged_rotary for `rotated` dimensions: base^(-2 i / rotated) radians a position.

    scaling, for contexts `factor` times as long: "linear" divides every frequency by it; "base" raises the base, so
    that the slowest pair is divided by it and the fastest stays; "parts" leaves the pairs that turn more than `fast`
    times over the `original` positions, divides those that turn fewer than `slow` times, passes over evenly in their
    turns between them, and lengthens the rows by a tenth of the factor's logarithm.  Worked out in 64 bits.  A model
    that was trained with other frequencies (passing over evenly in the pairs' numbers, say) brings its own table."""
    import torch
    if rotated < 0 or rotated % 2 or base <= 0 or factor <= 0 or scaling not in (None, "linear", "base", "parts") or (
            scaling == "parts" and not (fast > slow and original > 0)):
        raise CrError(CR_ERR_INVALID, f"rotary_frequencies: {rotated} dimensions, base {base}, scaling {scaling!r} by "
                                      f"{factor}")
    if scaling == "base" and rotated > 2:
        base = base * factor ** (rotated / (rotated - 2))
    freqs = base ** (-torch.arange(0, rotated, 2, dtype=torch.float64) / max(1, rotated))
    magnitude = 1.0
    if scaling == "linear":
        freqs = freqs / factor
    elif scaling == "parts":
        turns = original * freqs / (2 * np.pi)
        stays = ((turns - slow) / (fast - slow)).clamp(0, 1)
        freqs = freqs * (stays + (1 - stays) / factor)
        magnitude = max(1.0, 1.0 + 0.1 * float(np.log(factor)))
    return freqs.to(device), magnitude


def paged_rotary(d_k, d_v, d_positions, d_freqs, d_slots, d_k_cache, d_v_cache, d_q=None, d_q_out=None,
                 interleaved: bool = False, magnitude: float = 1.0, stream=None):
    """paged_append with keys, and queries d_q [T, heads, dim] into d_q_out, turned by their positions
    (cr_paged_rotary).

    d_positions: int32 [T].  d_freqs: float64 [rotated / 2], radians a position (rotary_frequencies makes them); the
    rows' first `rotated` dimensions are turned, in halves or, interleaved, in neighbouring pairs.  d_q_out: d_q itself
    by default.  stream: None is the null stream."""
    on = _device()
    cache, _, heads, dim = _cache(d_k_cache, d_v_cache, on)
    n, dtype = d_slots.numel(), d_k_cache.dtype
    q = q_token = q_head = out = out_token = out_head = n_heads = 0
    if d_q is not None:
        n_heads = d_q.shape[1] if d_q.dim() == 3 else 0
        q, q_token, q_head = _rows(d_q, "q", dtype, (n, n_heads, dim), on)
        out, out_token, out_head = (q, q_token, q_head) if d_q_out is None else _rows(d_q_out, "q_out", dtype,
                                                                                      (n, n_heads, dim), on)
    elif d_q_out is not None:
        raise CrError(CR_ERR_INVALID, "paged_rotary: q_out without q")
    shape = (n, heads, dim)
    k, k_token, k_head = _rows(d_k, "k", dtype, shape, on)
    v, v_token, v_head = _rows(d_v, "v", dtype, shape, on)
    a = _ROTARY.pack(q, q_token, q_head, out, out_token, out_head, k, k_token, k_head, v, v_token, v_head,
                     _array(d_positions, "positions", "int32", (n,), on), _array(d_freqs, "freqs", "float64", 0, on),
                     _array(d_slots, "slots", "int64", (n,), on), n, n_heads, 2 * d_freqs.numel(), interleaved, magnitude)
    _check(load().cr_paged_rotary(a, cache, _stream(stream)), "paged_rotary")


def paged_weights(d_q, d_k_cache, d_table, d_starts, d_kv_len, d_lse, d_out, d_past=None, decay: float = 1.0, d_new=None,
                  scale: Optional[float] = None, causal: bool = True, visible: Optional[GpuRoaring] = None,
                  continued: bool = False, max_new: int = 0, max_kv: int = 0, stream=None):
    """The attention weight that each cached token got from the rows q [T, heads, dim] (cr_paged_weights), summed over
    heads into d_out float32 [R, at least cols * page_size].

    d_lse: float32 [T, heads], what paged_attention left for the same rows and scale.  d_past (d_out itself, if need
    be): what the tokens older than these rows had, times decay; continued: what all had, times decay, as between the
    layers of a step whose weights are summed (decay 1 behind the first).  Rows of request r: [starts[r], starts[r + 1]), or
    new[r] of them from starts[r] where d_new int32 [R] is given (d_starts then has R or R + 1 entries): the last of its
    kv_len[r] positions.  visible: a bitmap of slots.  max_new and max_kv: the most rows and positions of a request if
    known; they choose how the work is split.  stream: None is the null stream."""
    on = _device()
    shape, (pages, page_size, kv_heads, dim) = d_q.shape, d_k_cache.shape
    if len(shape) != 3 or shape[2] != dim or d_q.dtype != d_k_cache.dtype:
        raise CrError(CR_ERR_INVALID, f"paged_weights: {d_k_cache.dtype} queries [tokens, heads, {dim}] are taken, not "
                                      f"{d_q.dtype} {tuple(shape)}")
    kp, ks, kh, one = d_k_cache.stride()
    if d_k_cache.get_device() != on or (one != 1 and dim > 1):
        raise CrError(CR_ERR_INVALID, "paged_weights: keys [pages, page size, heads, dim] with contiguous rows on the "
                                      "current CUDA device are taken")
    cache = _CACHE.pack(d_k_cache.data_ptr(), 0, kp, ks, kh, 0, 0, 0, pages, page_size, kv_heads, dim, _typed(d_k_cache))
    n, (tokens, heads, _) = d_kv_len.numel(), shape
    q, q_token, q_head = _rows(d_q, "q", d_q.dtype, shape, on)
    table, cols, stride = _table(d_table, n, on)
    out, out_stride = _matrix(d_out, "out", "float32", n, cols * page_size, on)
    past, past_stride = (0, 0) if d_past is None else _matrix(d_past, "past", "float32", n, cols * page_size, on)
    new = 0 if d_new is None else _array(d_new, "new", "int32", (n,), on)
    entries = n if d_new is not None and d_starts.numel() == n else n + 1
    if not (0 <= max_new < 1 << 32 and 0 <= max_kv < 1 << 32):
        raise CrError(CR_ERR_INVALID, f"paged_weights: max_new {max_new}, max_kv {max_kv}")
    a = _WEIGHTS.pack(q, q_token, q_head, _array(d_lse, "lse", "float32", (tokens, heads), on), tokens, heads, n,
                      _array(d_starts, "starts", "int32", (entries,), on), new,
                      _array(d_kv_len, "kv_len", "int32", (n,), on), table, cols, stride,
                      C.addressof(visible) if visible is not None else 0, past, past_stride, out, out_stride,
                      dim ** -0.5 if scale is None else scale, decay, causal, continued, max_new, max_kv)
    _check(load().cr_paged_weights(a, cache, _stream(stream)), "paged_weights")


def paged_evict(d_weights, d_kv_len, d_keep, d_table, page_size: int, d_weights_out, d_len, d_moves, d_n_moves, d_freed,
                d_counts, d_positions=None, d_kept=None, d_seen=None, d_positions_out=None, sinks: int = 0,
                recent: int = 0, pinned: Optional[GpuRoaring] = None, n_pages: Optional[int] = None, stream=None):
    """Which tokens of each request stay in the cache, by their weights (cr_paged_evict); paged_move then moves them.

    d_weights float32 [R, at least cols * page_size]; d_kv_len, d_keep int32 [R]: how many there are, and how many may
    stay.  Always safe are the first `sinks` and last `recent` of the d_seen int32 [R] tokens that a request has had
    (kv_len if not given), and slots in the bitmap `pinned`.  d_positions int32 [R, ...]: the positions of the first
    d_kept[r] entries, as the last call left them; the others are the newest in order.  Written: d_weights_out and
    d_positions_out (the inputs themselves, if need be), d_len int32 [R], d_moves int32 [R, at least half of
    cols * page_size, 2], d_n_moves int32 [R], d_freed int32 [any], d_counts int32 [2]: pages freed and moves in all.
    n_pages: the cache's (default: any, whatever pinned's universe).  stream: None is the null stream."""
    n, on = d_kv_len.numel(), _device()
    table, cols, stride = _table(d_table, n, on)
    if not (0 < page_size < 1 << 32 and (n_pages is None or 0 <= n_pages < 1 << 32)):
        raise CrError(CR_ERR_INVALID, f"paged_evict: page size {page_size}, {n_pages} pages")
    room = cols * page_size
    weights, weights_stride = _matrix(d_weights, "weights", "float32", n, room, on)
    w_out, w_out_stride = _matrix(d_weights_out, "weights_out", "float32", n, room, on)
    positions, positions_stride = (0, 0) if d_positions is None else _matrix(d_positions, "positions", "int32", n, room, on)
    p_out, p_out_stride = (0, 0) if d_positions_out is None else _matrix(d_positions_out, "positions_out", "int32", n,
                                                                         room, on)
    if d_moves.dim() != 3:
        raise CrError(CR_ERR_INVALID, f"paged_evict: moves [{n}, at least {room // 2}, 2] are taken")
    cap = d_moves.shape[1]
    if n_pages is None:
        n_pages = ((1 << 31) - 1) // page_size
    if not (0 <= sinks < 1 << 32 and 0 <= recent < 1 << 32):
        raise CrError(CR_ERR_INVALID, f"paged_evict: sinks {sinks}, recent {recent}")
    a = _EVICT.pack(weights, weights_stride, positions, positions_stride,
                    0 if d_kept is None else _array(d_kept, "kept", "int32", (n,), on),
                    0 if d_seen is None else _array(d_seen, "seen", "int32", (n,), on),
                    _array(d_kv_len, "kv_len", "int32", (n,), on), _array(d_keep, "keep", "int32", (n,), on), table, cols,
                    stride, page_size, n_pages, n, sinks, recent, C.addressof(pinned) if pinned is not None else 0, w_out,
                    w_out_stride, p_out, p_out_stride, _array(d_len, "len", "int32", (n,), on),
                    _array(d_moves, "moves", "int32", (n, cap, 2), on), cap, cap,
                    _array(d_n_moves, "n_moves", "int32", (n,), on), _array(d_freed, "freed", "int32", 0, on),
                    d_freed.numel(), _array(d_counts, "counts", "int32", (2,), on))
    _check(load().cr_paged_evict(a, _stream(stream)), "paged_evict")


def paged_move(d_moves, d_n_moves, d_k_cache, d_v_cache, stream=None):
    """Keys and values from slot to slot (cr_paged_move): paged_evict's moves int32 [R, any, 2] and n_moves int32 [R],
    once for each layer's cache.  stream: None is the null stream."""
    on = _device()
    cache = _cache(d_k_cache, d_v_cache, on)[0]
    n = d_n_moves.numel()
    cap = d_moves.shape[1] if d_moves.dim() == 3 else 0
    _check(load().cr_paged_move(_array(d_moves, "moves", "int32", (n, cap, 2), on), cap, cap,
                                _array(d_n_moves, "n_moves", "int32", (n,), on), n, cache, _stream(stream)), "paged_move")


def draft_verify(d_scores, d_tokens, d_starts, d_uniform, d_accepted, d_out, d_draft=None, temperature: float = 1.0,
                 allowed=None, stream=None):
    """Drafted tokens against the model's own probabilities, and the token behind the accepted ones (cr_draft_verify).

    d_scores [T, V] and d_draft (or None: looked-up drafts, without probabilities) of one type with contiguous rows: what
    the two models say after each of the step's tokens d_tokens int32 [T], of which request r's are [starts[r],
    starts[r + 1]) and those behind the first are its drafts.  d_uniform: float32 [T] in [0, 1).  Written: d_accepted
    int32 [R], d_out int32 [R, any]: the accepted drafts, one token more, then -1.  allowed: a bitmap over [0, V), or
    int32 bitsets [ceil(V / 32)] (one for all) or [T, ceil(V / 32)], or None.  stream: None is the null stream."""
    on = _device()
    if d_scores.dim() != 2 or d_scores.get_device() != on or (
            d_scores.numel() and d_scores.shape[1] > 1 and d_scores.stride(1) != 1):
        raise CrError(CR_ERR_INVALID, "draft_verify: scores [tokens, vocab] with contiguous rows on the current CUDA "
                                      f"device are taken, not {tuple(d_scores.shape)} on {d_scores.device}")
    rows, vocab = d_scores.shape
    draft = draft_stride = 0
    if d_draft is not None:
        if d_draft.dtype != d_scores.dtype or d_draft.shape != d_scores.shape or d_draft.get_device() != on or (
                rows and vocab > 1 and d_draft.stride(1) != 1):
            raise CrError(CR_ERR_INVALID, f"draft_verify: {d_scores.dtype} draft scores of shape {tuple(d_scores.shape)} "
                                          "with contiguous rows on the current CUDA device are taken")
        draft, draft_stride = d_draft.data_ptr(), d_draft.stride(0)
    n, words, bitmap, bits, bits_stride = d_accepted.numel(), (vocab + 31) // 32, 0, 0, 0
    if isinstance(allowed, GpuRoaring):
        bitmap = C.addressof(allowed)
    elif allowed is not None:
        bits = _array(allowed, "allowed", "int32", (words,) if allowed.dim() == 1 else (rows, words), on)
        bits_stride = 0 if allowed.dim() == 1 else words
    out, out_stride = _matrix(d_out, "out", "int32", n, 0, on)
    a = _VERIFY.pack(d_scores.data_ptr(), d_scores.stride(0), draft, draft_stride, _typed(d_scores), rows, n, vocab,
                     _array(d_tokens, "tokens", "int32", (rows,), on), _array(d_starts, "starts", "int32", (n + 1,), on),
                     _array(d_uniform, "uniform", "float32", (rows,), on), bitmap, bits, bits_stride, temperature,
                     _array(d_accepted, "accepted", "int32", (n,), on), out, d_out.shape[1], out_stride)
    _check(load().cr_draft_verify(a, _stream(stream)), "draft_verify")


def beam_select(d_scores, d_cum, d_out_scores, d_out_tokens, d_out_parents, d_lse=None, allowed=None, stream=None):
    """The k best continuations of each answer's beams (cr_beam_select): k is the outputs' second extent.

    d_scores: [B, W, V] with contiguous rows; d_cum, d_lse: float32 [B, W]; outputs: float32, int32, int32 [B, k].
    allowed: a bitmap over [0, V), or int32 bitsets [ceil(V / 32)] (one for all) or [B, W, ceil(V / 32)], or None.
    stream: None is the null stream."""
    b, w, v = d_scores.shape
    k = d_out_scores.shape[1]
    on = _device()
    if d_scores.get_device() != on or (v > 1 and d_scores.stride(2) != 1):
        raise CrError(CR_ERR_INVALID, "beam_select: scores with contiguous rows on the current CUDA device are taken, not "
                                      f"on {d_scores.device}")
    words, bitmap, bits, stride = (v + 31) // 32, None, None, 0
    if isinstance(allowed, GpuRoaring):
        bitmap = C.byref(allowed)
    elif allowed is not None:
        bits = _array(allowed, "allowed", "int32", (words,) if allowed.dim() == 1 else (b, w, words), on)
        stride = 0 if allowed.dim() == 1 else words
    per_batch, per_beam, _ = d_scores.stride()
    _check(load().cr_beam_select(_dptr(d_scores), _typed(d_scores), b, w, v, per_batch, per_beam,
                                 _array(d_cum, "cum", "float32", (b, w), on),
                                 _array(d_lse, "lse", "float32", (b, w), on) if d_lse is not None else None,
                                 bitmap, bits, stride, k,
                                 _array(d_out_scores, "out_scores", "float32", (b, k), on),
                                 _array(d_out_tokens, "out_tokens", "int32", (b, k), on),
                                 _array(d_out_parents, "out_parents", "int32", (b, k), on), _stream(stream)),
           "beam_select")


def beam_reorder(d_src, d_parents, d_dst, d_len=None, stream=None):
    """d_dst[b, i] = d_src[b, parents[b, i]] for states [B, W, ...] of any type (cr_beam_reorder).

    d_len: int32 [B, W]: only the first d_len[b, parent] entries along the third extent move.  Rows without a parent
    (-1) are left alone.  stream: None is the null stream."""
    b, w, *of_state = d_src.shape
    k = d_parents.shape[1]
    on = _device()
    if not (d_src.get_device() == on == d_dst.get_device() and d_src.is_contiguous() and d_dst.is_contiguous()) or (
            d_src.dtype != d_dst.dtype or d_dst.shape != (b, k, *of_state)):
        raise CrError(CR_ERR_INVALID, f"beam_reorder: contiguous states [{b}, {w}, ...] into [{b}, {k}, ...] on the current CUDA "
                                      "device")
    if d_len is not None and not of_state:
        raise CrError(CR_ERR_INVALID, "beam_reorder: lengths count along the states' third extent")
    row = d_src.nbytes // (b * w or 1)
    unit = row // (of_state[0] or 1) if d_len is not None else 0
    _check(load().cr_beam_reorder(_dptr(d_src), _array(d_parents, "parents", "int32", (b, k), on), b, w, k, row, row, row,
                                  _array(d_len, "len", "int32", (b, w), on) if d_len is not None else None, unit,
                                  _dptr(d_dst), _stream(stream)), "beam_reorder")


def device_free(ptr):
    if ptr:
        _check(load().cr_device_free(ptr), "device_free")


def synchronize(stream=None):
    _check(load().cr_stream_synchronize(_stream(stream)), "stream_synchronize")


def timing_enable(on: bool = True, every: int = 1):
    """Start (or stop) per-kernel HIP-event timing inside the library; clears records.
    every > 1 times only every every-th launch of each kernel."""
    _check(load().cr_timing_enable(max(1, int(every)) if on else 0), "timing_enable")


def timing_report() -> dict:
    """{kernel_name: (launches, total_ms, median_ms)} for the launches since timing_enable()."""
    buf = C.create_string_buffer(1 << 16)
    _check(load().cr_timing_report(buf, len(buf)), "timing_report")
    out = {}
    for line in buf.value.decode().splitlines():
        name, n, ms, med = line.split()
        out[name] = (int(n), float(ms), float(med))
    return out


# ---- download to host (canonical comparison) -----------------------------------
def _d2h(ptr, n, dtype):
    a = np.zeros(n, dtype=dtype)
    if n and ptr:
        _check(load().cr_memcpy_d2h(a.ctypes.data, ptr, a.nbytes), "memcpy_d2h")
    return a


def download(g: GpuRoaring) -> SimpleNamespace:
    """Host copy of every field and pool (same shape as the oracle's HostRoaring)."""
    n = g.n_containers
    kidx = _d2h(g.key_index, g.max_key + 1, np.uint16) if g.key_index else None
    return SimpleNamespace(
        keys=_d2h(g.keys, n, np.uint16),
        types=_d2h(g.types, n, np.uint8),
        offsets=_d2h(g.offsets, n, np.uint32),
        cards=_d2h(g.cardinalities, n, np.uint16),
        n_containers=n,
        universe_size=g.universe_size,
        total_cardinality=g.total_cardinality,
        bitmap_data=_d2h(g.bitmap_data, g.n_bitmap_containers * 1024, np.uint64),
        n_bitmap_containers=g.n_bitmap_containers,
        array_data=_d2h(g.array_data, g.array_pool_bytes // 2, np.uint16),
        n_array_containers=g.n_array_containers,
        array_pool_bytes=g.array_pool_bytes,
        run_data=_d2h(g.run_data, g.run_pool_bytes // 2, np.uint16),
        n_run_containers=g.n_run_containers,
        run_pool_bytes=g.run_pool_bytes,
        key_index=kidx,
        max_key=g.max_key,
        negated=bool(g.negated),
    )
