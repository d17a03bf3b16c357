"""ctypes binding of libhipattn.so, the C ABI declared in include/hipattn.h.

The library is loaded from the package directory; it is never built here.  If
it is missing the import fails loudly (there is no CPU fallback): build it with
``python -m aici_amd.build``.
"""
from __future__ import annotations

import ctypes
from ctypes import POINTER, c_bool, c_char_p, c_float, c_int, c_int32, c_int64, c_void_p
from pathlib import Path

LIB_PATH = Path(__file__).resolve().parent / "libhipattn.so"

MAX_DIMS = 5
F32, F16, BF16, I32, I64, U8 = range(6)


class Tensor(ctypes.Structure):
    """`hipattn_tensor`."""
    _fields_ = [
        ("data", c_void_p),
        ("dtype", c_int32),
        ("ndim", c_int32),
        ("sizes", c_int64 * MAX_DIMS),
        ("strides", c_int64 * MAX_DIMS),
    ]


class MemStats(ctypes.Structure):
    _fields_ = [("current", c_int64), ("peak", c_int64), ("allocated", c_int64), ("freed", c_int64)]


class DeviceProps(ctypes.Structure):
    _fields_ = [
        ("major", c_int32), ("minor", c_int32), ("multi_processor_count", c_int32),
        ("max_threads_per_multi_processor", c_int32), ("total_memory", c_int64),
    ]


class BatchInfo(ctypes.Structure):
    """`hipattn_batch_info`."""
    _fields_ = [
        ("num_tokens", c_int64),
        ("tokens", POINTER(c_int32)),
        ("positions", POINTER(c_int64)),
        ("slot_mapping", POINTER(c_int32)),
        ("num_seqs", c_int64),
        ("logit_idxs", POINTER(c_int32)),
        ("seq_ids", POINTER(c_int64)),
        ("num_multi", c_int64),
        ("seqlens_q", POINTER(c_int32)),
        ("seqlens_k", POINTER(c_int32)),
        ("max_seqlen_q", c_int64),
        ("max_seqlen_k", c_int64),
        ("num_gather", c_int64),
        ("gather_mapping", POINTER(c_int32)),
        ("q_multi", c_int64),
        ("num_paged", c_int64),
        ("paged_max_blocks", c_int64),
        ("paged_block_tables", POINTER(c_int32)),
        ("paged_context_lens", POINTER(c_int32)),
        ("paged_block_size", c_int64),
        ("paged_max_context_len", c_int64),
        ("multi_tables_valid", c_int32),
        ("multi_max_blocks", c_int64),
        ("multi_block_tables", POINTER(c_int32)),
        ("multi_context_lens", POINTER(c_int32)),
    ]


TP = POINTER(Tensor)
ERR = c_void_p  # char* that we must free ourselves

# name -> argtypes; every one of these returns `char*` (NULL = ok).
_ERR_FUNCS = {
    "hipattn_mha_varlen_fwd": [TP, TP, TP, TP, TP, TP, c_int, c_int, c_float, c_float, c_bool, c_bool, c_int, c_int,
                               TP, TP, c_void_p],
    "hipattn_mha_varlen_fwd_paged": [TP, TP, TP, TP, TP, TP, c_int, c_int, c_float, c_bool, TP, TP, c_void_p],
    "hipattn_mha_varlen_fwd_paged_window": [TP, TP, TP, TP, TP, TP, c_int, c_int, c_float, c_int, c_int, TP, TP, TP, c_void_p],
    "hipattn_mha_varlen_fwd_paged_window_workspace_size": [c_int64, c_int, c_int, POINTER(c_int64)],
    "hipattn_paged_attention_window": [TP, TP, TP, TP, c_int, c_float, TP, TP, c_int, c_int, c_int, c_int, TP, TP, c_void_p],
    "hipattn_paged_attention_window_workspace_size": [c_int64, c_int, c_int, c_int, c_int, c_int, c_int, c_int, c_int32,
                                                      POINTER(c_int64)],
    "hipattn_paged_attention_v1": [TP, TP, TP, TP, c_int, c_float, TP, TP, c_int, c_int, TP, c_void_p],
    "hipattn_paged_attention_v1_ws": [TP, TP, TP, TP, c_int, c_float, TP, TP, c_int, c_int, TP, c_void_p, c_int64,
                                      c_void_p],
    "hipattn_paged_attention_v1_static": [TP, TP, TP, TP, c_int, c_float, TP, TP, c_int, c_int, TP, c_void_p],
    "hipattn_init": [],
    "hipattn_paged_attention_workspace_size": [c_int64, c_int, c_int, c_int, c_int, c_int, c_int32, POINTER(c_int64)],
    "hipattn_paged_attention_v2": [TP, TP, TP, TP, TP, TP, TP, c_int, c_float, TP, TP, c_int, c_int, TP, c_void_p],
    "hipattn_reshape_and_cache": [TP, TP, TP, TP, TP, c_void_p],
    "hipattn_gather_cached_kv": [TP, TP, TP, TP, TP, c_void_p],
    "hipattn_copy_blocks_2": [TP, TP, TP, TP, c_void_p],
    "hipattn_copy_blocks_host": [POINTER(c_void_p), POINTER(c_void_p), c_int64, POINTER(c_int64), c_int64, c_int64,
                                 c_void_p],
    "hipattn_swap_blocks": [TP, c_int, TP, c_int, POINTER(c_int64), c_int64, c_void_p],
    "hipattn_rotary_embedding": [TP, TP, TP, c_int, TP, c_bool, c_void_p],
    "hipattn_rotary_embedding_and_cache": [TP, TP, TP, TP, c_int, TP, c_bool, TP, TP, TP, c_void_p],
    "hipattn_rms_norm": [TP, TP, TP, c_float, c_void_p],
    "hipattn_fused_add_rms_norm": [TP, TP, TP, c_float, c_void_p],
    "hipattn_add_rms_norm": [TP, TP, TP, TP, c_float, c_void_p],
    "hipattn_linear": [TP, TP, TP, TP, TP, TP, c_void_p],
    "hipattn_linear_silu_and_mul": [TP, TP, TP, TP, c_void_p],
    "hipattn_rms_norm_linear": [TP, TP, TP, c_float, TP, c_bool, c_void_p],
    "hipattn_qkv_linear": [TP, TP, TP, c_float, TP, TP, TP, TP, TP, TP, c_void_p],
    "hipattn_linear_workspace_size": [TP, TP, POINTER(c_int64)],
    "hipattn_linear_rms_norm": [TP, TP, TP, TP, TP, TP, TP, c_float, TP, c_void_p],
    "hipattn_linear_rms_norm_workspace_size": [TP, TP, POINTER(c_int64)],
    "hipattn_silu_and_mul": [TP, TP, c_void_p],
    "hipattn_gelu_new": [TP, TP, c_void_p],
    "hipattn_gelu_fast": [TP, TP, c_void_p],
    "hipattn_bias_argmax": [TP, TP, TP, TP, TP, TP, c_void_p],
    "hipattn_bias_sample": [TP, TP, TP, TP, TP, TP, TP, TP, c_void_p],
    "hipattn_penalize_logits": [TP, TP, TP, TP, TP, TP, TP, TP, TP, TP, TP, c_void_p],
    "hipattn_step_blocks": [TP, TP, TP, TP, TP, c_int, c_int, c_int, c_int, TP, TP, TP, TP, TP, TP, TP, TP, TP, TP, c_void_p],
    "hipattn_reset_peak_memory_stats": [c_int],
    "hipattn_empty_cache": [],
    "hipattn_get_stats_allocated_bytes": [c_int, POINTER(MemStats)],
    "hipattn_get_device_properties": [c_int, POINTER(DeviceProps)],
    "hipattn_stream_get": [c_int, c_int, POINTER(c_void_p)],
    "hipattn_stream_free": [c_void_p],
    "hipattn_stream_clone": [c_void_p, POINTER(c_void_p)],
    "hipattn_stream_query": [c_void_p, POINTER(c_int)],
    "hipattn_stream_synchronize": [c_void_p],
    "hipattn_stream_set_current": [c_void_p],
    "hipattn_stream_device_index": [c_void_p, POINTER(c_int)],
    "hipattn_stream_id": [c_void_p, POINTER(c_int64)],
    "hipattn_stream_raw": [c_void_p, POINTER(c_void_p)],
    "hipattn_event_create": [c_bool, c_bool, POINTER(c_void_p)],
    "hipattn_event_record": [c_void_p, c_void_p],
    "hipattn_event_block": [c_void_p, c_void_p],
    "hipattn_event_elapsed_time": [c_void_p, c_void_p, POINTER(c_float)],
    "hipattn_event_query": [c_void_p, POINTER(c_int)],
    "hipattn_event_synchronize": [c_void_p],
    "hipattn_event_free": [c_void_p],
    "hipattn_shutdown": [],
    "hipattn_tuning_set": [c_char_p, c_int],
    "hipattn_tuning_get": [c_char_p, POINTER(c_int)],
    "hipattn_block_allocator_new": [c_int64, c_int64, POINTER(c_void_p)],
    "hipattn_block_allocator_alloc_seq": [c_void_p, c_int64, c_int64],
    "hipattn_block_allocator_set_watermark": [c_void_p, ctypes.c_float],
    "hipattn_block_allocator_append_slots": [c_void_p, c_int64, c_int64, c_int64, POINTER(c_int64), c_int64,
                                             POINTER(c_int64)],
    "hipattn_block_allocator_copy": [c_void_p, c_int64, c_int64, c_int64],
    "hipattn_block_allocator_trim": [c_void_p, c_int64, c_int64],
    "hipattn_block_allocator_delete": [c_void_p, c_int64],
    "hipattn_block_allocator_get_block_idxes": [c_void_p, c_int64, c_int64, POINTER(c_int64)],
    "hipattn_block_allocator_swap_out": [c_void_p, c_int64, POINTER(c_int64), c_int64, POINTER(c_int64)],
    "hipattn_block_allocator_swap_in": [c_void_p, c_int64, POINTER(c_int64), c_int64, POINTER(c_int64), c_int64,
                                        POINTER(c_int64)],
    "hipattn_batch_builder_new": [c_int64, c_int64, c_int, POINTER(c_void_p)],
    "hipattn_batch_builder_add": [c_void_p, c_int64, POINTER(c_int64), POINTER(c_int32), c_int64, POINTER(c_int64),
                                  c_int64],
    "hipattn_batch_builder_add_seq": [c_void_p, c_void_p, c_int64, POINTER(c_int32), c_int64, c_int64],
    "hipattn_batch_builder_finish": [c_void_p, POINTER(BatchInfo)],
    "hipattn_decode_batch_new": [c_int64, c_int64, POINTER(c_void_p)],
    "hipattn_decode_batch_add": [c_void_p, c_void_p, c_int64, c_int32, c_int64],
    "hipattn_decode_batch_advance": [c_void_p, c_void_p, c_int64, c_int32],
    "hipattn_decode_batch_advance_all": [c_void_p, c_void_p, POINTER(c_int32), c_int64],
    "hipattn_decode_batch_remove": [c_void_p, c_int64],
    "hipattn_decode_batch_info": [c_void_p, POINTER(BatchInfo)],
    "hipattn_block_allocator_step_generation": [c_void_p, POINTER(c_int64), POINTER(c_int64), POINTER(c_int64), c_int64,
                                                POINTER(c_int64), POINTER(c_int64), POINTER(c_int64), POINTER(c_int64),
                                                POINTER(c_int64), c_int64, POINTER(c_int64)],
    "hipattn_block_space_step_generation": [c_void_p, c_void_p, c_int64, POINTER(c_int64), POINTER(c_int64),
                                            POINTER(c_int64), POINTER(c_int32), POINTER(c_int64), POINTER(c_int64),
                                            POINTER(c_int32), POINTER(c_int64), c_int64, POINTER(c_int64),
                                            POINTER(c_int64), c_int64, POINTER(c_int64)],
    "hipattn_varlen_attn": [TP, TP, TP, TP, TP, TP, TP, TP, TP, c_int64, c_int, c_int, TP, TP, c_int, c_int, c_float,
                            TP, TP, TP, c_void_p],
    "hipattn_varlen_attn_paged": [TP, TP, TP, TP, TP, TP, TP, TP, TP, c_int64, c_int, c_int, TP, TP, c_int, c_int,
                                  c_float, TP, c_void_p],
    "hipattn_varlen_attn_paged_window": [TP, TP, TP, TP, TP, TP, TP, TP, TP, c_int64, c_int, c_int, TP, TP, c_int, c_int,
                                         c_float, c_int, c_int, TP, c_void_p],
    "hipattn_varlen_attn_paged_window_ws": [TP, TP, TP, TP, TP, TP, TP, TP, TP, c_int64, c_int, c_int, TP, TP, c_int, c_int,
                                            c_float, c_int, c_int, TP, TP, c_void_p],
}

# name -> (restype, argtypes) for the few calls that do not return an error string.
_PLAIN_FUNCS = {
    "hipattn_free_error": (None, [c_void_p]),
    "hipattn_version": (c_char_p, []),
    "hipattn_block_allocator_free": (None, [c_void_p]),
    "hipattn_block_allocator_num_free": (c_int64, [c_void_p]),
    "hipattn_block_allocator_can_allocate": (ctypes.c_int, [c_void_p, c_int64]),
    "hipattn_block_allocator_can_append_slot": (ctypes.c_int, [c_void_p, c_int64]),
    "hipattn_block_allocator_num_allocated": (c_int64, [c_void_p, c_int64]),
    "hipattn_batch_builder_free": (None, [c_void_p]),
    "hipattn_decode_batch_free": (None, [c_void_p]),
    "hipattn_decode_batch_size": (c_int64, [c_void_p]),
    "hipattn_cache_x": (c_int64, [c_int32]),
    "hipattn_cache_block_bytes": (c_int64, [c_int64, c_int64, c_int64, c_int64, c_int32]),
}

EXPORTED_SYMBOLS = sorted(list(_ERR_FUNCS) + list(_PLAIN_FUNCS))


class HipAttnError(RuntimeError):
    """A C-ABI call returned an error string (the reference's Rust side panics here,
    rllm/tch-cuda/src/lib.rs:22-27)."""


_lib = None


def load() -> ctypes.CDLL:
    global _lib
    if _lib is not None:
        return _lib
    if not LIB_PATH.exists():
        raise ImportError(
            f"{LIB_PATH} is missing: the HIP extension is not built. "
            "Run `python -m aici_amd.build` (needs hipcc; no GPU required).")
    lib = ctypes.CDLL(str(LIB_PATH))
    for name, argtypes in _ERR_FUNCS.items():
        fn = getattr(lib, name)
        fn.restype = ERR
        fn.argtypes = argtypes
    for name, (restype, argtypes) in _PLAIN_FUNCS.items():
        fn = getattr(lib, name)
        fn.restype = restype
        fn.argtypes = argtypes
    _lib = lib
    return lib


def call(name: str, *args) -> None:
    """Calls an error-returning entry point; raises HipAttnError on a message."""
    lib = load()
    err = getattr(lib, name)(*args)
    if err:
        msg = ctypes.string_at(err).decode("utf-8", "replace")
        lib.hipattn_free_error(err)
        raise HipAttnError(f"{name}: {msg}")
