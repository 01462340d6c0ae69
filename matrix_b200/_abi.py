"""ctypes binding of include/mtxc.h (libmtxc.so).

This is the binding a Python caller of the C ABI needs; it loads the in-tree library built by
``matrix_b200/build.py`` and fails loudly when it is missing -- there is no CPU fallback.
"""
from __future__ import annotations

import ctypes as C
import struct
from pathlib import Path

LIB_PATH = Path(__file__).resolve().parent / "lib" / "libmtxc.so"

MAX_DIMS = 8
OK = 0
ERR_INVALID_ARGUMENT = 1
ERR_UNSUPPORTED_DTYPE = 2
ERR_SHAPE = 3
ERR_CUDA = 4
ERR_TIMEOUT = 5
ERR_NOT_INITIALIZED = 6
ERR_WORKSPACE = 7
ERR_COMM = 8
COMM_ID_BYTES = 128

REDUCE_OPS = {"sum": 0, "max": 1, "min": 2, "argmax": 3, "argmin": 4}
BINARY_OPS = {"add": 0, "sub": 1, "mul": 2, "div": 3, "max": 4, "min": 5, "equal": 6}
UNARY_OPS = {"exp": 0, "sqrt": 1}
STATS = {"mean": 0, "rms": 1, "norm": 2}
POINTWISE_OPS = {"greater": 0, "less": 1, "logical_and": 2, "where": 3, "floor": 4, "full": 5, "arctan2": 6,
                 "arcsin": 7}



def _layout(*fields: str) -> struct.Struct:
    """A C struct of include/mtxc.h as its fields in order, each "name:type" (struct module letters, native
    alignment); packed bytes are passed as the pointer to it."""
    return struct.Struct("@" + "".join(f.split(":")[1] for f in fields) + "0P")


DROPOUT_FIELDS = ("p:d", "seed:Q", "offset:Q", "device_offset:P")
DROPOUT_STATE = _layout(*DROPOUT_FIELDS)
BLOCK_NORM_FIELDS = (
    "rows:Q", "width:Q", "residual:P", "residual_stride:Q", "branch:P", "branch_stride:Q", "post_weight:P",
    "next_weight:P", "gate:P", "gate_stride:Q", "gate_rows:Q", "residual_out:P", "residual_out_stride:Q", "normed:P",
    "normed_stride:Q", "post_rstd:P", "next_rstd:P", "weight_dtype:i", "gate_dtype:i", "residual_scale:f",
    "branch_scale:f", "weight_offset:f", "eps:f", *("drop." + f for f in DROPOUT_FIELDS))
BLOCK_NORM_ARGS = _layout(*BLOCK_NORM_FIELDS)
BLOCK_NORM_BACKWARD_FIELDS = (
    "rows:Q", "width:Q", "d_residual_out:P", "d_residual_out_stride:Q", "d_normed:P", "d_normed_stride:Q",
    "residual_out:P", "residual_out_stride:Q", "branch:P", "branch_stride:Q", "post_rstd:P", "next_rstd:P",
    "post_weight:P", "next_weight:P", "gate:P", "gate_stride:Q", "gate_rows:Q", "d_residual:P", "d_residual_stride:Q",
    "d_branch:P", "d_branch_stride:Q", "d_post_weight:P", "d_next_weight:P", "d_gate:P", "d_gate_stride:Q",
    "weight_dtype:i", "gate_dtype:i", "residual_scale:f", "branch_scale:f", "weight_offset:f",
    *("drop." + f for f in DROPOUT_FIELDS))
BLOCK_NORM_BACKWARD_ARGS = _layout(*BLOCK_NORM_BACKWARD_FIELDS)
ROTARY_FIELDS = (
    "batch:Q", "length:Q", "head_dim:I", "rotary_dim:I", "heads:2I", "dst:2P", "dst_strides:6Q", "src:2P",
    "src_strides:6Q", "positions:P", "position_dtype:i", "position_strides:2Q", "frequencies:P", "scale:f",
    "interleaved:i", "inverse:i")
ROTARY_ARGS = _layout(*ROTARY_FIELDS)
LOGITS_FIELDS = (
    "rows:Q", "vocab:Q", "dst:P", "dst_stride:Q", "src:P", "src_stride:Q", "tokens:P", "tokens_stride:Q", "history:Q",
    "lengths:P", "prompt_lengths:P", "repetition:P", "frequency:P", "presence:P", "bias_tokens:P",
    "bias_tokens_stride:Q", "bias_values:P", "bias_values_stride:Q", "biases:Q", "mask:P", "mask_stride:Q")
LOGITS_ARGS = _layout(*LOGITS_FIELDS)
HEAD_NORM_FIELDS = (
    "batch:Q", "length:Q", "head_dim:I", "rotary_dim:I", "heads:2I", "dst:2P", "dst_strides:6Q", "src:2P",
    "src_strides:6Q", "weight:2P", "rstd:2P", "positions:P", "position_strides:2Q", "frequencies:P", "position_dtype:i",
    "weight_dtype:i", "scale:f", "weight_offset:f", "eps:f", "interleaved:i", "d_out:2P", "d_out_strides:6Q",
    "d_weight:2P", "workspace:P", "workspace_bytes:N")
HEAD_NORM_ARGS = _layout(*HEAD_NORM_FIELDS)
KV_CACHE_FIELDS = (
    "pages:Q", "page_size:I", "heads:I", "head_dim:I", "dtype:i", "data:2P", "strides:6Q", "exponents:2P",
    "exponent_strides:6Q")
KV_CACHE = _layout(*KV_CACHE_FIELDS)
CACHE_ROWS_FIELDS = (
    *("cache." + f for f in KV_CACHE_FIELDS), "tokens:Q", "rows:2P", "row_strides:4Q", "slots:P", "slot_stride:Q",
    "slot_dtype:i")
CACHE_ROWS_ARGS = _layout(*CACHE_ROWS_FIELDS)
DECODE_ATTENTION_FIELDS = (
    *("cache." + f for f in KV_CACHE_FIELDS), "batch:Q", "max_pages:Q", "heads:I", "scale:f", "q:P", "q_strides:2Q",
    "out:P", "out_strides:2Q", "page_table:P", "page_table_stride:Q", "lengths:P", "workspace:P", "workspace_bytes:N")
DECODE_ATTENTION_ARGS = _layout(*DECODE_ATTENTION_FIELDS)
PROMPT_ATTENTION_FIELDS = (
    "tokens:Q", "k_tokens:Q", "sequences:Q", "heads:I", "kv_heads:I", "head_dim:I", "scale:f", "q:P", "q_strides:2Q",
    "k:P", "k_strides:2Q", "v:P", "v_strides:2Q", "out:P", "out_strides:2Q", "starts:P", "k_starts:P", "causal:i")
PROMPT_ATTENTION_ARGS = _layout(*PROMPT_ATTENTION_FIELDS)
FLOAT8_E4M3 = 32  # of caches only
ROTARY_SCALINGS = {"none": 0, "linear": 1, "base": 2, "by_parts": 3}


class MtxcError(RuntimeError):
    """A non-zero status from the C ABI, with mtxc_last_error()'s message."""

    def __init__(self, code: int, message: str):
        super().__init__(f"mtxc error {code}: {message}")
        self.code = code


U32P = C.POINTER(C.c_uint32)
_lib = None


def lib() -> C.CDLL:
    global _lib
    if _lib is None:
        if not LIB_PATH.exists():
            raise ImportError(f"{LIB_PATH} not found: build it with `python -m matrix_b200.build`")
        L = C.CDLL(str(LIB_PATH))
        i32, u32, u64, sz, vp = C.c_int, C.c_uint32, C.c_uint64, C.c_size_t, C.c_void_p
        sigs = {
            "mtxc_abi_version": (i32, []),
            "mtxc_init": (i32, [i32]),
            "mtxc_shutdown": (i32, []),
            "mtxc_last_error": (C.c_char_p, []),
            "mtxc_device_count": (i32, [C.POINTER(i32)]),
            "mtxc_set_stream": (i32, [vp]),
            "mtxc_use_own_stream": (i32, []),
            "mtxc_get_stream": (vp, []),
            "mtxc_sync": (i32, []),
            "mtxc_set_workspace": (i32, [vp, sz]),
            "mtxc_workspace_size": (i32, [C.POINTER(sz)]),
            "mtxc_reduce_workspace_bytes": (i32, [i32, i32, u32, u32, u32, U32P, U32P, U32P, C.POINTER(sz)]),
            "mtxc_alloc": (i32, [sz, C.POINTER(vp)]),
            "mtxc_free": (i32, [vp]),
            "mtxc_host_alloc": (i32, [sz, C.POINTER(vp)]),
            "mtxc_host_free": (i32, [vp]),
            "mtxc_upload": (i32, [vp, vp, sz]),
            "mtxc_download": (i32, [vp, vp, sz]),
            "mtxc_copy_device": (i32, [vp, vp, sz]),
            "mtxc_memset": (i32, [vp, i32, sz]),
            "mtxc_collapse_dims1": (u32, [U32P, U32P, u32, u64, U32P, U32P]),
            "mtxc_collapse_dims2": (u32, [U32P, U32P, U32P, u32, u64, U32P, U32P, U32P]),
            "mtxc_collapse_dims3": (u32, [U32P, U32P, U32P, U32P, u32, u64, U32P, U32P, U32P, U32P]),
            "mtxc_collapse_dims_reduce1": (u32, [U32P, U32P, u32, i32, i32, u64, U32P, U32P]),
            "mtxc_collapse_dims_reduce2": (u32, [U32P, U32P, U32P, u32, i32, i32, i32, u64, U32P, U32P, U32P]),
            "mtxc_collapse_dims_reduce3": (u32, [U32P, U32P, U32P, U32P, u32, i32, i32, u64, U32P, U32P, U32P, U32P]),
            "mtxc_broadcast_shapes": (i32, [U32P, U32P, i32, U32P, U32P, i32, U32P, U32P, U32P, U32P, U32P, U32P]),
            "mtxc_promote_types": (i32, [i32, i32]),
            "mtxc_reduce": (i32, [i32, i32, vp, vp, u32, u32, u32, U32P, U32P, U32P]),
            "mtxc_reduce_noalloc": (i32, [i32, i32, vp, vp, u32, u32, u32, U32P, U32P, U32P]),
            "mtxc_reduce_pair": (i32, [i32, i32, vp, vp, vp, u32, u32, u32, U32P, U32P, U32P]),
            "mtxc_merge_partials": (i32, [i32, i32, vp, vp, vp, vp, vp, u32, u64]),
            "mtxc_broadcast_binary": (i32, [i32, i32, vp, vp, vp, u32, U32P, U32P, U32P, U32P]),
            "mtxc_broadcast_binary_mixed": (i32, [i32, i32, i32, i32, vp, vp, vp, u32, U32P, U32P, U32P, U32P]),
            "mtxc_unary": (i32, [i32, i32, vp, vp, u32, U32P, U32P, U32P]),
            "mtxc_softmax_lastdim": (i32, [i32, vp, vp, u64, u32, u64, u64]),
            "mtxc_astype": (i32, [i32, i32, vp, vp, u32, U32P, U32P, U32P]),
            "mtxc_reduce_stat": (i32, [i32, i32, vp, vp, u32, u32, u32, U32P, U32P, U32P]),
            "mtxc_reduce_stat_dtype": (i32, [i32, i32, u32]),
            "mtxc_pointwise_collapse": (u32, [U32P, u32, U32P, u32, U32P, U32P]),
            "mtxc_pointwise": (i32, [i32, i32, vp, C.POINTER(vp), u32, u32, U32P, U32P]),
            "mtxc_comm_unique_id": (i32, [vp, sz]),
            "mtxc_comm_init": (i32, [i32, i32, vp, sz]),
            "mtxc_comm_destroy": (i32, []),
            "mtxc_comm_size": (i32, [C.POINTER(i32), C.POINTER(i32)]),
            "mtxc_comm_status": (i32, [C.POINTER(i32), C.POINTER(i32)]),
            "mtxc_reduce_sharded": (i32, [i32, i32, vp, vp, u32, u32, u32, U32P, U32P, U32P, C.POINTER(C.c_int64)]),
            "mtxc_allreduce": (i32, [i32, i32, vp, u64]),
            "mtxc_get_device": (i32, [C.POINTER(i32)]),
            "mtxc_arange": (i32, [i32, vp, vp, vp, u64]),
            "mtxc_dropout": (i32, [i32, vp, vp, u64, u64, u64, u64, C.c_char_p]),
            "mtxc_block_norm": (i32, [i32, C.c_char_p]),
            "mtxc_block_norm_backward": (i32, [i32, C.c_char_p]),
            "mtxc_rotary": (i32, [i32, C.c_char_p]),
            "mtxc_rotary_frequencies": (i32, [i32, u32, C.c_double, C.c_double, C.c_double, C.c_double, C.c_double,
                                              C.POINTER(C.c_double), C.POINTER(C.c_double)]),
            "mtxc_logits_rules": (i32, [i32, C.c_char_p]),
            "mtxc_head_norm_rotary": (i32, [i32, C.c_char_p]),
            "mtxc_head_norm_rotary_backward": (i32, [i32, C.c_char_p]),
            "mtxc_head_norm_rotary_backward_workspace": (i32, [i32, C.c_char_p, C.POINTER(sz)]),
            "mtxc_cache_write": (i32, [i32, C.c_char_p]),
            "mtxc_cache_read": (i32, [i32, C.c_char_p]),
            "mtxc_decode_attention": (i32, [i32, C.c_char_p]),
            "mtxc_decode_attention_workspace": (i32, [i32, C.c_char_p, C.POINTER(sz)]),
            "mtxc_prompt_attention": (i32, [i32, C.c_char_p]),
            "mtxc_waits_gave_up": (i32, [C.POINTER(i32)]),
            "mtxc_graph_begin": (i32, []),
            "mtxc_graph_recording": (i32, [C.POINTER(i32)]),
            "mtxc_graph_end": (i32, [C.POINTER(vp)]),
            "mtxc_graph_launch": (i32, [vp]),
            "mtxc_graph_destroy": (i32, [vp]),
        }
        for name, (res, args) in sigs.items():
            f = getattr(L, name)
            f.restype, f.argtypes = res, args
        _lib = L
    return _lib


def check(rc: int) -> None:
    if rc != OK:
        msg = lib().mtxc_last_error()
        raise MtxcError(rc, msg.decode() if msg else "")


def u32_array(values, n: int = MAX_DIMS):
    a = (C.c_uint32 * n)()
    for i, v in enumerate(values):
        v = int(v)
        if v < 0 or v > 0xFFFFFFFF:
            raise ValueError(f"value {v} does not fit the reference's 32-bit size_m")
        a[i] = v
    return a
