"""Python host binding of the C-ABI in include/minirun_hip.h.

The library is loaded from minirun-app_amd/lib/ (built by build.py); there is
no fallback: if it is missing, every call raises.  torch is used only for
device memory, streams and dtypes; all arithmetic runs in the HIP library.

Names follow the reference operators they stand in for:
  mla_decode            K3MLA absorbed attention core (MLA.swift:174-197)
  sparse_attention      DeepSeekV4SparseAttention.forward (DeepSeekV4Attention.swift:747-770)
  validate_indices      its index checks (DeepSeekV4Attention.swift:884-895)
  MXFP4Weights          the MXFP4 storage (MXFP4Weights.swift:36-60); mxfp4_quantize,
                        mxfp4_dequantize, mxfp4_mm, mxfp4_expert_mm
  expert_sort           tokens by expert and back, for QwenExpertBackends.swift:77-260;
                        expert_dispatch, expert_combine and their gradients
  head_norm_rope        norms of query and key heads with the rotation, of
                        QwenAttention.forward (QwenMoEModel.swift:193-264), and
                        head_norm_rope_backward; KVCache, kv_append, kv_attention:
                        its keys, values and attention, in pages
"""
from __future__ import annotations

import contextlib
import ctypes as C
import threading
import os

HERE = os.path.dirname(os.path.abspath(__file__))
LIB_DIR = os.path.join(HERE, "lib")
LIB_PATH = os.path.join(LIB_DIR, "libminirun_hip.so")
SELFTEST_PATH = os.path.join(LIB_DIR, "libminirun_selftest.so")

OK, INVALID_SHAPE, INVALID_DTYPE, INDEX_OUT_OF_RANGE, DUPLICATE_INDEX, NONFINITE, HIP_ERROR, \
    INVALID_ARGUMENT, WORKSPACE_TOO_SMALL = range(9)
BF16, F16, F32, U32, I32, U8 = range(6)

DECODE_VALIDATE_INDICES = 1
DECODE_SPLIT_ONLY = 4
DECODE_UNCHECKED = 8
DECODE_NOALLOC_SCRATCH_BYTES = 48 * 1024 * 1024


class MRError(RuntimeError):
    def __init__(self, status: int, message: str):
        super().__init__(f"[mr_status {status}] {message}")
        self.status = status
        self.message = message


class DecodeArgs(C.Structure):
    _fields_ = [
        ("batch", C.c_int32), ("heads", C.c_int32), ("n_ctx", C.c_int32), ("kv_rank", C.c_int32),
        ("rope_dim", C.c_int32), ("scale", C.c_float),
        ("q_lat", C.c_void_p), ("q_lat_batch_stride", C.c_int64), ("q_lat_head_stride", C.c_int64),
        ("q_rope", C.c_void_p), ("q_rope_batch_stride", C.c_int64), ("q_rope_head_stride", C.c_int64),
        ("latent", C.c_void_p), ("latent_row_stride", C.c_int64), ("latent_batch_stride", C.c_int64),
        ("rope_keys", C.c_void_p), ("rope_row_stride", C.c_int64), ("rope_batch_stride", C.c_int64),
        ("indices", C.c_void_p), ("n_idx", C.c_int32),
        ("sinks", C.c_void_p),
        ("out", C.c_void_p), ("out_dtype", C.c_int), ("out_batch_stride", C.c_int64),
        ("out_head_stride", C.c_int64),
        ("workspace", C.c_void_p), ("workspace_bytes", C.c_size_t),
        ("num_splits", C.c_int32), ("flags", C.c_uint32),
        ("phase_events", C.c_void_p),
        ("index_status", C.c_void_p),
    ]


class AffineWeightDesc(C.Structure):
    _fields_ = [
        ("packed", C.c_void_p), ("scales", C.c_void_p), ("biases", C.c_void_p), ("scale_dtype", C.c_int),
        ("out_features", C.c_int64), ("in_features", C.c_int64), ("group", C.c_int32), ("bits", C.c_int32),
    ]


class DenseWeightDesc(C.Structure):
    _fields_ = [
        ("weight", C.c_void_p), ("dtype", C.c_int), ("out_features", C.c_int64), ("in_features", C.c_int64),
        ("row_stride", C.c_int64),
    ]


PROJ_NONE, PROJ_AFFINE, PROJ_DENSE = 0, 1, 2


class ProjectionDesc(C.Structure):
    _fields_ = [("kind", C.c_int), ("affine", AffineWeightDesc), ("dense", DenseWeightDesc)]


class BlockArgs(C.Structure):
    _fields_ = [
        ("hidden", C.c_int32), ("q_lora_rank", C.c_int32), ("heads", C.c_int32), ("qk_nope_dim", C.c_int32),
        ("qk_rope_dim", C.c_int32), ("v_head_dim", C.c_int32), ("kv_rank", C.c_int32),
        ("eps", C.c_float), ("scale", C.c_float),
        ("x", C.c_void_p), ("input_norm_w", C.c_void_p), ("q_a_norm_w", C.c_void_p), ("kv_a_norm_w", C.c_void_p),
        ("norm_w_dtype", C.c_int),
        ("q_a", ProjectionDesc), ("q_b", ProjectionDesc), ("kv_a", ProjectionDesc), ("kv_b", ProjectionDesc),
        ("o_proj", ProjectionDesc), ("g_proj", ProjectionDesc),
        ("cache_latent", C.c_void_p), ("latent_row_stride", C.c_int64),
        ("cache_rope", C.c_void_p), ("rope_row_stride", C.c_int64),
        ("position", C.c_int32), ("capacity", C.c_int32),
        ("rope_cos", C.c_void_p), ("rope_sin", C.c_void_p),
        ("out", C.c_void_p),
        ("workspace", C.c_void_p), ("workspace_bytes", C.c_size_t),
    ]


class PrefillArgs(C.Structure):
    _fields_ = [
        ("tokens", C.c_int32), ("n_ctx", C.c_int32), ("heads", C.c_int32),
        ("qk_nope_dim", C.c_int32), ("qk_rope_dim", C.c_int32), ("v_head_dim", C.c_int32), ("kv_rank", C.c_int32),
        ("scale", C.c_float),
        ("q", C.c_void_p), ("q_token_stride", C.c_int64), ("q_head_stride", C.c_int64),
        ("latent", C.c_void_p), ("latent_row_stride", C.c_int64),
        ("rope_keys", C.c_void_p), ("rope_row_stride", C.c_int64),
        ("kv_b", C.c_void_p), ("kv_b_row_stride", C.c_int64),
        ("out", C.c_void_p), ("out_dtype", C.c_int), ("out_token_stride", C.c_int64), ("out_head_stride", C.c_int64),
        ("workspace", C.c_void_p), ("workspace_bytes", C.c_size_t),
        ("phase_events", C.c_void_p),
    ]


class PrefillBlockArgs(C.Structure):
    _fields_ = [
        ("tokens", C.c_int32),
        ("hidden", C.c_int32), ("q_lora_rank", C.c_int32), ("heads", C.c_int32), ("qk_nope_dim", C.c_int32),
        ("qk_rope_dim", C.c_int32), ("v_head_dim", C.c_int32), ("kv_rank", C.c_int32),
        ("eps", C.c_float), ("scale", C.c_float),
        ("x", C.c_void_p), ("x_token_stride", C.c_int64),
        ("input_norm_w", C.c_void_p), ("q_a_norm_w", C.c_void_p), ("kv_a_norm_w", C.c_void_p),
        ("norm_w_dtype", C.c_int),
        ("q_a", ProjectionDesc), ("q_b", ProjectionDesc), ("kv_a", ProjectionDesc), ("kv_b", ProjectionDesc),
        ("o_proj", ProjectionDesc), ("g_proj", ProjectionDesc),
        ("cache_latent", C.c_void_p), ("latent_row_stride", C.c_int64),
        ("cache_rope", C.c_void_p), ("rope_row_stride", C.c_int64),
        ("position", C.c_int32), ("capacity", C.c_int32),
        ("rope_cos", C.c_void_p), ("rope_sin", C.c_void_p),
        ("out", C.c_void_p), ("out_token_stride", C.c_int64),
        ("workspace", C.c_void_p), ("workspace_bytes", C.c_size_t),
    ]


class TopkArgs(C.Structure):
    _fields_ = [
        ("scores", C.c_void_p), ("score_row_stride", C.c_int64), ("rows", C.c_int32), ("cols", C.c_int32),
        ("top_k", C.c_int32), ("ratio", C.c_int32), ("start_pos", C.c_int32), ("offset", C.c_int32),
        ("out", C.c_void_p), ("out_row_stride", C.c_int64), ("status", C.c_void_p), ("flags", C.c_int32),
        ("workspace", C.c_void_p), ("workspace_bytes", C.c_size_t),
    ]


class MXFP4Desc(C.Structure):
    _fields_ = [("packed", C.c_void_p), ("scales", C.c_void_p), ("rows", C.c_int64), ("cols", C.c_int64)]


class MXFP4ExpertArgs(C.Structure):
    _fields_ = [
        ("x", C.c_void_p), ("x_dtype", C.c_int), ("x_stride", C.c_int64), ("x_scales", C.c_void_p), ("x_rows", C.c_int32),
        ("w", MXFP4Desc), ("experts", C.c_int32), ("offsets", C.c_void_p), ("pair_of_row", C.c_void_p),
        ("per_token", C.c_int32), ("rows", C.c_int32),
        ("y", C.c_void_p), ("y_dtype", C.c_int), ("y_stride", C.c_int64),
    ]


class Rotary(C.Structure):
    _fields_ = [("cos_t", C.c_void_p), ("sin_t", C.c_void_p), ("positions", C.c_void_p), ("table_rows", C.c_int64),
                ("dim", C.c_int32), ("col0", C.c_int32), ("pairs", C.c_int)]


class HeadRows(C.Structure):
    _fields_ = [
        ("heads", C.c_int32), ("x", C.c_void_p), ("x_token_stride", C.c_int64), ("x_head_stride", C.c_int64),
        ("weight", C.c_void_p), ("out", C.c_void_p), ("out_token_stride", C.c_int64), ("out_head_stride", C.c_int64),
        ("d_out", C.c_void_p), ("d_out_token_stride", C.c_int64), ("d_out_head_stride", C.c_int64), ("d_weight", C.c_void_p),
    ]


class HeadNormArgs(C.Structure):
    _fields_ = [
        ("tokens", C.c_int32), ("dim", C.c_int32), ("q", HeadRows), ("k", HeadRows), ("x_dtype", C.c_int),
        ("weight_dtype", C.c_int), ("out_dtype", C.c_int), ("eps", C.c_float), ("rope", Rotary), ("workspace", C.c_void_p),
        ("workspace_bytes", C.c_size_t),
    ]


class KVCacheDesc(C.Structure):
    _fields_ = [
        ("k", C.c_void_p), ("v", C.c_void_p), ("k_scales", C.c_void_p), ("v_scales", C.c_void_p), ("pages", C.c_int32),
        ("page_size", C.c_int32), ("kv_heads", C.c_int32), ("head_dim", C.c_int32), ("page_stride", C.c_int64),
        ("scale_page_stride", C.c_int64),
    ]


class KVAppendArgs(C.Structure):
    _fields_ = [
        ("cache", KVCacheDesc), ("tokens", C.c_int32), ("k", C.c_void_p), ("v", C.c_void_p), ("dtype", C.c_int),
        ("k_token_stride", C.c_int64), ("k_head_stride", C.c_int64), ("v_token_stride", C.c_int64),
        ("v_head_stride", C.c_int64), ("slots", C.c_void_p), ("normalize", C.c_int32), ("norm_w", C.c_void_p),
        ("norm_w_dtype", C.c_int), ("eps", C.c_float), ("rope", Rotary),
    ]


class KVAttentionArgs(C.Structure):
    _fields_ = [
        ("cache", KVCacheDesc), ("batch", C.c_int32), ("tokens", C.c_int32), ("heads", C.c_int32), ("q", C.c_void_p),
        ("q_token_stride", C.c_int64), ("q_head_stride", C.c_int64), ("page_table", C.c_void_p),
        ("page_table_stride", C.c_int64), ("max_pages", C.c_int32), ("kv_lens", C.c_void_p), ("q_offsets", C.c_void_p),
        ("max_kv_len", C.c_int32), ("window", C.c_int32), ("scale", C.c_float), ("sinks", C.c_void_p), ("out", C.c_void_p),
        ("out_dtype", C.c_int), ("out_token_stride", C.c_int64), ("out_head_stride", C.c_int64), ("lse", C.c_void_p),
        ("workspace", C.c_void_p), ("workspace_bytes", C.c_size_t),
    ]


TOPK_CHECK = 1
TOPK_UNCHECKED = 2

_P = C.c_void_p
_I32P = C.POINTER(C.c_int32)
_I64P = C.POINTER(C.c_int64)

# Every symbol include/minirun_hip.h declares, with its ctypes signature.
SIGNATURES = {
    "mr_version": (C.c_char_p, []),
    "mr_get_last_error": (C.c_char_p, []),
    "mr_mla_decode_workspace_size": (C.c_size_t, [C.POINTER(DecodeArgs)]),
    "mr_mla_decode": (C.c_int, [C.POINTER(DecodeArgs), C.c_void_p]),
    "mr_mla_decode_noalloc": (C.c_int, [C.POINTER(DecodeArgs), C.c_void_p]),
    "mr_validate_indices_workspace_size": (C.c_size_t, [C.c_int32, C.c_int32]),
    "mr_validate_indices": (C.c_int, [C.c_void_p, C.c_int32, C.c_int32, C.c_int32, C.c_void_p, C.c_size_t,
                                      C.POINTER(C.c_int32), C.POINTER(C.c_int32), C.c_void_p]),
    "mr_affine_validate": (C.c_int, [C.c_int, C.c_int32, _I64P, C.c_int, C.c_int32, _I64P, C.c_int, C.c_int32, _I64P,
                                     C.c_int32, C.c_int32, _I64P, _I64P, _I64P]),
    "mr_affine_dequantize": (C.c_int, [C.POINTER(AffineWeightDesc), _P, C.c_int, _P]),
    "mr_affine_matmul": (C.c_int, [_P, C.c_int, C.c_int32, C.c_int64, C.POINTER(AffineWeightDesc), _P, C.c_int,
                                   C.c_int64, _P]),
    "mr_affine_tile_view": (C.c_int, [_P, C.c_int64, C.c_int64, C.c_int32, C.c_int32, C.c_int,
                                      C.POINTER(AffineWeightDesc), C.POINTER(C.c_int64)]),
    "mr_tile_upload": (C.c_int, [_P, _P, C.c_int64, _P]),
    "mr_affine_adopt": (C.c_int, [_P, _P, _P, C.c_int, C.c_int64, C.c_int64, C.c_int64, C.c_int32, C.c_int32,
                                  _P, _P, _P, _P, _P, _P, C.POINTER(_P)]),
    "mr_adopted_affine_weight": (C.c_int, [_P, C.POINTER(AffineWeightDesc)]),
    "mr_adopted_affine_retain": (C.c_int, [_P]),
    "mr_adopted_affine_release": (C.c_int, [_P, _P]),
    "mr_adopted_affine_release_now": (C.c_int, [_P]),
    "mr_affine_gather_matmul": (C.c_int, [_P, C.c_int, C.c_int32, C.c_int64, C.POINTER(AffineWeightDesc), C.c_int64,
                                          _P, C.c_int32, _P, C.c_int, _P]),
    "mr_rmsnorm": (C.c_int, [_P, C.c_int, C.c_int64, C.c_int32, C.c_int64, _P, C.c_int, C.c_float, _P, C.c_int,
                             C.c_int64, _P]),
    "mr_rope_frequencies": (C.c_int, [C.c_int32, C.c_int32, C.c_double, C.c_double, C.c_double, C.c_double, _P]),
    "mr_rope_table": (C.c_int, [_P, C.c_int64, _P, C.c_int32, C.c_int32, _P, _P]),
    "mr_rope_apply": (C.c_int, [_P, C.c_int, C.c_int64, C.c_int64, C.c_int64, C.c_int64, C.c_int32, _P, _P, _P]),
    "mr_mla_cache_append": (C.c_int, [_P, C.c_int, C.c_int64, C.c_int64, _P, C.c_int, C.c_float, C.c_int32, C.c_int32,
                                      _P, _P, _P, C.c_int64, _P, C.c_int64, C.c_int64, _P]),
    "mr_mla_absorb_query": (C.c_int, [_P, C.c_int64, C.c_int32, C.c_int32, C.c_int32, C.POINTER(ProjectionDesc), _P,
                                      C.c_int64, _P]),
    "mr_mla_unabsorb_values": (C.c_int, [_P, C.c_int64, C.c_int32, C.c_int32, C.c_int32, C.POINTER(ProjectionDesc),
                                         _P, C.c_int, _P]),
    "mr_linear": (C.c_int, [_P, C.c_int, C.c_int32, C.c_int64, C.POINTER(DenseWeightDesc), _P, C.c_int, C.c_int64,
                            _P]),
    "mr_mla_decode_block_workspace_size": (C.c_size_t, [C.POINTER(BlockArgs)]),
    "mr_mla_decode_block": (C.c_int, [C.POINTER(BlockArgs), _P]),
    "mr_mla_prefill_workspace_size": (C.c_size_t, [C.POINTER(PrefillArgs)]),
    "mr_mla_prefill": (C.c_int, [C.POINTER(PrefillArgs), _P]),
    "mr_mla_prefill_block_workspace_size": (C.c_size_t, [C.POINTER(PrefillBlockArgs)]),
    "mr_mla_prefill_block": (C.c_int, [C.POINTER(PrefillBlockArgs), _P]),
    "mr_topk_geometry": (C.c_int, [C.c_int32, C.c_int32, C.c_int32, C.c_int32, C.c_int32, C.c_int32, _I32P]),
    "mr_topk_workspace_size": (C.c_size_t, [C.c_int32, C.c_int32, C.c_int32]),
    "mr_topk_select": (C.c_int, [C.POINTER(TopkArgs), _P]),
    "mr_indexer_scores": (C.c_int, [_P, C.c_int, C.c_int32, C.c_int32, C.c_int32, C.c_int64, C.c_int64, _P, C.c_int,
                                    C.c_int32, C.c_int32, C.c_int64, _P, C.c_int, C.c_int32, C.c_int32, C.c_int64,
                                    _P, C.c_int64, _P]),
    "mr_mxfp4_validate": (C.c_int, [C.c_int, C.c_int32, _I64P, C.c_int, C.c_int32, _I64P, _I64P, _I64P, _I64P]),
    "mr_mxfp4_quantize": (C.c_int, [_P, C.c_int, C.c_int64, C.c_int64, C.c_int64, _P, _P, _P]),
    "mr_mxfp4_dequantize": (C.c_int, [C.POINTER(MXFP4Desc), _P, C.c_int, C.c_int64, _P]),
    "mr_mxfp4_matmul": (C.c_int, [_P, C.c_int, C.c_int32, C.c_int64, C.POINTER(MXFP4Desc), _P, C.c_int, C.c_int64, _P]),
    "mr_mxfp4_matmul_quantized": (C.c_int, [C.POINTER(MXFP4Desc), C.POINTER(MXFP4Desc), _P, C.c_int, C.c_int64, _P]),
    "mr_mxfp4_expert_matmul": (C.c_int, [C.POINTER(MXFP4ExpertArgs), _P]),
    "mr_expert_sort_workspace_size": (C.c_size_t, [C.c_int32, C.c_int32, C.c_int32]),
    "mr_expert_sort": (C.c_int, [_P, C.c_int32, C.c_int32, C.c_int32, _P, _P, _P, _P, C.c_size_t, _P]),
    "mr_expert_dispatch": (C.c_int, [_P, C.c_int, C.c_int32, C.c_int64, C.c_int64, _P, C.c_int32, _P, C.c_int64, _P]),
    "mr_expert_combine": (C.c_int, [_P, C.c_int, C.c_int64, C.c_int64, _P, _P, C.c_int32, C.c_int32, _P, C.c_int64,
                                    _P]),
    "mr_expert_combine_backward": (C.c_int, [_P, C.c_int, C.c_int64, C.c_int64, _P, C.c_int64, _P, _P, C.c_int32,
                                             C.c_int32, _P, C.c_int64, _P, _P]),
    "mr_head_norm_rope": (C.c_int, [C.POINTER(HeadNormArgs), _P]),
    "mr_head_norm_rope_backward_workspace_size": (C.c_size_t, [C.POINTER(HeadNormArgs)]),
    "mr_head_norm_rope_backward": (C.c_int, [C.POINTER(HeadNormArgs), _P]),
    "mr_kv_append": (C.c_int, [C.POINTER(KVAppendArgs), _P]),
    "mr_kv_attention_workspace_size": (C.c_size_t, [C.POINTER(KVAttentionArgs)]),
    "mr_kv_attention": (C.c_int, [C.POINTER(KVAttentionArgs), _P]),
    "mr_attention_indices_window": (C.c_int, [C.c_int32, C.c_int32, C.c_int32, _P, _I32P, _I32P]),
    "mr_attention_indices_compressed": (C.c_int, [C.c_int32, C.c_int32, C.c_int32, C.c_int32, _P, _I32P, _I32P]),
}

_lib = None


def load(path: str = LIB_PATH):
    """Load the HIP library (raises if it is not built)."""
    global _lib
    if _lib is None:
        if not os.path.exists(path):
            raise FileNotFoundError(f"{path} is not built: run `python minirun-app_amd/build.py`")
        lib = C.CDLL(path)
        for name, (res, args) in SIGNATURES.items():
            fn = getattr(lib, name)
            fn.restype = res
            fn.argtypes = args
        _lib = lib
    return _lib


def last_error() -> str:
    return load().mr_get_last_error().decode()


def _check(status: int):
    if status != OK:
        raise MRError(status, last_error())


def version() -> str:
    return load().mr_version().decode()


# ------------------------------------------------------------------ torch helpers
_torch_module = None


def _torch():
    global _torch_module
    if _torch_module is None:  # (an import statement costs 0.3 us each time)
        import torch

        _torch_module = torch
    return _torch_module


def _stream(stream):
    """A stream argument as the C-ABI takes it: a torch stream, a raw handle
    (int or c_void_p), or None for torch's current stream."""
    if isinstance(stream, C.c_void_p):
        return stream
    if isinstance(stream, int):
        return C.c_void_p(stream)
    torch = _torch()
    if stream is None:
        stream = torch.cuda.current_stream()
    return C.c_void_p(stream.cuda_stream)


def _ptr(t):
    return None if t is None else C.c_void_p(t.data_ptr())


_dtype_codes = {}


def _dtype_code(dt):
    if not _dtype_codes:
        torch = _torch()
        _dtype_codes.update({torch.bfloat16: BF16, torch.float16: F16, torch.float32: F32})
    return _dtype_codes[dt]


def _need(t, name, dtype=None):
    torch = _torch()
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise TypeError(f"{name} must be a CUDA (HIP) tensor")
    if dtype is not None and t.dtype != dtype:
        raise TypeError(f"{name} must be {dtype}, got {t.dtype}")
    if t.stride(-1) != 1:
        raise ValueError(f"{name} must be contiguous in its last dimension")


def decode_args(q_lat, q_rope, latent, rope_keys, *, scale, indices=None, sinks=None, out=None,
                out_dtype=None, num_splits=0, flags=0, workspace=None, index_status=None):
    """Fill a DecodeArgs from torch tensors.

    q_lat [B,H,R] bf16 (R = kv_rank, 512 for the split kernel, else up to 2048
    on the any-width kernel); q_rope [B,H,dr] bf16 or None; latent [B,N,*] or
    [N,*] bf16 rows (first R columns used); rope_keys likewise (dr columns) or
    None; indices [B,K] int32 or None; sinks [H] f32 or None; index_status
    int32 [B,3] device tensor or None (the device-side index check).
    """
    torch = _torch()
    _need(q_lat, "q_lat", torch.bfloat16)
    if q_lat.dim() == 2:
        q_lat = q_lat.unsqueeze(0)
    B, H, R = q_lat.shape
    rope_dim = 0 if q_rope is None else q_rope.shape[-1]
    if q_rope is not None:
        _need(q_rope, "q_rope", torch.bfloat16)
        if q_rope.dim() == 2:
            q_rope = q_rope.unsqueeze(0)
    _need(latent, "latent", torch.bfloat16)
    lat3 = latent if latent.dim() == 3 else latent.unsqueeze(0)
    lat_bs = lat3.stride(0) if lat3.shape[0] > 1 else (0 if latent.dim() == 2 else lat3.stride(0))
    rk3 = None
    if rope_keys is not None:
        _need(rope_keys, "rope_keys", torch.bfloat16)
        rk3 = rope_keys if rope_keys.dim() == 3 else rope_keys.unsqueeze(0)
    n_ctx = lat3.shape[1]
    if out is None:
        out = torch.empty((B, H, R), dtype=out_dtype or torch.bfloat16, device=q_lat.device)
    a = DecodeArgs()
    a.batch, a.heads, a.n_ctx, a.kv_rank, a.rope_dim = B, H, n_ctx, R, rope_dim
    a.scale = float(scale)
    a.q_lat, a.q_lat_batch_stride, a.q_lat_head_stride = q_lat.data_ptr(), q_lat.stride(0), q_lat.stride(1)
    if q_rope is not None:
        a.q_rope, a.q_rope_batch_stride, a.q_rope_head_stride = q_rope.data_ptr(), q_rope.stride(0), q_rope.stride(1)
    a.latent, a.latent_row_stride, a.latent_batch_stride = lat3.data_ptr(), lat3.stride(1), lat_bs
    if rk3 is not None:
        rk_bs = rk3.stride(0) if rope_keys.dim() == 3 else 0
        a.rope_keys, a.rope_row_stride, a.rope_batch_stride = rk3.data_ptr(), rk3.stride(1), rk_bs
    if indices is not None:
        _need(indices, "indices", torch.int32)
        idx = indices if indices.dim() == 2 else indices.unsqueeze(0)
        if idx.stride(0) != idx.shape[1] and idx.shape[0] > 1:
            raise ValueError("indices must be a contiguous [B, K] tensor")
        if idx.numel() == 0:  # an empty list is still a (non-NULL) sparse request
            idx = torch.full((idx.shape[0], 1), -1, dtype=torch.int32, device=idx.device)
            a._keep = idx
            a.indices, a.n_idx = idx.data_ptr(), 0
        else:
            a.indices, a.n_idx = idx.data_ptr(), idx.shape[1]
    if sinks is not None:
        _need(sinks, "sinks", torch.float32)
        a.sinks = sinks.data_ptr()
    _need(out, "out")
    a.out, a.out_dtype = out.data_ptr(), _dtype_code(out.dtype)
    o3 = out if out.dim() == 3 else out.unsqueeze(0)
    a.out_batch_stride, a.out_head_stride = o3.stride(0), o3.stride(1)
    a.num_splits, a.flags = int(num_splits), int(flags)
    if index_status is not None:
        _need(index_status, "index_status", torch.int32)
        if index_status.numel() < 3 * B or not index_status.is_contiguous():
            raise ValueError("index_status must be a contiguous int32 tensor of at least 3 * batch entries")
        a.index_status = index_status.data_ptr()
    need = load().mr_mla_decode_workspace_size(C.byref(a))
    if workspace is None:
        workspace = torch.empty(max(need, 256), dtype=torch.uint8, device=q_lat.device)
    a.workspace, a.workspace_bytes = workspace.data_ptr(), workspace.numel() * workspace.element_size()
    return a, out, workspace


def mla_decode(q_lat, q_rope, latent, rope_keys, *, scale, indices=None, sinks=None, out=None,
               out_dtype=None, num_splits=0, flags=0, workspace=None, index_status=None, stream=None):
    """Absorbed MLA decode / sparse decode.  Returns the [B,H,512] context.

    With indices, the lists are checked as the reference does: by default
    before the launch (a bad list raises MRError, the call synchronises);
    with an index_status tensor on the device in the same launch (read it
    later: per token (status, position, value)); not at all with
    DECODE_UNCHECKED in flags."""
    a, out, ws = decode_args(q_lat, q_rope, latent, rope_keys, scale=scale, indices=indices, sinks=sinks,
                             out=out, out_dtype=out_dtype, num_splits=num_splits, flags=flags, workspace=workspace,
                             index_status=index_status)
    _check(load().mr_mla_decode(C.byref(a), _stream(stream)))
    return out


def sparse_attention(queries_lat, queries_rope, cache, indices, *, scale, sinks=None, validate=True, **kw):
    """DeepSeekV4SparseAttention.forward over a [B, N, 512+dr] cache (rows
    shared by all heads, K = row[0:512+dr], V = row[0:512]).  validate=False
    skips the index checks (DECODE_UNCHECKED)."""
    lat = cache[..., :512]
    rk = cache[..., 512:] if queries_rope is not None else None
    flags = kw.pop("flags", 0) | (0 if validate else DECODE_UNCHECKED)
    return mla_decode(queries_lat, queries_rope, lat, rk, scale=scale, indices=indices, sinks=sinks,
                      flags=flags, **kw)


def validate_indices(indices, n_rows, stream=None):
    """Returns (status, bad_token, bad_position, message) for an int32 [B, K] tensor."""
    torch = _torch()
    idx = indices if indices.dim() == 2 else indices.unsqueeze(0)
    B, K = idx.shape
    need = load().mr_validate_indices_workspace_size(B, K)
    ws = torch.empty(max(need, 256), dtype=torch.uint8, device=idx.device)
    bt, bp = C.c_int32(-1), C.c_int32(-1)
    st = load().mr_validate_indices(_ptr(idx), B, K, int(n_rows), _ptr(ws), ws.numel(), C.byref(bt), C.byref(bp),
                                    _stream(stream))
    return st, bt.value, bp.value, (last_error() if st != OK else "")


# ------------------------------------------------------------------ affine weights
class AffineWeights:
    """MLXBridge.AffineWeights (AffineWeights.swift:65-157) over device tensors.

    packed: uint32 (torch.int32 storage) [out, in*bits/32]; scales, biases:
    [out, in/group] bf16 / f16 / f32.  Construction validates through
    mr_affine_validate, so the errors are the reference's.
    """

    def __init__(self, packed, scales, biases, group_size=64, bits=4):
        torch = _torch()
        dt = {torch.bfloat16: BF16, torch.float16: F16, torch.float32: F32}
        sdt = dt.get(scales.dtype, 99)
        bdt = dt.get(biases.dtype, 99)
        pdt = U32 if packed.dtype in (torch.int32, torch.uint32) else (F32 if packed.dtype == torch.float32 else 99)
        ps = (C.c_int64 * packed.dim())(*packed.shape)
        ss = (C.c_int64 * scales.dim())(*scales.shape)
        bs = (C.c_int64 * biases.dim())(*biases.shape)
        ex, of, inf = C.c_int64(), C.c_int64(), C.c_int64()
        _check(load().mr_affine_validate(pdt, packed.dim(), ps, sdt, scales.dim(), ss, bdt, biases.dim(), bs,
                                         group_size, bits, C.byref(ex), C.byref(of), C.byref(inf)))
        for t, n in ((packed, "packed"), (scales, "scales"), (biases, "biases")):
            _need(t, n)
            if not t.is_contiguous():
                raise ValueError(f"{n} must be contiguous")
        self.packed, self.scales, self.biases = packed, scales, biases
        self.group_size, self.bits = group_size, bits
        self.experts = ex.value or None
        self.out_features, self.in_features = of.value, inf.value
        self.scale_dtype = sdt

    def desc(self):
        return AffineWeightDesc(self.packed.data_ptr(), self.scales.data_ptr(), self.biases.data_ptr(),
                                self.scale_dtype, self.out_features, self.in_features, self.group_size, self.bits)


FINALIZER = C.CFUNCTYPE(None, C.c_void_p)

# One C callback for every adopted weight's finalizers, alive as long as the
# module: the library calls it with a context id, which names the Python
# finalizer and its argument in _FINALIZERS.  The library may call it on a
# HIP runtime thread after the AdoptedAffineWeights object is gone, so no
# per-object ctypes thunk is ever handed to it.
_FINALIZERS = {}
_FIN_LOCK = threading.Lock()
_FIN_NEXT = [1]


@FINALIZER
def _finalizer_trampoline(ctx):
    with _FIN_LOCK:
        fn, arg = _FINALIZERS.pop(ctx)
    fn(arg)


def _register_finalizer(fn, arg):
    with _FIN_LOCK:
        key = _FIN_NEXT[0]
        _FIN_NEXT[0] += 1
        _FINALIZERS[key] = (fn, arg)
    return key


class AdoptedAffineWeights:
    """AffineWeights.adopting (AffineWeights.swift:159-198): the three buffers
    (device pointers, or pinned host memory the device reads) pass to the
    library with a finalizer each (Python callables of one argument, the
    context value).  Each finalizer runs exactly once, when the last
    reference is released and the named stream has passed every read; a
    failed adoption runs them before raising.  Shapes: packed [experts?, out,
    in*bits/32], scales/biases [experts?, out, in/group]."""

    def __init__(self, packed_ptr, scales_ptr, biases_ptr, scale_dtype, out_features, in_features, *,
                 experts=0, group_size=64, bits=4, finalizers=(None, None, None), contexts=(None, None, None)):
        cb, ctx = [], []
        for f, c in zip(finalizers, contexts):
            if f is None:
                cb.append(None)
                ctx.append(None)
            else:
                cb.append(C.cast(_finalizer_trampoline, _P))
                ctx.append(_register_finalizer(f, c))
        h = _P()
        _check(load().mr_affine_adopt(packed_ptr, scales_ptr, biases_ptr, scale_dtype, experts, out_features,
                                      in_features, group_size, bits, cb[0], ctx[0], cb[1], ctx[1], cb[2], ctx[2],
                                      C.byref(h)))
        self.handle = h.value
        self.out_features, self.in_features = out_features, in_features

    def desc(self):
        d = AffineWeightDesc()
        _check(load().mr_adopted_affine_weight(self.handle, C.byref(d)))
        return d

    def retain(self):
        _check(load().mr_adopted_affine_retain(self.handle))

    def release(self, stream=None):
        """Drop one reference; the last one runs the finalizers behind the
        work on `stream` (a torch stream or a raw handle; None: torch's
        current stream, as for every other call here)."""
        _check(load().mr_adopted_affine_release(self.handle, _stream(stream)))

    def release_now(self):
        """Drop one reference; the last one runs the finalizers before this
        returns (for a weight no GPU work reads any more)."""
        _check(load().mr_adopted_affine_release_now(self.handle))


class DenseWeights:
    """A dense projection weight for k3Linear (Linear.swift:55-57): output-major
    [out, in] bf16 or f32 on the device."""

    def __init__(self, weight):
        torch = _torch()
        _need(weight, "weight")
        if weight.dim() != 2 or weight.dtype not in (torch.bfloat16, torch.float32):
            raise ValueError("a dense weight is a 2-D bf16 or f32 [out_features, in_features] tensor")
        self.weight = weight
        self.out_features, self.in_features = weight.shape

    def desc(self):
        return DenseWeightDesc(self.weight.data_ptr(), _dtype_code(self.weight.dtype), self.out_features,
                               self.in_features, self.weight.stride(0))


def projection(w):
    """ProjectionDesc of an AffineWeights, a DenseWeights, or None (absent)."""
    p = ProjectionDesc()
    if w is None:
        p.kind = PROJ_NONE
    elif isinstance(w, AffineWeights):
        p.kind, p.affine = PROJ_AFFINE, w.desc()
    elif isinstance(w, DenseWeights):
        p.kind, p.dense = PROJ_DENSE, w.desc()
    else:
        raise TypeError("a projection is AffineWeights, DenseWeights or None")
    return p


def linear(x, w: DenseWeights, out_dtype=None, stream=None):
    """k3Linear (Linear.swift:55-57): x [tokens, in] -> x . W^T [tokens, out]."""
    torch = _torch()
    _need(x, "x")
    x2 = x if x.dim() == 2 else x.reshape(1, -1)
    y = torch.empty(x2.shape[0], w.out_features, dtype=out_dtype or x.dtype, device=x.device)
    _check(load().mr_linear(_ptr(x2), _dtype_code(x2.dtype), x2.shape[0], x2.stride(0), C.byref(w.desc()), _ptr(y),
                            _dtype_code(y.dtype), y.stride(0), _stream(stream)))
    return y if x.dim() == 2 else y.reshape(w.out_features)


def affine_dequantize(w: AffineWeights, dtype=None, stream=None):
    """affineDequantize (AffineWeights.swift:328-342): dense [out, in], f32 by default."""
    torch = _torch()
    out = torch.empty(w.out_features, w.in_features, dtype=dtype or torch.float32, device=w.packed.device)
    _check(load().mr_affine_dequantize(C.byref(w.desc()), _ptr(out), _dtype_code(out.dtype), _stream(stream)))
    return out


def affine_mm(x, w: AffineWeights, out_dtype=None, stream=None):
    """affineMM (AffineWeights.swift:239-254): x [tokens, in] -> [tokens, out]."""
    torch = _torch()
    _need(x, "x")
    x2 = x if x.dim() == 2 else x.reshape(1, -1)
    y = torch.empty(x2.shape[0], w.out_features, dtype=out_dtype or x.dtype, device=x.device)
    _check(load().mr_affine_matmul(_ptr(x2), _dtype_code(x2.dtype), x2.shape[0], x2.stride(0), C.byref(w.desc()),
                                   _ptr(y), _dtype_code(y.dtype), y.stride(0), _stream(stream)))
    return y if x.dim() == 2 else y.reshape(w.out_features)


def affine_tile_view(tile_ptr, rows, cols, group=64, bits=4, scale_dtype=BF16):
    """A StorageCore affine tile [packed | scales | biases] (QuantizedTileContainer
    .swift:219-343) as a weight descriptor over its bytes, and the tile size."""
    d = AffineWeightDesc()
    n = C.c_int64()
    _check(load().mr_affine_tile_view(tile_ptr, rows, cols, group, bits, scale_dtype, C.byref(d), C.byref(n)))
    return d, n.value


def affine_gather_mm(x, w: AffineWeights, rhs_indices, out_dtype=None, stream=None):
    """affineGatherMM (AffineWeights.swift:255-318): x [tokens, in], a
    stacked w (experts != None), rhs_indices int32 [tokens, experts_per_token]
    -> [tokens, experts_per_token, out], row (t, j) = W[rhs[t, j]] . x[t].
    The reference's preconditions raise MRError (INVALID_ARGUMENT)."""
    torch = _torch()
    _need(x, "x")
    experts = w.experts or 0
    if x.dim() != 2:
        raise ValueError("x must be [tokens, inFeatures]; this function inserts the broadcast axes itself")
    if rhs_indices.dim() != 2 or rhs_indices.shape[0] != x.shape[0]:
        _check(load().mr_affine_gather_matmul(None, 0, -1, 0, C.byref(w.desc()), max(experts, 1), None, 0, None, 0,
                                              None))  # raises the reference's message
    if rhs_indices.dtype != torch.int32 or not rhs_indices.is_contiguous():
        raise ValueError("rhs_indices must be contiguous int32")
    T, K = rhs_indices.shape
    y = torch.empty(T, K, w.out_features, dtype=out_dtype or x.dtype, device=x.device)
    _check(load().mr_affine_gather_matmul(_ptr(x), _dtype_code(x.dtype), T, x.stride(0) if T else w.in_features,
                                          C.byref(w.desc()), experts, _ptr(rhs_indices), K, _ptr(y),
                                          _dtype_code(y.dtype), _stream(stream)))
    return y


# ------------------------------------------------------------------ MXFP4 and routed experts
_HERE = contextlib.nullcontext()


def _call_stream(device, stream):
    """The stream handle of a call on `device`, and a context in which what the
    call allocates belongs to that stream (None: the current one there)."""
    torch = _torch()
    cuda = torch.cuda
    if stream is None:
        # current_stream(device).cuda_stream without the two Python objects
        # between, which cost 2 of a small call's 10 us; not part of torch's public
        # interface, so not relied on
        raw = getattr(torch._C, "_cuda_getCurrentRawStream", None)
        handle = raw(device.index) if raw else cuda.current_stream(device).cuda_stream
        return handle, _HERE if device.index == cuda.current_device() else cuda.device(device)
    if isinstance(stream, cuda.Stream):
        if stream.device != device:
            raise ValueError(f"the stream is on {stream.device}, the tensors on {device}")
        return stream.cuda_stream, cuda.stream(stream)
    handle = stream.value if isinstance(stream, C.c_void_p) else stream
    s = cuda.ExternalStream(handle, device) if handle else cuda.default_stream(device)
    return handle, cuda.stream(s)


def _same_device(first, *others):
    for t in others:
        if t is not None and t.device != first.device:
            raise ValueError(f"a tensor is on {t.device}, the first on {first.device}")


def _need_whole(t, name, dtype=None):
    """A GPU tensor without gaps (axes of one entry may have any stride)."""
    if not isinstance(t, _torch().Tensor) or not t.is_cuda:
        raise TypeError(f"{name} must be a CUDA (HIP) tensor")
    if dtype is not None and t.dtype != dtype:
        raise TypeError(f"{name} must be {dtype}, got {t.dtype}")
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")


def _rows2d(t, name, shape=None):
    """Row stride of a 2-D tensor with contiguous rows."""
    if not isinstance(t, _torch().Tensor) or not t.is_cuda:
        raise TypeError(f"{name} must be a CUDA (HIP) tensor")
    if t.dim() != 2 or (shape is not None and t.shape != shape):
        raise ValueError(f"{name} must be {'2-D' if shape is None else list(shape)}, got {list(t.shape)}")
    ld, step = t.stride()
    if step != 1 and t.shape[1] != 1:
        raise ValueError(f"{name} must be contiguous in its last dimension")
    return ld if t.shape[0] > 1 else max(ld, t.shape[1])


class MXFP4Weights:
    """MXFP4Weights (MXFP4Weights.swift:36-60) over device tensors: packed
    uint32 (torch.int32 or uint32 storage) [experts?, rows, cols / 8], scales
    uint8 (E8M0) [experts?, rows, cols / 32].  Also the form in which
    activations come out of mxfp4_quantize.  Construction validates through
    mr_mxfp4_validate."""

    def __init__(self, packed, scales):
        torch = _torch()
        pdt = U32 if packed.dtype in (torch.int32, torch.uint32) else 99
        sdt = U8 if scales.dtype == torch.uint8 else 99
        ps = (C.c_int64 * packed.dim())(*packed.shape)
        ss = (C.c_int64 * scales.dim())(*scales.shape)
        ex, rows, cols = C.c_int64(), C.c_int64(), C.c_int64()
        _check(load().mr_mxfp4_validate(pdt, packed.dim(), ps, sdt, scales.dim(), ss, C.byref(ex), C.byref(rows),
                                        C.byref(cols)))
        _need_whole(packed, "packed")
        _need_whole(scales, "scales")
        _same_device(packed, scales)
        self._set(packed, scales, ex.value or None, rows.value, cols.value)

    def _set(self, packed, scales, experts, rows, cols):
        self.packed, self.scales, self.experts, self.rows, self.cols = packed, scales, experts, rows, cols
        self.out_features, self.in_features = rows, cols

    @classmethod
    def _made(cls, packed, scales, experts, rows, cols):
        """Of tensors that this module has just made to fit."""
        w = cls.__new__(cls)
        w._set(packed, scales, experts, rows, cols)
        return w

    def desc(self):
        """One matrix (one expert of a stack)."""
        return MXFP4Desc(self.packed.data_ptr(), self.scales.data_ptr(), self.rows, self.cols)


def mxfp4_quantize(x, stream=None):
    """x [rows, cols] (or a vector, one row; or a stack [experts, rows, cols])
    bf16 or f32 -> MXFP4Weights: per 32 values the power of two that puts the
    largest magnitude into [4, 8) and the nearest e2m1 numbers (ties to even,
    at most 6); a block with a NaN or an infinity is NaN whole."""
    torch = _torch()
    _need(x, "x")
    if x.dim() not in (1, 2, 3):
        raise ValueError(f"x must be [rows, cols], a row or a stack of matrices, got {list(x.shape)}")
    lead, cols = (1,) if x.dim() == 1 else x.shape[:-1], x.shape[-1]
    handle, ctx = _call_stream(x.device, stream)
    with ctx:
        x2 = x if x.dim() == 2 else x.reshape(-1, cols)
        packed = torch.empty((*lead, cols // 8), dtype=torch.int32, device=x.device)
        scales = torch.empty((*lead, cols // 32), dtype=torch.uint8, device=x.device)
        _check(load().mr_mxfp4_quantize(x2.data_ptr(), _dtype_code(x2.dtype), x2.shape[0], cols, _rows2d(x2, "x"),
                                        packed.data_ptr(), scales.data_ptr(), handle))
    if x.dim() == 3 and not lead[0]:
        raise ValueError("a stack needs one matrix at least")
    return MXFP4Weights._made(packed, scales, lead[0] if x.dim() == 3 else None, lead[-1], cols)


def mxfp4_dequantize(w: MXFP4Weights, dtype=None, stream=None):
    """The values that w stands for, f32 by default or bf16, in w's shape."""
    torch = _torch()
    handle, ctx = _call_stream(w.packed.device, stream)
    with ctx:
        out = torch.empty((*w.scales.shape[:-1], w.cols), dtype=dtype or torch.float32, device=w.packed.device)
        d = w.desc()
        d.rows = w.rows * (w.experts or 1)
        _check(load().mr_mxfp4_dequantize(C.byref(d), out.data_ptr(), _dtype_code(out.dtype), w.cols, handle))
    return out


def mxfp4_mm(x, w: MXFP4Weights, out_dtype=None, stream=None):
    """x [tokens, in] (or one row) -> x . W^T [tokens, out], f32 sums.  x is
    bf16 or f32 (16-byte aligned rows; y in its dtype unless out_dtype says
    otherwise), or MXFP4Weights (y in bf16 by default)."""
    torch = _torch()
    if w.experts is not None:
        raise ValueError("mxfp4_mm takes one matrix; mxfp4_expert_mm a stack of experts")
    if isinstance(x, MXFP4Weights):
        if x.experts is not None:
            raise ValueError("x must be one matrix [tokens, in], got a stack")
        _same_device(w.packed, x.packed)
        handle, ctx = _call_stream(w.packed.device, stream)
        with ctx:
            y = torch.empty(x.rows, w.rows, dtype=out_dtype or torch.bfloat16, device=w.packed.device)
            _check(load().mr_mxfp4_matmul_quantized(C.byref(x.desc()), C.byref(w.desc()), y.data_ptr(), _dtype_code(y.dtype),
                                                    w.rows, handle))
        return y
    x2 = x.unsqueeze(0) if x.dim() == 1 else x
    ld = _rows2d(x2, "x")
    if x2.shape[1] != w.cols:
        raise ValueError(f"x has {x2.shape[1]} features, the weight {w.cols}")
    _same_device(w.packed, x)
    handle, ctx = _call_stream(x.device, stream)
    with ctx:
        y = torch.empty(x2.shape[0], w.rows, dtype=out_dtype or x.dtype, device=x.device)
        _check(load().mr_mxfp4_matmul(x2.data_ptr(), _dtype_code(x2.dtype), x2.shape[0], ld, C.byref(w.desc()), y.data_ptr(),
                                      _dtype_code(y.dtype), w.rows, handle))
    return y if x.dim() == 2 else y.reshape(w.rows)


class ExpertOrder:
    """Pairs (token, slot) in expert order, as expert_sort leaves them: offsets
    int32 [experts + 1], pair_of_row int32 [tokens * per_token], row_of_pair
    int32 [tokens, per_token] (-1: no row)."""

    def __init__(self, offsets, pair_of_row, row_of_pair, experts):
        torch = _torch()
        for t, n in ((offsets, "offsets"), (pair_of_row, "pair_of_row"), (row_of_pair, "row_of_pair")):
            _need_whole(t, n, torch.int32)
        _same_device(offsets, pair_of_row, row_of_pair)
        if row_of_pair.dim() != 2 or offsets.numel() != experts + 1 or pair_of_row.numel() != row_of_pair.numel():
            raise ValueError("an order is offsets [experts + 1], pair_of_row [tokens * per_token] and row_of_pair "
                             "[tokens, per_token]")
        self._set(offsets, pair_of_row, row_of_pair, experts)

    def _set(self, offsets, pair_of_row, row_of_pair, experts):
        self.offsets, self.pair_of_row, self.row_of_pair, self.experts = offsets, pair_of_row, row_of_pair, experts
        self.tokens, self.per_token = row_of_pair.shape

    @classmethod
    def _made(cls, offsets, pair_of_row, row_of_pair, experts):
        o = cls.__new__(cls)
        o._set(offsets, pair_of_row, row_of_pair, experts)
        return o


def expert_sort(ids, experts, stream=None):
    """ids int32 [tokens, per_token] -> ExpertOrder: the pairs with an id in
    [0, experts) by expert, inside an expert by pair index; other ids have no
    row."""
    torch = _torch()
    _need_whole(ids, "ids", torch.int32)
    if ids.dim() != 2:
        raise ValueError(f"ids must be [tokens, per_token], got {list(ids.shape)}")
    T, K = ids.shape
    if max(T, K, abs(experts)) > 1 << 30:
        raise ValueError(f"{T} tokens of {K} experts of {experts}")
    handle, ctx = _call_stream(ids.device, stream)
    lib = load()
    with ctx:
        n = lib.mr_expert_sort_workspace_size(T, K, experts)
        head, pairs = max(experts, 0) + 1, T * K
        buf = torch.empty(head + 2 * pairs, dtype=torch.int32, device=ids.device)
        ws = torch.empty(n, dtype=torch.uint8, device=ids.device) if n else None
        at = buf.data_ptr()
        _check(lib.mr_expert_sort(ids.data_ptr(), T, K, experts, at, at + 4 * head, at + 4 * (head + pairs),
                                  ws.data_ptr() if n else None, n, handle))
    part = buf.as_strided  # (a third of three slices' time)
    return ExpertOrder._made(part((head,), (1,)), part((pairs,), (1,), head), part((T, K), (K, 1), head + pairs), experts)


def expert_dispatch(x, order: ExpertOrder, out=None, stream=None):
    """x [tokens, dim] bf16 or f32 -> rows [tokens * per_token, dim] in expert
    order, bit for bit.  Rows past the last of the order are not written (give
    `out` to keep what they hold)."""
    torch = _torch()
    ld = _rows2d(x, "x")
    _same_device(x, order.offsets, out)
    if x.shape[0] != order.tokens:
        raise ValueError(f"x has {x.shape[0]} tokens, the order {order.tokens}")
    shape = (order.tokens * order.per_token, x.shape[1])
    handle, ctx = _call_stream(x.device, stream)
    with ctx:
        rows = torch.empty(shape, dtype=x.dtype, device=x.device) if out is None else out
        if rows.dtype != x.dtype:
            raise TypeError(f"out must be {x.dtype}, got {rows.dtype}")
        _check(load().mr_expert_dispatch(x.data_ptr(), _dtype_code(x.dtype), order.tokens, x.shape[1], ld,
                                         order.row_of_pair.data_ptr(), order.per_token, rows.data_ptr(),
                                         _rows2d(rows, "out", shape), handle))
    return rows


def mxfp4_expert_mm(x, w: MXFP4Weights, order: ExpertOrder, sorted_rows=False, out_dtype=None, out=None, stream=None):
    """Rows in expert order [tokens * per_token, out]: row r is W_e . x of its
    expert e and its token's x (x [tokens, in]), or with sorted_rows of row r of
    x [tokens * per_token, in].  x and the result's dtype as for mxfp4_mm; w is
    a stack.  Rows past the last of the order are not written (give `out` to
    keep what they hold)."""
    torch = _torch()
    if w.experts != order.experts:
        raise ValueError(f"the weight has {w.experts} experts, the order {order.experts}")
    rows = order.tokens * order.per_token
    a = MXFP4ExpertArgs()
    if isinstance(x, MXFP4Weights):
        if x.experts is not None:
            raise ValueError("x must be one matrix, got a stack")
        dtype, shape = out_dtype or torch.bfloat16, (x.rows, x.cols)
        a.x, a.x_dtype, a.x_scales = x.packed.data_ptr(), U32, x.scales.data_ptr()
        _same_device(w.packed, x.packed, order.offsets, out)
    else:
        a.x_stride = _rows2d(x, "x")
        dtype, shape = out_dtype or x.dtype, tuple(x.shape)
        a.x, a.x_dtype = x.data_ptr(), _dtype_code(x.dtype)
        _same_device(w.packed, x, order.offsets, out)
    if shape != (rows if sorted_rows else order.tokens, w.cols):
        raise ValueError(f"x must be {[rows if sorted_rows else order.tokens, w.cols]}, got {list(shape)}")
    handle, ctx = _call_stream(w.packed.device, stream)
    with ctx:
        y = torch.empty(rows, w.rows, dtype=dtype, device=w.packed.device) if out is None else out
        if out is not None and out_dtype is not None and out.dtype != out_dtype:
            raise TypeError(f"out must be {out_dtype}, got {out.dtype}")
        a.x_rows, a.w, a.experts, a.offsets = shape[0], w.desc(), order.experts, order.offsets.data_ptr()
        a.per_token, a.rows = order.per_token, rows
        if not sorted_rows:
            a.pair_of_row = order.pair_of_row.data_ptr()
        a.y_stride = _rows2d(y, "out", (rows, w.rows))
        a.y, a.y_dtype = y.data_ptr(), _dtype_code(y.dtype)
        _check(load().mr_mxfp4_expert_matmul(C.byref(a), handle))
    return y


def _expert_weights(weights, order):
    torch = _torch()
    if weights is None:
        return
    _need_whole(weights, "weights", torch.float32)
    if tuple(weights.shape) != (order.tokens, order.per_token):
        raise ValueError(f"weights must be [{order.tokens}, {order.per_token}], got {list(weights.shape)}")


def expert_combine(rows, order: ExpertOrder, weights=None, stream=None):
    """rows [tokens * per_token, dim] in expert order -> [tokens, dim]: per
    token the sum of its rows times weights f32 [tokens, per_token] (None:
    ones), in f32, rounded once."""
    torch = _torch()
    ld = _rows2d(rows, "rows")
    _expert_weights(weights, order)
    _same_device(rows, order.offsets, weights)
    if rows.shape[0] != order.tokens * order.per_token:
        raise ValueError(f"rows has {rows.shape[0]} rows, the order {order.tokens * order.per_token}")
    handle, ctx = _call_stream(rows.device, stream)
    with ctx:
        out = torch.empty(order.tokens, rows.shape[1], dtype=rows.dtype, device=rows.device)
        _check(load().mr_expert_combine(rows.data_ptr(), _dtype_code(rows.dtype), ld, rows.shape[1],
                                        order.row_of_pair.data_ptr(), (None if weights is None else weights.data_ptr()), order.tokens, order.per_token,
                                        out.data_ptr(), rows.shape[1], handle))
    return out


def expert_combine_backward(d_out, rows, order: ExpertOrder, weights=None, out=None, stream=None):
    """Gradients of expert_combine for d_out [tokens, dim]: (d_rows, in expert
    order; d_weights f32 [tokens, per_token], 0 where a pair has no row).  Rows
    of d_rows past the last of the order are not written (give `out` to keep
    what they hold); rows and d_out have one dtype."""
    torch = _torch()
    ld_g, ld = _rows2d(d_out, "d_out"), _rows2d(rows, "rows")
    _expert_weights(weights, order)
    _same_device(d_out, rows, order.offsets, weights, out)
    shape = (order.tokens * order.per_token, d_out.shape[1])
    if d_out.shape[0] != order.tokens or tuple(rows.shape) != shape or rows.dtype != d_out.dtype:
        raise ValueError(f"d_out must be [{order.tokens}, dim] and rows {list(shape)} of its dtype, got "
                         f"{list(d_out.shape)} and {list(rows.shape)} {rows.dtype}")
    handle, ctx = _call_stream(d_out.device, stream)
    with ctx:
        d_rows = torch.empty(shape, dtype=rows.dtype, device=rows.device) if out is None else out
        if d_rows.dtype != rows.dtype:
            raise TypeError(f"out must be {rows.dtype}, got {d_rows.dtype}")
        d_weights = torch.empty(order.tokens, order.per_token, dtype=torch.float32, device=rows.device)
        _check(load().mr_expert_combine_backward(d_out.data_ptr(), _dtype_code(d_out.dtype), ld_g, d_out.shape[1],
                                                 rows.data_ptr(), ld, order.row_of_pair.data_ptr(), (None if weights is None else weights.data_ptr()),
                                                 order.tokens, order.per_token, d_rows.data_ptr(),
                                                 _rows2d(d_rows, "out", shape), d_weights.data_ptr(), handle))
    return d_rows, d_weights


def expert_dispatch_backward(d_rows, order: ExpertOrder, stream=None):
    """Gradient of expert_dispatch: per token the sum of its rows' gradients."""
    return expert_combine(d_rows, order, None, stream)


# ------------------------------------------------------------------ attention heads and the paged cache
# (Of a small call's 10 us most is Python, about 0.1 us a tensor's attribute and 0.4 a
# nested call, so tensors are checked in one comparison each and structures filled at
# once.)
def _past_int32(what):
    """For numbers that the library takes in 32 bits: ctypes would keep their low half."""
    raise ValueError(f"{what} must be 0 to 2^31 - 1")


def _first_heads(t, name):
    """Shape, device and type of a call's first tensor [tokens, heads, dim]."""
    if not isinstance(t, _torch().Tensor) or not t.is_cuda:
        raise TypeError(f"{name} must be a CUDA (HIP) tensor")
    shape = t.shape
    if len(shape) != 3:
        raise ValueError(f"{name} must be [tokens, heads, dim], got {list(shape)}")
    if (shape[0] | shape[1] | shape[2]) >> 31:
        _past_int32("tokens, heads and dim")
    return shape, t.device, t.dtype


def _heads_like(t, name, shape, device, dtype):
    """Token and head strides of a tensor of this shape (heads None: any), place and type."""
    got = t.shape
    if len(got) != 3 or got[0] != shape[0] or got[2] != shape[2] or (shape[1] is not None and got[1] != shape[1]):
        raise ValueError(f"{name} must be {['any' if n is None else n for n in shape]}, got {list(got)}")
    if t.dtype is not dtype or t.device != device:
        raise TypeError(f"{name} must be {dtype} on {device}, got {t.dtype} on {t.device}")
    ts, hs, step = t.stride()
    if step != 1 and got[2] != 1:
        raise ValueError(f"{name} must be contiguous in its last dimension")
    return ts, hs


def _room(t, dtype):
    """A new tensor of t's shape and place without gaps.  (Where t has none, empty_like takes 1.1 us, empty 1.6.)"""
    if dtype is t.dtype and t.is_contiguous():
        return _torch().empty_like(t)
    return _torch().empty(t.shape, dtype=dtype, device=t.device)


def _vector(t, name, n, device, dtype):
    """The address of a whole vector of n entries; None for None."""
    if t is None:
        return None
    if t.shape != (n,) or t.dtype is not dtype or t.device != device or (n > 1 and t.stride(0) != 1):
        raise ValueError(f"{name} must be a whole {dtype} [{n}] on {device}, got {t.dtype} {list(t.shape)} on {t.device}")
    return t.data_ptr()


def _code(dtype):
    """An mr_dtype; the library refuses what has none."""
    return _dtype_codes.get(dtype, 99) if _dtype_codes else (_dtype_code(_torch().float32), _code(dtype))[1]


def _rotary(device, tokens, cos_t, sin_t, positions, col0, halves):
    """The rotation of `tokens` tokens' heads; no tables: none."""
    if cos_t is None and sin_t is None:
        return Rotary()
    torch = _torch()
    f32 = torch.float32
    if (cos_t is None or sin_t is None or cos_t.dim() != 2 or cos_t.shape != sin_t.shape or cos_t.dtype is not f32
            or sin_t.dtype is not f32 or cos_t.device != device or sin_t.device != device or not cos_t.is_contiguous()
            or not sin_t.is_contiguous()):
        raise ValueError(f"cos_t and sin_t must both be whole float32 [rows, pairs] on {device}")
    rows, half = cos_t.shape
    if (col0 | 2 * half) >> 31:
        _past_int32("col0 and the rotated columns")
    return Rotary(cos_t.data_ptr(), sin_t.data_ptr(), _vector(positions, "positions", tokens, device, torch.int32), rows,
                  2 * half, col0, 1 if halves else 0)


def head_norm_rope(q, k=None, *, q_weight=None, k_weight=None, eps=1e-6, cos_t=None, sin_t=None, positions=None, col0=0,
                   halves=False, out_dtype=None, q_out=None, k_out=None, stream=None):
    """RMSNorm of every head of q [tokens, heads, dim] and k [tokens, kv_heads,
    dim] (bf16 or f32) with the rotation by the tokens' positions: (q, k), or q
    alone without k.  q_weight, k_weight [dim], or None for ones.  cos_t, sin_t
    [rows, n] f32 rotate columns col0 .. col0 + 2 n - 1, token t by row
    positions[t] (int32; None: t), as adjacent pairs or (halves) column i with
    i + n.  q_out, k_out: where to (q and k themselves, for one).  Records nothing
    for autograd: head_norm_rope_backward is the gradient."""
    torch = _torch()
    shape, device, dtype = _first_heads(q, "q")
    T, H, D = shape
    w = q_weight if q_weight is not None else k_weight
    wtype = torch.float32 if w is None else w.dtype
    otype = out_dtype or (dtype if q_out is None else q_out.dtype)
    handle, ctx = _call_stream(device, stream)
    with ctx:
        strides = _heads_like(q, "q", shape, device, dtype)
        y = _room(q, otype) if q_out is None else q_out
        rows_q = HeadRows(H, q.data_ptr(), *strides, _vector(q_weight, "q_weight", D, device, wtype), y.data_ptr(),
                          *((H * D, D) if q_out is None else _heads_like(y, "q_out", shape, device, otype)))
        if k is None:
            if k_weight is not None or k_out is not None:
                raise ValueError("k_weight or k_out without k")
            rows_k = HeadRows()
        else:
            strides = _heads_like(k, "k", (T, None, D), device, dtype)
            z = _room(k, otype) if k_out is None else k_out
            heads = k.shape[1]
            if heads >> 31:
                _past_int32("k's heads")
            rows_k = HeadRows(heads, k.data_ptr(), *strides, _vector(k_weight, "k_weight", D, device, wtype), z.data_ptr(),
                              *((heads * D, D) if k_out is None else _heads_like(z, "k_out", k.shape, device, otype)))
        a = HeadNormArgs(T, D, rows_q, rows_k, _code(dtype), _code(wtype), _code(otype), eps,
                         _rotary(device, T, cos_t, sin_t, positions, col0, halves))
        _check(load().mr_head_norm_rope(C.byref(a), handle))
    return y if k is None else (y, z)


def head_norm_rope_backward(d_q, q, d_k=None, k=None, *, q_weight=None, k_weight=None, eps=1e-6, cos_t=None, sin_t=None,
                            positions=None, col0=0, halves=False, stream=None):
    """Gradients of head_norm_rope for d_q, d_k, those of its outputs (in q's
    dtype): (dq, dk, d_q_weight, d_k_weight), the inputs' in their dtype, the
    weights' f32 [dim] or None without a weight; (dq, d_q_weight) without k."""
    torch = _torch()
    if (d_k is None) != (k is None) or (k is None and k_weight is not None):
        raise ValueError("d_k, k and k_weight go together")
    shape, device, dtype = _first_heads(q, "q")
    T, _, D = shape
    w = q_weight if q_weight is not None else k_weight
    wtype = torch.float32 if w is None else w.dtype
    lib = load()
    handle, ctx = _call_stream(device, stream)
    with ctx:
        made, rows = [], []
        for x, d, weight, name in ((q, d_q, q_weight, "q"), (k, d_k, k_weight, "k")):
            if x is None:
                rows.append(HeadRows())
                continue
            strides = _heads_like(x, name, (T, None, D), device, dtype)
            dx = _room(x, dtype)
            dw = None if weight is None else _room(weight, torch.float32)
            heads = x.shape[1]
            if heads >> 31:
                _past_int32(f"{name}'s heads")
            rows.append(HeadRows(heads, x.data_ptr(), *strides, _vector(weight, f"{name}_weight", D, device, wtype),
                                 dx.data_ptr(), heads * D, D, d.data_ptr(),
                                 *_heads_like(d, f"d_{name}", x.shape, device, dtype), None if dw is None else dw.data_ptr()))
            made.append((dx, dw))
        a = HeadNormArgs(T, D, *rows, _code(dtype), _code(wtype), _code(dtype), eps,
                         _rotary(device, T, cos_t, sin_t, positions, col0, halves))
        if w is not None:
            n = a.workspace_bytes = lib.mr_head_norm_rope_backward_workspace_size(C.byref(a))
            ws = torch.empty(n, dtype=torch.uint8, device=device)
            a.workspace = ws.data_ptr()
        _check(lib.mr_head_norm_rope_backward(C.byref(a), handle))
    return made[0] if k is None else (made[0][0], made[1][0], made[0][1], made[1][1])


class KVCache:
    """One layer's keys and values in pages: k, v [pages, kv_heads, page_size,
    head_dim] bf16, or MXFP4: int32 (or uint32) words [..., head_dim / 8] with
    k_scales, v_scales uint8 [..., head_dim / 32].  page_size is a multiple of 16,
    head_dim one of 32 up to 256; pages may lie apart (their stride, the same for
    k and v), what is inside one may not.  Its attributes stay as they are: calls take
    the tensors' addresses from here, so other tensors are another KVCache."""

    def __setattr__(self, name, value):
        if self.__dict__.get(name, value) is not value:  # (the same one comes back from `cache.k += 1`)
            raise AttributeError(f"{name} of a KVCache stays as it is; make another one of other tensors")
        super().__setattr__(name, value)

    def __init__(self, k, v, k_scales=None, v_scales=None):
        torch = _torch()
        mx = k_scales is not None
        if mx != (v_scales is not None):
            raise ValueError("k_scales and v_scales go together")
        for t, n in ((k, "k"), (v, "v")):
            if t.dim() != 4 or not t.is_cuda:
                raise ValueError(f"{n} must be a CUDA (HIP) tensor [pages, kv_heads, page_size, head_dim], got {list(t.shape)}")
            if t.dtype not in ((torch.int32, torch.uint32) if mx else (torch.bfloat16,)):
                raise TypeError(f"{n} must be {'int32 or uint32 words' if mx else 'bfloat16'}, got {t.dtype}")
        self.k, self.v, self.k_scales, self.v_scales = k, v, k_scales, v_scales
        self.device = k.device
        self.pages, self.kv_heads, self.page_size, last = k.shape
        self.head_dim = 8 * last if mx else last
        d = self.desc = KVCacheDesc()
        d.pages, d.page_size, d.kv_heads, d.head_dim = self.pages, self.page_size, self.kv_heads, self.head_dim
        d.page_stride = self._pages(k, v, "v", k.shape)
        d.k, d.v = k.data_ptr(), v.data_ptr()
        if mx:
            for t, n in ((k_scales, "k_scales"), (v_scales, "v_scales")):
                if not t.is_cuda or t.dtype != torch.uint8:
                    raise TypeError(f"{n} must be a uint8 CUDA (HIP) tensor, got {t.dtype}")
            d.scale_page_stride = self._pages(k_scales, v_scales, "v_scales", (*k.shape[:3], self.head_dim // 32))
            d.k_scales, d.v_scales = k_scales.data_ptr(), v_scales.data_ptr()
        _same_device(k, v, k_scales, v_scales)

    @staticmethod
    def _pages(a, b, name, shape):
        """The two tensors' common page stride."""
        for t in (a, b):
            if tuple(t.shape) != tuple(shape):
                raise ValueError(f"{name} must be {list(shape)}, got {list(t.shape)}")
            if t.shape[0] and not t[0].is_contiguous():
                raise ValueError("a page must be contiguous")
        if a.shape[0] > 1 and a.stride(0) != b.stride(0):
            raise ValueError(f"{name} must have the page stride of its counterpart, {a.stride(0)}, got {b.stride(0)}")
        return a.stride(0)

    @classmethod
    def zeros(cls, pages, kv_heads, page_size, head_dim, mxfp4=False, device="cuda"):
        torch = _torch()
        made = lambda last, dt: [torch.zeros(pages, kv_heads, page_size, last, dtype=dt, device=device) for _ in range(2)]
        if not mxfp4:
            return cls(*made(head_dim, torch.bfloat16))
        return cls(*made(head_dim // 8, torch.int32), *made(head_dim // 32, torch.uint8))

    def values(self, dtype=None, stream=None):
        """(keys, values) of all pages [pages, kv_heads, page_size, head_dim], f32 by default or bf16."""
        torch = _torch()
        dtype = dtype or torch.float32
        if self.k_scales is None:
            with _call_stream(self.k.device, stream)[1]:
                return self.k.to(dtype, copy=True), self.v.to(dtype, copy=True)
        lib, device, n = load(), self.k.device, self.pages * self.kv_heads * self.page_size
        handle, ctx = _call_stream(device, stream)
        with ctx:
            shape = (*self.k.shape[:3], self.head_dim)
            both = torch.empty(shape, dtype=dtype, device=device), torch.empty(shape, dtype=dtype, device=device)
            for out, words, scales in zip(both, (self.k, self.v), (self.k_scales, self.v_scales)):
                if not words.is_contiguous() or not scales.is_contiguous():
                    words, scales = words.contiguous(), scales.contiguous()
                d = MXFP4Desc(words.data_ptr(), scales.data_ptr(), n, self.head_dim)
                _check(lib.mr_mxfp4_dequantize(C.byref(d), out.data_ptr(), _code(dtype), self.head_dim, handle))
        return both


def kv_append(cache: KVCache, k, v, slots, *, normalize=False, norm_weight=None, eps=1e-6, cos_t=None, sin_t=None,
              positions=None, col0=0, halves=False, stream=None):
    """Writes k, v [tokens, kv_heads, head_dim] (bf16 or f32) into the cache's rows
    slots int32 [tokens] (page * page_size + row; outside the pages: passed over),
    the keys normalised first (normalize; norm_weight [head_dim] or None for ones)
    and rotated (as head_norm_rope).  Values are rounded once, to what the cache
    holds.  No two tokens may name one slot."""
    torch = _torch()
    shape, device, dtype = _first_heads(k, "k")
    if device != cache.device:
        raise ValueError(f"k is on {device}, the cache on {cache.device}")
    T = shape[0]
    want = (T, cache.kv_heads, cache.head_dim)
    wtype = torch.float32
    if norm_weight is not None:
        if not normalize:
            raise ValueError("norm_weight needs normalize=True")
        wtype = norm_weight.dtype
    slots_at = _vector(slots, "slots", T, device, torch.int32)
    a = KVAppendArgs(cache.desc, T, k.data_ptr(), v.data_ptr(), _code(dtype), *_heads_like(k, "k", want, device, dtype),
                     *_heads_like(v, "v", want, device, dtype), slots_at, 1 if normalize else 0,
                     _vector(norm_weight, "norm_weight", cache.head_dim, device, wtype), _code(wtype), eps,
                     _rotary(device, T, cos_t, sin_t, positions, col0, halves))
    handle, ctx = _call_stream(device, stream)
    with ctx:
        _check(load().mr_kv_append(C.byref(a), handle))


def kv_attention(q, cache: KVCache, page_table, kv_lens, *, scale, q_offsets=None, max_kv_len=0, window=0, sinks=None,
                 out=None, out_dtype=None, return_lse=False, stream=None):
    """Causal attention of q [tokens, heads, head_dim] bf16 over a paged cache:
    page_table int32 [batch, max_pages], kv_lens int32 [batch]; one token a
    sequence, or sequence b's are q_offsets[b] .. q_offsets[b + 1] - 1 (int32
    [batch + 1]), the last of them at its last key.  window: the last so many keys
    only; sinks f32 [heads]; max_kv_len: about the most keys of a sequence (0: what
    a table row holds, which is slower where that is much more).  out [tokens, heads, head_dim] bf16 (or f32); tokens of no
    sequence are not written (give `out` to keep what they hold).  return_lse: also
    the log of the sum of exp, f32 [tokens, heads]."""
    torch = _torch()
    shape, device, dtype = _first_heads(q, "q")
    if device != cache.device:
        raise ValueError(f"q is on {device}, the cache on {cache.device}")
    T, H, D = shape
    i32 = torch.int32
    if page_table.dim() != 2 or page_table.dtype is not i32 or page_table.device != device:
        raise ValueError(f"page_table must be int32 [batch, max_pages] on {device}, got {page_table.dtype} "
                         f"{list(page_table.shape)} on {page_table.device}")
    B, most = page_table.shape
    if (B | most | window | max_kv_len) >> 31:
        _past_int32("page_table's sizes, window and max_kv_len")
    ld, step = page_table.stride()
    if step != 1 and most > 1:
        raise ValueError("page_table must be contiguous in its last dimension")
    otype = out_dtype or (torch.bfloat16 if out is None else out.dtype)
    lib = load()
    handle, ctx = _call_stream(device, stream)
    with ctx:
        q_strides = _heads_like(q, "q", (T, H, cache.head_dim), device, torch.bfloat16)
        if out is None:
            out, out_strides = _room(q, otype), (H * D, D)
        else:
            out_strides = _heads_like(out, "out", shape, device, otype)
        lse = torch.empty(T, H, dtype=torch.float32, device=device) if return_lse else None
        a = KVAttentionArgs(cache.desc, B, T, H, q.data_ptr(), *q_strides, page_table.data_ptr(), ld,
                            most, _vector(kv_lens, "kv_lens", B, device, i32),
                            _vector(q_offsets, "q_offsets", B + 1, device, i32), max_kv_len, window, scale,
                            _vector(sinks, "sinks", H, device, torch.float32), out.data_ptr(), _code(otype), *out_strides,
                            None if lse is None else lse.data_ptr())
        n = lib.mr_kv_attention_workspace_size(C.byref(a))
        if n:
            ws = torch.empty(n, dtype=torch.uint8, device=device)
            a.workspace, a.workspace_bytes = ws.data_ptr(), n
        _check(lib.mr_kv_attention(C.byref(a), handle))
    return (out, lse) if return_lse else out


def rms_norm(x, weight, eps=1e-6, out_dtype=None, stream=None):
    """K3Norm.rms (Normalization.swift:15-19) over the last axis."""
    torch = _torch()
    _need(x, "x")
    _need(weight, "weight")
    x2 = x.reshape(-1, x.shape[-1])
    out = torch.empty(x2.shape, dtype=out_dtype or x.dtype, device=x.device)
    _check(load().mr_rmsnorm(_ptr(x2), _dtype_code(x2.dtype), x2.shape[0], x2.shape[1], x2.stride(0), _ptr(weight),
                             _dtype_code(weight.dtype), eps, _ptr(out), _dtype_code(out.dtype), out.stride(0),
                             _stream(stream)))
    return out.reshape(x.shape)


def rope_frequencies(dim, base=10000.0, original_len=0, factor=1.0, beta_fast=32.0, beta_slow=1.0):
    import numpy as np

    out = np.empty(dim // 2, np.float64)
    _check(load().mr_rope_frequencies(dim, original_len, base, factor, beta_fast, beta_slow,
                                      out.ctypes.data_as(C.c_void_p)))
    return out


def rope_table(positions, freqs, inverse=False):
    import numpy as np

    pos = np.ascontiguousarray(positions, np.int64)
    half = len(freqs)
    cos = np.empty((pos.size, half), np.float32)
    sin = np.empty((pos.size, half), np.float32)
    _check(load().mr_rope_table(pos.ctypes.data_as(C.c_void_p), pos.size,
                                np.ascontiguousarray(freqs, np.float64).ctypes.data_as(C.c_void_p), half, int(inverse),
                                cos.ctypes.data_as(C.c_void_p), sin.ctypes.data_as(C.c_void_p)))
    return cos, sin


def rope_apply_(x, cos_t, sin_t, col0, dim, stream=None):
    """DeepSeekV4Rotary.apply in place on x [n_pos, inner..., row] (device tables)."""
    _need(x, "x")
    n_pos = x.shape[0]
    inner = 1
    for d in x.shape[1:-1]:
        inner *= d
    _check(load().mr_rope_apply(_ptr(x), _dtype_code(x.dtype), n_pos, inner, x.shape[-1], col0, dim, _ptr(cos_t),
                                _ptr(sin_t), _stream(stream)))
    return x


def mla_cache_append(kv, norm_w, eps, cos_t, sin_t, latent, rope, start_row, kv_rank=512, rope_dim=64, stream=None):
    _need(kv, "kv")
    kv2 = kv.reshape(-1, kv.shape[-1])
    _check(load().mr_mla_cache_append(_ptr(kv2), _dtype_code(kv2.dtype), kv2.stride(0), kv2.shape[0], _ptr(norm_w),
                                      _dtype_code(norm_w.dtype), eps, kv_rank, rope_dim, _ptr(cos_t), _ptr(sin_t),
                                      _ptr(latent), latent.stride(0), _ptr(rope), rope.stride(0), start_row,
                                      _stream(stream)))


def mla_absorb_query(q, heads, nope_dim, v_dim, kv_b, stream=None):
    """q_lat = q_nope . W_UK per head (MLA.swift:180-188); kv_b AffineWeights or DenseWeights."""
    torch = _torch()
    q_lat = torch.empty(heads, 512, dtype=torch.bfloat16, device=q.device)
    _check(load().mr_mla_absorb_query(_ptr(q), q.stride(0), heads, nope_dim, v_dim, C.byref(projection(kv_b)),
                                      _ptr(q_lat), 512, _stream(stream)))
    return q_lat


def mla_unabsorb_values(ctx, heads, nope_dim, v_dim, kv_b, out_dtype=None, stream=None):
    """out = ctx . W_UV^T per head (MLA.swift:196-197); kv_b AffineWeights or DenseWeights."""
    torch = _torch()
    out = torch.empty(heads, v_dim, dtype=out_dtype or torch.bfloat16, device=ctx.device)
    _check(load().mr_mla_unabsorb_values(_ptr(ctx), ctx.stride(0), heads, nope_dim, v_dim, C.byref(projection(kv_b)),
                                         _ptr(out), _dtype_code(out.dtype), _stream(stream)))
    return out


def block_args(x, weights, cache, position, rope_cos, rope_sin, out, *, hidden=7168, q_lora_rank=1536, heads=128,
               nope=128, rope=64, v=128, kv_rank=512, eps=1e-6, scale=None, workspace=None):
    """Fill BlockArgs; `weights` is a dict with input_norm (or None), q_a_norm,
    kv_a_norm (tensors) and q_a, q_b, kv_a, kv_b, o_proj, optional g_proj
    (AffineWeights or DenseWeights).  rope_cos = rope_sin = None: NoPE."""
    torch = _torch()
    a = BlockArgs()
    a.hidden, a.q_lora_rank, a.heads, a.qk_nope_dim, a.qk_rope_dim, a.v_head_dim, a.kv_rank = \
        hidden, q_lora_rank, heads, nope, rope, v, kv_rank
    a.eps = eps
    a.scale = scale if scale is not None else (nope + rope) ** -0.5
    a.x = x.data_ptr()
    a.input_norm_w = weights["input_norm"].data_ptr() if weights.get("input_norm") is not None else None
    a.q_a_norm_w = weights["q_a_norm"].data_ptr()
    a.kv_a_norm_w = weights["kv_a_norm"].data_ptr()
    a.norm_w_dtype = _dtype_code(weights["q_a_norm"].dtype)
    for n in ("q_a", "q_b", "kv_a", "kv_b", "o_proj", "g_proj"):
        setattr(a, n, projection(weights.get(n)))
    a.cache_latent, a.latent_row_stride = cache.data_ptr(), cache.stride(0)
    a.cache_rope, a.rope_row_stride = cache[:, kv_rank:].data_ptr(), cache.stride(0)
    a.position, a.capacity = position, cache.shape[0]
    a.rope_cos = rope_cos.data_ptr() if rope_cos is not None else None
    a.rope_sin = rope_sin.data_ptr() if rope_sin is not None else None
    a.out = out.data_ptr()
    need = load().mr_mla_decode_block_workspace_size(C.byref(a))
    if workspace is None:
        workspace = torch.empty(need, dtype=torch.uint8, device=x.device)
    a.workspace, a.workspace_bytes = workspace.data_ptr(), workspace.numel()
    return a, workspace


def mla_decode_block(x, weights, cache, position, rope_cos, rope_sin, stream=None, **kw):
    """K3MLA.forwardWithoutTrace for one decode token (affine or dense
    projections, optional gate, rotary or NoPE)."""
    torch = _torch()
    out = torch.empty(kw.get("hidden", 7168), dtype=torch.bfloat16, device=x.device)
    a, ws = block_args(x, weights, cache, position, rope_cos, rope_sin, out, **kw)
    _check(load().mr_mla_decode_block(C.byref(a), _stream(stream)))
    return out


def prefill_args(q, latent, rope_keys, kv_b, *, scale=None, out=None, out_dtype=None, workspace=None):
    """Fill PrefillArgs: q [T,H,nope+rope] bf16; latent [P,>=kv_rank] and
    rope_keys [P,>=rope] bf16 row views (both may be views of one cache);
    kv_b [H*(nope+v), kv_rank] bf16 (kv_b_proj, output-major), which fixes
    kv_rank and v_head.  The widths 128 / 64 / 128 / 512 run on MFMA, others
    on the any-width kernels."""
    torch = _torch()
    for t, n in ((q, "q"), (latent, "latent"), (rope_keys, "rope_keys"), (kv_b, "kv_b")):
        _need(t, n, torch.bfloat16)
    T, H, D = q.shape
    P = latent.shape[0]
    nope = D - rope_keys.shape[1]
    a = PrefillArgs()
    a.tokens, a.n_ctx, a.heads = T, P, H
    a.qk_nope_dim, a.qk_rope_dim = nope, rope_keys.shape[1]
    a.v_head_dim, a.kv_rank = kv_b.shape[0] // H - nope, kv_b.shape[1]
    a.scale = scale if scale is not None else D ** -0.5
    a.q, a.q_token_stride, a.q_head_stride = q.data_ptr(), q.stride(0), q.stride(1)
    a.latent, a.latent_row_stride = latent.data_ptr(), latent.stride(0)
    a.rope_keys, a.rope_row_stride = rope_keys.data_ptr(), rope_keys.stride(0)
    a.kv_b, a.kv_b_row_stride = kv_b.data_ptr(), kv_b.stride(0)
    if out is None:
        out = torch.empty(T, H, a.v_head_dim, dtype=out_dtype or torch.bfloat16, device=q.device)
    a.out, a.out_dtype = out.data_ptr(), _dtype_code(out.dtype)
    a.out_token_stride, a.out_head_stride = out.stride(0), out.stride(1)
    need = load().mr_mla_prefill_workspace_size(C.byref(a))
    if workspace is None:
        workspace = torch.empty(need, dtype=torch.uint8, device=q.device)
    a.workspace, a.workspace_bytes = workspace.data_ptr(), workspace.numel()
    a._keep = (q, latent, rope_keys, kv_b, out, workspace)
    return a, out, workspace


def mla_prefill(q, latent, rope_keys, kv_b, *, scale=None, out=None, out_dtype=None, workspace=None, stream=None):
    """K3MLA.forward eager prefill (MLA.swift:159-168,198-206): causal
    attention of the T queries over the P cached rows, per-head keys/values
    up-projected through kv_b."""
    a, out, _ = prefill_args(q, latent, rope_keys, kv_b, scale=scale, out=out, out_dtype=out_dtype,
                             workspace=workspace)
    _check(load().mr_mla_prefill(C.byref(a), _stream(stream)))
    return out


def prefill_block_args(x, weights, cache, position, rope_cos, rope_sin, out, *, q_lora_rank=1536, heads=128,
                       nope=128, rope=64, v=128, kv_rank=512, eps=1e-6, scale=None, workspace=None):
    """Fill PrefillBlockArgs for the T prompt rows of x [T, hidden] (bf16);
    `weights` as for block_args; cache [capacity, kv_rank + rope] bf16, rows
    0 .. position-1 already written; rope_cos / rope_sin [T, rope/2] f32
    tensors (the angles at position .. position+T-1) or None (NoPE)."""
    torch = _torch()
    a = PrefillBlockArgs()
    a.tokens = x.shape[0]
    a.hidden, a.q_lora_rank, a.heads, a.qk_nope_dim, a.qk_rope_dim, a.v_head_dim, a.kv_rank = \
        x.shape[1], q_lora_rank, heads, nope, rope, v, kv_rank
    a.eps = eps
    a.scale = scale if scale is not None else (nope + rope) ** -0.5
    a.x, a.x_token_stride = x.data_ptr(), x.stride(0)
    a.input_norm_w = weights["input_norm"].data_ptr() if weights.get("input_norm") is not None else None
    a.q_a_norm_w = weights["q_a_norm"].data_ptr()
    a.kv_a_norm_w = weights["kv_a_norm"].data_ptr()
    a.norm_w_dtype = _dtype_code(weights["q_a_norm"].dtype)
    for n in ("q_a", "q_b", "kv_a", "kv_b", "o_proj", "g_proj"):
        setattr(a, n, projection(weights.get(n)))
    a.cache_latent, a.latent_row_stride = cache.data_ptr(), cache.stride(0)
    a.cache_rope, a.rope_row_stride = (cache[:, kv_rank:].data_ptr() if rope else None), cache.stride(0)
    a.position, a.capacity = position, cache.shape[0]
    a.rope_cos = rope_cos.data_ptr() if rope_cos is not None else None
    a.rope_sin = rope_sin.data_ptr() if rope_sin is not None else None
    a.out, a.out_token_stride = out.data_ptr(), out.stride(0)
    need = load().mr_mla_prefill_block_workspace_size(C.byref(a))
    if workspace is None:
        workspace = torch.empty(need, dtype=torch.uint8, device=x.device)
    a.workspace, a.workspace_bytes = workspace.data_ptr(), workspace.numel()
    return a, workspace


def mla_prefill_block(x, weights, cache, position, rope_cos, rope_sin, stream=None, **kw):
    """K3MLA.forward over a prompt (MLA.swift:124-229): the T rows of x
    through the block, appending cache rows position .. position+T-1;
    returns out [T, hidden] bf16."""
    torch = _torch()
    out = torch.empty(x.shape[0], x.shape[1], dtype=torch.bfloat16, device=x.device)
    a, ws = prefill_block_args(x, weights, cache, position, rope_cos, rope_sin, out, **kw)
    _check(load().mr_mla_prefill_block(C.byref(a), _stream(stream)))
    return out


def topk_geometry(rows, cols, top_k, ratio, start_pos, offset):
    """The reference's selection-geometry checks (DeepSeekV4Attention.swift:
    590-612); returns the number of keys each row receives."""
    sel = C.c_int32()
    _check(load().mr_topk_geometry(rows, cols, top_k, ratio, start_pos, offset, C.byref(sel)))
    return sel.value


def lightning_index_scores(queries, compressed_keys, head_weights, *, out=None, stream=None):
    """DeepSeekV4LightningIndexer.scores (DeepSeekV4Attention.swift:530-549):
    queries [S, H, D], compressed_keys [T, D], head_weights [S, H] (bf16 or
    f32, weights already scaled) -> f32 [S, T], sum_h w * max(q . k, 0).
    Geometry errors are the reference's (MRError INVALID_SHAPE)."""
    torch = _torch()
    if queries.dim() != 3 or compressed_keys.dim() != 2 or head_weights.dim() != 2:
        # a zero geometry makes the library raise the reference's error
        _check(load().mr_indexer_scores(None, BF16, 0, 0, 0, 0, 0, None, BF16, 0, 0, 0, None, BF16, 0, 0, 0, None, 0,
                                        None))
    S, H, D = queries.shape
    T, KD = compressed_keys.shape
    WR, WC = head_weights.shape
    codes = {torch.bfloat16: BF16, torch.float32: F32}
    for t, n in ((queries, "queries"), (compressed_keys, "compressed_keys"), (head_weights, "head_weights")):
        if t.dtype not in codes:
            raise ValueError(f"{n} must be bf16 or f32")
        if t.numel() and t.stride(-1) != 1:
            raise ValueError(f"{n} must have a unit last-dimension stride")
    if out is None:
        out = torch.empty(max(S, 0), max(T, 0), dtype=torch.float32, device=queries.device)
    _check(load().mr_indexer_scores(queries.data_ptr(), codes[queries.dtype], S, H, D,
                                    queries.stride(0) if S else 0, queries.stride(1) if H else 0,
                                    compressed_keys.data_ptr(), codes[compressed_keys.dtype], T, KD,
                                    compressed_keys.stride(0) if T else 0, head_weights.data_ptr(),
                                    codes[head_weights.dtype], WR, WC, head_weights.stride(0) if WR else 0,
                                    out.data_ptr(), out.stride(0) if out.numel() else max(T, 0), _stream(stream)))
    return out


def lightning_select(scores, top_k, ratio, start_pos, offset, *, check=True, status=None, stream=None):
    """DeepSeekV4LightningIndexer.select on the device: scores [rows, cols]
    f32 -> int32 [rows, selected] (offset + key, -1 past the visible keys).
    check=True synchronises and raises MRError (NONFINITE) on a NaN score,
    as the reference throws."""
    torch = _torch()
    _need(scores, "scores", torch.float32)
    rows, cols = scores.shape
    sel = topk_geometry(rows, cols, top_k, ratio, start_pos, offset)
    out = torch.empty(rows, max(sel, 1), dtype=torch.int32, device=scores.device)
    ws = torch.empty(max(load().mr_topk_workspace_size(rows, cols, top_k), 1), dtype=torch.uint8,
                     device=scores.device)
    a = TopkArgs()
    a.scores, a.score_row_stride, a.rows, a.cols = scores.data_ptr(), scores.stride(0), rows, cols
    a.top_k, a.ratio, a.start_pos, a.offset = top_k, ratio, start_pos, offset
    a.out, a.out_row_stride = out.data_ptr(), out.stride(0)
    a.status = status.data_ptr() if status is not None else None
    a.flags = TOPK_CHECK if check else (0 if status is not None else TOPK_UNCHECKED)
    a.workspace, a.workspace_bytes = ws.data_ptr(), ws.numel()
    _check(load().mr_topk_select(C.byref(a), _stream(stream)))
    return out[:, :sel]


def attention_indices_window(window, seq_len, start_pos):
    import numpy as np

    n = max(seq_len * min(seq_len, window), window, 1)
    out = np.empty(n, np.int32)
    r, c = C.c_int32(), C.c_int32()
    _check(load().mr_attention_indices_window(window, seq_len, start_pos, out.ctypes.data_as(C.c_void_p), C.byref(r),
                                              C.byref(c)))
    return out[: r.value * c.value].reshape(r.value, c.value)


def attention_indices_compressed(ratio, seq_len, start_pos, offset):
    import numpy as np

    width = max(seq_len // max(ratio, 1), (start_pos + 1) // max(ratio, 1), 1)
    out = np.empty(max(seq_len, 1) * width, np.int32)
    r, c = C.c_int32(), C.c_int32()
    _check(load().mr_attention_indices_compressed(ratio, seq_len, start_pos, offset, out.ctypes.data_as(C.c_void_p),
                                                  C.byref(r), C.byref(c)))
    return out[: r.value * c.value].reshape(r.value, c.value)
