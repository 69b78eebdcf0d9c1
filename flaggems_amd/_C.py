"""ctypes binding of libfg_mi355.so, the C-ABI library that holds every gfx950 kernel.

The library links the HIP runtime by soname; torch is imported first so that the runtime torch
already mapped is the one the kernels launch on (two HIP runtimes in one process would not share
streams or allocations).  Nothing here falls back to another implementation: when the library is
missing, or a call fails, the caller gets an exception.
"""
import ctypes
import os
import struct
import threading

import torch

_HERE = os.path.dirname(os.path.abspath(__file__))
# FG_LIB_PATH names another build of the same library (csrc/build.py --variant ... --tag TAG: kernel variants on trial)
LIB_PATH = os.environ.get("FG_LIB_PATH") or os.path.join(_HERE, "libfg_mi355.so")

FG_F16, FG_BF16, FG_F32 = 0, 1, 2
SCHED_AUTO, SCHED_DATA_PARALLEL, SCHED_STREAM_K = 0, 1, 2

CACHE_SAME, CACHE_E4M3, CACHE_E5M2 = 0, 1, 2

_DTYPE_ID = {torch.float16: FG_F16, torch.bfloat16: FG_BF16, torch.float32: FG_F32}

c_i64 = ctypes.c_int64
c_int = ctypes.c_int
c_vp = ctypes.c_void_p
c_f32 = ctypes.c_float
I64x3 = c_i64 * 3


class FgFlashParams(ctypes.Structure):
    """Mirror of struct FgFlashParams in include/fg_mi355.h (field order and widths must match)."""

    _fields_ = [
        ("q", c_vp),
        ("k_cache", c_vp),
        ("v_cache", c_vp),
        ("out", c_vp),
        ("lse", c_vp),
        ("cu_seqlens_q", c_vp),
        ("seqused_k", c_vp),
        ("block_table", c_vp),
        ("alibi_slopes", c_vp),
        ("q_row_stride", c_i64),
        ("q_head_stride", c_i64),
        ("o_row_stride", c_i64),
        ("o_head_stride", c_i64),
        ("k_page_stride", c_i64),
        ("k_row_stride", c_i64),
        ("k_head_stride", c_i64),
        ("v_page_stride", c_i64),
        ("v_row_stride", c_i64),
        ("v_head_stride", c_i64),
        ("block_table_stride", c_i64),
        ("alibi_batch_stride", c_i64),
        ("total_q", c_i64),
        ("batch", ctypes.c_int32),
        ("Hq", ctypes.c_int32),
        ("Hk", ctypes.c_int32),
        ("D", ctypes.c_int32),
        ("page_size", ctypes.c_int32),
        ("max_seqlen_q", ctypes.c_int32),
        ("max_seqlen_k", ctypes.c_int32),
        ("is_causal", ctypes.c_int32),
        ("window_left", ctypes.c_int32),
        ("window_right", ctypes.c_int32),
        ("softmax_scale", c_f32),
        ("softcap", c_f32),
        ("dtype", ctypes.c_int32),
        ("workspace", c_vp),
        ("workspace_bytes", c_i64),
    ]


class FgCacheAttnParams(ctypes.Structure):
    """Mirror of struct FgCacheAttnParams in include/fg_mi355.h."""

    _fields_ = [
        ("base", FgFlashParams),
        ("cache_format", ctypes.c_int32),
        ("num_sink_tokens", ctypes.c_int32),
        ("num_pages", c_i64),
        ("table_width", ctypes.c_int32),
        ("k_scale", c_vp),
        ("v_scale", c_vp),
        ("k_scale_batch_stride", c_i64),
        ("k_scale_head_stride", c_i64),
        ("v_scale_batch_stride", c_i64),
        ("v_scale_head_stride", c_i64),
    ]


# The same struct as one format, native sizes and alignment: packing it is several times faster than setting its fields.
CACHE_ATTN_FORMAT = struct.Struct("@9P13q10i2fiPq2iqi2P4q")
assert CACHE_ATTN_FORMAT.size == ctypes.sizeof(FgCacheAttnParams)

_SIGNATURES = {
    "fg_last_error": (ctypes.c_char_p, []),
    "fg_abi_version": (c_int, []),
    "fg_device_info": (c_int, [c_int, ctypes.POINTER(c_int), ctypes.POINTER(c_int), ctypes.POINTER(c_int)]),
    "fg_mfma_probe": (c_int, [c_vp, c_vp, c_int, c_int, ctypes.POINTER(ctypes.c_double), c_vp]),
    "fg_rms_norm": (c_int, [c_vp, c_vp, c_vp, c_vp, c_i64, c_i64, c_i64, c_i64, c_f32, c_int, c_vp]),
    "fg_fused_add_rms_norm": (c_int, [c_vp, c_vp, c_vp, c_i64, c_i64, c_i64, c_i64, c_f32, c_int, c_vp]),
    "fg_softmax": (c_int, [c_vp, c_vp, c_i64, c_i64, c_i64, c_int, c_int, c_vp]),
    "fg_log_softmax": (c_int, [c_vp, c_vp, c_i64, c_i64, c_i64, c_int, c_int, c_vp]),
    "fg_rope": (
        c_int,
        [c_vp, c_vp, c_vp, c_vp, c_vp, c_vp, c_vp, c_int, c_i64, c_i64, c_int, c_int, c_int,
         ctypes.POINTER(c_i64), ctypes.POINTER(c_i64), ctypes.POINTER(c_i64), ctypes.POINTER(c_i64),
         c_i64, c_i64, c_i64, c_i64, c_int, c_int, c_int, c_vp],
    ),
    "fg_reshape_and_cache_flash": (
        c_int,
        [c_vp, c_vp, c_vp, c_vp, c_vp, c_int, c_i64, c_int, c_int, c_int, c_i64, c_i64, c_i64, c_int, c_vp],
    ),
    "fg_reshape_and_cache": (
        c_int,
        [c_vp, c_vp, c_vp, c_vp, c_vp, c_int, c_i64, c_int, c_int, c_int, c_int, c_i64, c_i64, c_i64, c_int, c_vp],
    ),
    "fg_reshape_and_cache_flash_8bit": (
        c_int,
        [c_vp, c_vp, c_vp, c_vp, c_vp, c_int, c_i64, c_int, c_int, c_int, c_i64, c_i64, c_i64, c_i64, c_i64, c_vp, c_i64,
         c_vp, c_i64, c_int, c_int, c_vp],
    ),
    "fg_gather_cache_flash": (
        c_int,
        [c_vp, c_vp, c_vp, c_vp, c_vp, c_i64, c_int, c_vp, c_vp, c_int, c_i64, c_int, c_int, c_int, c_i64, c_i64, c_i64,
         c_i64, c_i64, c_vp, c_i64, c_vp, c_i64, c_int, c_int, c_vp],
    ),
    "fg_silu_and_mul": (c_int, [c_vp, c_vp, c_vp, c_i64, c_i64, c_i64, c_i64, c_i64, c_int, c_vp]),
    "fg_silu_and_mul_backward": (c_int, [c_vp, c_vp, c_vp, c_vp, c_vp, c_i64, c_i64, c_i64, c_i64, c_i64, c_i64, c_i64,
                                         c_int, c_vp]),
    "fg_softmax_backward": (c_int, [c_vp, c_vp, c_vp, c_i64, c_i64, c_i64, c_int, c_int, c_vp]),
    "fg_log_softmax_backward": (c_int, [c_vp, c_vp, c_vp, c_i64, c_i64, c_i64, c_int, c_int, c_vp]),
    "fg_rms_norm_backward_partial_rows": (c_i64, [c_i64, c_i64, c_int, c_int]),
    "fg_rms_norm_backward": (c_int, [c_vp, c_vp, c_vp, c_vp, c_vp, c_vp, c_i64, c_i64, c_i64, c_int, c_vp]),
    "fg_rms_norm_backward_dw": (c_int, [c_vp, c_i64, c_i64, c_vp, c_int, c_vp]),
    "fg_transpose2d": (c_int, [c_vp, c_vp, c_i64, c_i64, c_i64, c_i64, c_int, c_vp]),
    "fg_reload_options": (None, []),
    "fg_gemm_workspace_layout": (c_int, [c_int, ctypes.POINTER(ctypes.c_size_t), ctypes.POINTER(ctypes.c_size_t)]),
    "fg_stream_capture_id": (c_int, [c_vp, ctypes.POINTER(ctypes.c_ulonglong)]),
    "fg_gemm_workspace_bytes": (ctypes.c_size_t, [c_i64, c_i64, c_i64, c_int, c_int, c_int]),
    "fg_gemm": (
        c_int,
        [c_vp, c_vp, c_vp, c_vp, c_i64, c_i64, c_i64, c_i64, c_i64, c_i64, c_i64, c_i64, c_i64, c_i64, c_i64,
         c_f32, c_f32, c_int, c_int, c_int, c_int, c_vp, ctypes.c_size_t, ctypes.POINTER(c_int), c_vp],
    ),
    "fg_gemm_skinny_static": (
        c_int,
        [c_vp, c_vp, c_vp, c_vp, c_i64, c_i64, c_i64, c_i64, c_i64, c_i64, c_i64, c_i64, c_i64, c_i64, c_i64,
         c_f32, c_f32, c_int, c_int, c_int, c_vp],
    ),
    "fg_bmm": (
        c_int,
        [c_vp, c_vp, c_vp, c_i64, c_i64, c_i64, c_i64, c_i64, c_i64, c_i64, c_i64, c_i64, c_i64, c_i64, c_i64, c_i64,
         c_int, c_vp],
    ),
    "fg_gemm_tile_order": (c_int, [c_int, c_int, c_int, ctypes.POINTER(c_int), ctypes.POINTER(c_int)]),
    "fg_gemm_plan": (
        c_int,
        [c_i64, c_i64, c_i64, c_int, ctypes.POINTER(c_int), ctypes.POINTER(c_int), ctypes.POINTER(ctypes.c_double),
         ctypes.POINTER(c_int), ctypes.POINTER(ctypes.c_double), ctypes.POINTER(c_int)],
    ),
    "fg_streamk_partition": (
        c_int,
        [c_i64, c_i64, c_i64, ctypes.POINTER(c_i64), ctypes.POINTER(c_i64), ctypes.POINTER(c_i64)],
    ),
    "fg_flash_attn_varlen_fwd": (c_int, [ctypes.POINTER(FgFlashParams), c_vp]),
    "fg_flash_attn_workspace_bytes": (ctypes.c_size_t, [ctypes.POINTER(FgFlashParams), c_int]),
    "fg_cache_attn_fwd": (c_int, [c_vp, c_vp]),  # FgCacheAttnParams by reference, or packed bytes
    "fg_cache_attn_workspace_bytes": (ctypes.c_size_t, [c_vp, c_int]),
}

_lib = None
_lock = threading.Lock()


class ExtensionMissing(RuntimeError):
    pass


def lib():
    """The loaded library (loads on first use)."""
    global _lib
    if _lib is not None:
        return _lib
    with _lock:
        if _lib is not None:
            return _lib
        if not os.path.exists(LIB_PATH):
            raise ExtensionMissing(
                "libfg_mi355.so is not built (%s). Build it with `python flaggems_amd/csrc/build.py`; "
                "there is no fallback implementation." % LIB_PATH
            )
        # torch's bundled HIP runtime must already be mapped (import torch above does that); load it
        # by its file name as well so the soname lookup below resolves to the same object.
        hip_rt = os.path.join(os.path.dirname(torch.__file__), "lib", "libamdhip64.so")
        if os.path.exists(hip_rt):
            ctypes.CDLL(hip_rt, mode=ctypes.RTLD_GLOBAL)
        handle = ctypes.CDLL(LIB_PATH)
        for name, (res, args) in _SIGNATURES.items():
            fn = getattr(handle, name)  # AttributeError here means header and library disagree
            fn.restype = res
            fn.argtypes = args
        _lib = handle
    return _lib


def exported_symbols():
    return list(_SIGNATURES)


def last_error():
    return lib().fg_last_error().decode("utf-8", "replace")


def check(rc, what):
    if rc != 0:
        raise RuntimeError("%s failed (code %d): %s" % (what, rc, last_error()))


def dtype_id(dtype):
    try:
        return _DTYPE_ID[dtype]
    except KeyError:
        raise TypeError("dtype %s is not supported by the gfx950 kernels (fp16, bf16, fp32 only)" % dtype)


# 8-bit caches: the format a torch type stands for, and the formats that a kv_cache_dtype names (a cache of plain bytes
# has no type of its own)
_CACHE_FORMAT = {torch.float8_e4m3fn: CACHE_E4M3, torch.float8_e5m2: CACHE_E5M2}
CACHE_8BIT = (torch.float8_e4m3fn, torch.float8_e5m2, torch.uint8)
_CACHE_NAMES = {"fp8": CACHE_E4M3, "fp8_e4m3": CACHE_E4M3, "fp8_e5m2": CACHE_E5M2}


def cache_format(cache_dtype, kv_cache_dtype="auto"):
    """Format id of an 8-bit cache, or None for a cache of any other type."""
    if cache_dtype == torch.uint8:
        if kv_cache_dtype not in _CACHE_NAMES:
            raise ValueError("a cache of bytes needs kv_cache_dtype fp8, fp8_e4m3 or fp8_e5m2, got %r" % (kv_cache_dtype,))
        return _CACHE_NAMES[kv_cache_dtype]
    fmt = _CACHE_FORMAT.get(cache_dtype)
    if fmt is not None and kv_cache_dtype != "auto" and _CACHE_NAMES.get(kv_cache_dtype) != fmt:
        raise ValueError("kv_cache_dtype %r does not fit a cache of %s" % (kv_cache_dtype, cache_dtype))
    return fmt


def head_scale(scale, heads, index, name):
    """(pointer, head stride) of an fp32 scale tensor: one number, or one for each head.  None: no scale (1)."""
    if scale is None:
        return None, 0
    _check_scale(scale, index, name)
    if scale.numel() == 1:
        return scale.data_ptr(), 0
    if scale.shape != (heads,) or scale.stride(0) != 1:
        raise ValueError("%s must hold one number or a contiguous one for each of the %d heads, got shape %s" % (
            name, heads, tuple(scale.shape)))
    return scale.data_ptr(), 1


def sequence_scale(scale, batch, heads, index, name):
    """(pointer, batch stride, head stride) of an fp32 scale tensor that expands to (batch, heads).  None: no scale (1)."""
    if scale is None:
        return 0, 0, 0
    _check_scale(scale, index, name)
    if scale.numel() == 1:
        return scale.data_ptr(), 0, 0
    try:
        full = scale.expand(batch, heads)
    except RuntimeError:
        raise ValueError("%s must expand to (batch, kv heads) = (%d, %d), got shape %s" % (name, batch, heads, tuple(scale.shape)))
    return full.data_ptr(), full.stride(0), full.stride(1)


def _check_scale(scale, index, name):
    if not isinstance(scale, torch.Tensor):
        raise TypeError("%s must be a tensor, got %s" % (name, type(scale).__name__))
    if scale.dtype is not torch.float32 or scale.get_device() != index:
        raise ValueError("%s must be float32 on the device of the other tensors (%d), got %s on %s" % (
            name, index, scale.dtype, scale.device))


def rows_dense(t, strides, inner):
    """Whether t[i] is one dense block for every i; `inner`: the strides of its inner dimensions if it is (sizes of 1 aside)."""
    return strides[1:] == inner or t.numel() == 0 or t[0].is_contiguous()


def supported_dtype(dtype):
    return dtype in _DTYPE_ID


def current_stream(device):
    """Raw handle of torch's current stream on `device` (the launches of this library go there)."""
    index = device.index
    if index is None:
        index = torch.cuda.current_device()
    return torch._C._cuda_getCurrentRawStream(index)


class _NoGuard:
    def __enter__(self):
        return None

    def __exit__(self, *exc):
        return False


_NO_GUARD = _NoGuard()


def device_guard(device):
    """Context that makes `device` current for the library call.  Switching devices costs several
    microseconds per call, as much as a small kernel runs; when the device is current already (the
    usual case) nothing is switched."""
    index = device.index
    if index is None or index == torch.cuda.current_device():
        return _NO_GUARD
    return torch.cuda.device(device)


_dev_info = {}


def device_info(index):
    """(num_cu, lds_bytes, gcn_arch) of a device, cached."""
    if index not in _dev_info:
        a, b, c = c_int(), c_int(), c_int()
        check(lib().fg_device_info(index, ctypes.byref(a), ctypes.byref(b), ctypes.byref(c)), "fg_device_info")
        _dev_info[index] = (a.value, b.value, c.value)
    return _dev_info[index]
