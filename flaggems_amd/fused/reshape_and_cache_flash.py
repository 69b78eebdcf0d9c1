"""Scatter of K/V rows into the paged cache
(reference: src/flag_gems/fused/reshape_and_cache_flash.py:61-112)."""
import logging

import torch

from .. import _C

logger = logging.getLogger("flag_gems.fused.reshape_and_cache_flash")


def reshape_and_cache_flash(
    key,  # [num_tokens, num_heads, head_size]
    value,  # [num_tokens, num_heads, head_size]
    key_cache,  # [num_blocks, block_size, num_heads, head_size]
    value_cache,  # [num_blocks, block_size, num_heads, head_size]
    slot_mapping,  # [num_tokens]
    kv_cache_dtype,
    k_scale,
    v_scale,
):
    """A cache of the rows' own type takes their bytes; kv_cache_dtype, k_scale and v_scale are then accepted and ignored,
    as in the reference.  Only the token stride of key/value and the page stride of the caches are consulted:
    the inner [heads, head_size] block of a token must be dense.

    An 8-bit cache (torch.float8_e4m3fn or torch.float8_e5m2, with kv_cache_dtype "auto" or the name of that format, or
    torch.uint8 with "fp8", "fp8_e4m3", which are one format, or "fp8_e5m2") takes clamp(row / scale), a float32 quotient,
    rounded to the nearest value of the format, ties to even; infinities become the largest value, NaN stays NaN.  k_scale /
    v_scale: float32 tensors of one number or one for each head, None for 1.  Rows are fp16, bf16 or fp32.  A slot outside
    the cache is skipped like a negative one; slots must differ."""
    logger.debug("GEMS RESHAPE_AND_CACHE_FLASH")
    if key_cache.dtype in _C.CACHE_8BIT and key.dtype is not key_cache.dtype:
        return _quantize_and_cache(key, value, key_cache, value_cache, slot_mapping, kv_cache_dtype, k_scale, v_scale)
    num_tokens = slot_mapping.size(0)
    num_heads = key.size(1)
    head_size = key.size(2)
    block_size = key_cache.size(1)
    assert key_cache.stride(0) == value_cache.stride(0)
    assert key.dtype == value.dtype == key_cache.dtype == value_cache.dtype, "key/value/cache dtypes must match"
    assert slot_mapping.dtype in (torch.int64, torch.int32), "slot_mapping must be int64 or int32"
    assert slot_mapping.stride(0) == 1 or num_tokens <= 1, "slot_mapping must be contiguous"
    if num_tokens == 0:
        return
    with _C.device_guard(key.device):
        rc = _C.lib().fg_reshape_and_cache_flash(
            key.data_ptr(), value.data_ptr(), key_cache.data_ptr(), value_cache.data_ptr(),
            slot_mapping.data_ptr(), 1 if slot_mapping.dtype == torch.int64 else 0,
            num_tokens, num_heads, head_size, block_size,
            key.stride(0), value.stride(0), key_cache.stride(0), key.element_size(),
            _C.current_stream(key.device),
        )
    _C.check(rc, "fg_reshape_and_cache_flash")


def _quantize_and_cache(key, value, key_cache, value_cache, slot_mapping, kv_cache_dtype, k_scale, v_scale):
    num_tokens, = slot_mapping.shape
    rows, num_heads, head_size = key.shape
    v_rows, v_heads, v_size = value.shape
    num_blocks, block_size, cache_heads, cache_size = key_cache.shape
    dtype, cache_dtype, slot_dtype, index = key.dtype, key_cache.dtype, slot_mapping.dtype, key.get_device()
    assert value_cache.dtype is cache_dtype and value.dtype is dtype, "key/value and their caches must match"
    assert cache_heads == num_heads and cache_size == head_size and value_cache.shape == key_cache.shape, "cache shape"
    assert v_heads == num_heads and v_size == head_size and rows >= num_tokens <= v_rows, "key/value shape"
    assert key.is_cuda, "the tensors must be on a GPU"
    assert slot_dtype is torch.int64 or slot_dtype is torch.int32, "slot_mapping must be int64 or int32"
    assert num_tokens <= 1 or slot_mapping.stride(0) == 1, "slot_mapping must be contiguous"
    token, page = (head_size, 1), (num_heads * head_size, head_size, 1)
    k_strides, v_strides, kc_strides, vc_strides = key.stride(), value.stride(), key_cache.stride(), value_cache.stride()
    assert _C.rows_dense(key, k_strides, token) and _C.rows_dense(value, v_strides, token), "a token's [heads, head_size] block must be dense"
    assert _C.rows_dense(key_cache, kc_strides, page) and _C.rows_dense(value_cache, vc_strides, page), "a page must be dense"
    assert value.get_device() == key_cache.get_device() == value_cache.get_device() == slot_mapping.get_device() == index, "all tensors must be on one device"
    fmt = _C.cache_format(cache_dtype, kv_cache_dtype)
    k_ptr, k_stride = _C.head_scale(k_scale, num_heads, index, "k_scale")
    v_ptr, v_stride = _C.head_scale(v_scale, num_heads, index, "v_scale")
    dtype_id = _C.dtype_id(dtype)
    if num_tokens == 0:
        return
    device = key.device
    with _C.device_guard(device):
        rc = _C.lib().fg_reshape_and_cache_flash_8bit(
            key.data_ptr(), value.data_ptr(), key_cache.data_ptr(), value_cache.data_ptr(),
            slot_mapping.data_ptr(), slot_dtype is torch.int64,
            num_tokens, num_heads, head_size, block_size, num_blocks, k_strides[0], v_strides[0],
            kc_strides[0], vc_strides[0], k_ptr, k_stride, v_ptr, v_stride, dtype_id, fmt,
            _C.current_stream(device),
        )
    if rc:
        _C.check(rc, "fg_reshape_and_cache_flash_8bit")
