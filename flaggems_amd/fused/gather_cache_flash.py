"""Packed rows of sequences read back from the paged cache that reshape_and_cache_flash writes."""
import logging

import torch

from .. import _C

logger = logging.getLogger("flag_gems.fused.gather_cache_flash")


def gather_cache_flash(
    key_cache,  # [num_blocks, block_size, num_heads, head_size]
    value_cache,  # [num_blocks, block_size, num_heads, head_size]
    block_table,  # [batch, max_blocks], int32
    cu_seqlens,  # [batch + 1], int32: the output rows of sequence b are cu_seqlens[b] .. cu_seqlens[b + 1]
    num_rows,  # rows of the outputs, at least cu_seqlens[-1]
    kv_cache_dtype="auto",
    k_scale=None,
    v_scale=None,
    seq_starts=None,  # [batch], int32: position of a sequence's first row, None for 0
    dtype=None,
    key=None,  # [num_rows, num_heads, head_size]
    value=None,
):
    """Returns (key, value): row cu_seqlens[b] + i holds what the cache has for position seq_starts[b] + i of sequence b.

    A cache of fp16, bf16 or fp32 is copied (dtype, if given, is its own).  An 8-bit cache (see reshape_and_cache_flash) is
    read as cache * scale, rounded once to `dtype` (bf16 if neither dtype nor outputs are given).  key / value, if given,
    are written and returned; rows that belong to no sequence are left as they were.  A position whose page is not in the
    table, or not in the cache, gives zeros."""
    logger.debug("GEMS GATHER_CACHE_FLASH")
    num_blocks, block_size, num_heads, head_size = key_cache.shape
    batch = cu_seqlens.numel() - 1
    assert key_cache.dtype == value_cache.dtype and key_cache.shape == value_cache.shape, "the caches must match"
    for t in (key_cache, value_cache):
        assert t[0].is_contiguous() if num_blocks else True, "a page must be dense"
    assert block_table.dtype == torch.int32 and block_table.dim() == 2 and block_table.size(0) >= batch, "block_table must be int32 [batch, blocks]"
    assert block_table.stride(1) == 1 or block_table.size(1) <= 1, "block_table must have contiguous rows"
    assert cu_seqlens.dtype == torch.int32 and cu_seqlens.dim() == 1 and cu_seqlens.is_contiguous() and batch >= 0, "cu_seqlens must be contiguous int32 [batch + 1]"
    if seq_starts is not None:
        assert seq_starts.dtype == torch.int32 and seq_starts.is_contiguous() and seq_starts.shape == (batch,), "seq_starts must be contiguous int32 [batch]"
    fmt = _C.cache_format(key_cache.dtype, kv_cache_dtype)
    if dtype is None:
        dtype = key.dtype if key is not None else torch.bfloat16 if fmt is not None else key_cache.dtype
    if fmt is None:
        assert dtype == key_cache.dtype, "a cache of %s is read back as it is" % key_cache.dtype
        fmt, k_scale, v_scale = _C.CACHE_SAME, None, None
    for t in (value_cache, block_table, cu_seqlens, seq_starts, key, value):
        assert t is None or t.device == key_cache.device, "all tensors must be on one device"
    k_ptr, k_stride = _C.head_scale(k_scale, num_heads, key_cache.device, "k_scale")
    v_ptr, v_stride = _C.head_scale(v_scale, num_heads, key_cache.device, "v_scale")
    dtype_id = _C.dtype_id(dtype)
    with _C.device_guard(key_cache.device):
        key, value = (torch.empty((num_rows, num_heads, head_size), dtype=dtype, device=key_cache.device) if t is None else t
                      for t in (key, value))
        for t in (key, value):
            assert t.shape == (num_rows, num_heads, head_size) and t.dtype == dtype, "key/value must be [num_rows, heads, head_size] of %s" % dtype
            assert t[0].is_contiguous() if num_rows else True, "a row must be dense"
            assert num_rows <= 1 or t.stride(0) >= num_heads * head_size, "rows must not overlap"
        if num_rows == 0 or batch == 0 or num_heads * head_size == 0:
            return key, value
        rc = _C.lib().fg_gather_cache_flash(
            key_cache.data_ptr(), value_cache.data_ptr(), key.data_ptr(), value.data_ptr(), block_table.data_ptr(),
            block_table.stride(0), block_table.size(1), cu_seqlens.data_ptr(),
            seq_starts.data_ptr() if seq_starts is not None else None, batch, num_rows, num_heads, head_size, block_size,
            num_blocks, key_cache.stride(0), value_cache.stride(0),
            max(key.stride(0), num_heads * head_size), max(value.stride(0), num_heads * head_size),
            k_ptr, k_stride, v_ptr, v_stride, dtype_id, fmt, _C.current_stream(key_cache.device),
        )
    _C.check(rc, "fg_gather_cache_flash")
    return key, value
