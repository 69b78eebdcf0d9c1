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
    table, or not in the cache (which has one page at least), gives zeros."""
    logger.debug("GEMS GATHER_CACHE_FLASH")
    num_blocks, block_size, num_heads, head_size = key_cache.shape
    batch = cu_seqlens.size(0) - 1
    table_rows, table_width = block_table.shape
    cache_dtype, index = key_cache.dtype, key_cache.get_device()
    row_size = num_heads * head_size
    page, row = (row_size, head_size, 1), (head_size, 1)
    k_strides, v_strides, table_strides = key_cache.stride(), value_cache.stride(), block_table.stride()
    assert value_cache.dtype is cache_dtype and value_cache.shape == key_cache.shape, "the caches must match"
    assert _C.rows_dense(key_cache, k_strides, page) and _C.rows_dense(value_cache, v_strides, page), "a page must be dense"
    assert block_table.dtype is torch.int32 and table_rows >= batch, "block_table must be int32 [batch, blocks]"
    assert table_strides[1] == 1 or table_width <= 1, "block_table must have contiguous rows"
    assert cu_seqlens.dtype is torch.int32 and batch >= 0 and cu_seqlens.is_contiguous(), "cu_seqlens must be contiguous int32 [batch + 1]"
    if seq_starts is not None:
        assert seq_starts.dtype is torch.int32 and seq_starts.is_contiguous() and seq_starts.shape == (batch,), "seq_starts must be contiguous int32 [batch]"
    assert key_cache.is_cuda, "the tensors must be on a GPU"
    fmt = _C.cache_format(cache_dtype, kv_cache_dtype)
    if dtype is None:
        given = key if key is not None else value
        dtype = given.dtype if given is not None else torch.bfloat16 if fmt is not None else cache_dtype
    if fmt is None:
        assert dtype is cache_dtype, "a cache of %s is read back as it is" % cache_dtype
        fmt, k_scale, v_scale = _C.CACHE_SAME, None, None
    for t in (value_cache, block_table, cu_seqlens, seq_starts, key, value):
        assert t is None or t.get_device() == index, "all tensors must be on one device"
    k_ptr, k_stride = _C.head_scale(k_scale, num_heads, index, "k_scale")
    v_ptr, v_stride = _C.head_scale(v_scale, num_heads, index, "v_scale")
    dtype_id = _C.dtype_id(dtype)
    device = key_cache.device
    with _C.device_guard(device):
        shape = (num_rows, num_heads, head_size)
        if key is None:
            key, key_row = torch.empty(shape, dtype=dtype, device=device), row_size
        else:
            key_row = _check_output(key, shape, row, dtype)
        if value is None:
            value, value_row = torch.empty(shape, dtype=dtype, device=device), row_size
        else:
            value_row = _check_output(value, shape, row, dtype)
        if num_rows == 0 or batch == 0 or row_size == 0:
            return key, value
        rc = _C.lib().fg_gather_cache_flash(
            key_cache.data_ptr(), value_cache.data_ptr(), key.data_ptr(), value.data_ptr(), block_table.data_ptr(),
            table_strides[0], table_width, cu_seqlens.data_ptr(), None if seq_starts is None else seq_starts.data_ptr(),
            batch, num_rows, num_heads, head_size, block_size, num_blocks, k_strides[0], v_strides[0], key_row, value_row,
            k_ptr, k_stride, v_ptr, v_stride, dtype_id, fmt, _C.current_stream(device),
        )
    if rc:
        _C.check(rc, "fg_gather_cache_flash")
    return key, value


def _check_output(given, shape, row, dtype):
    """The elements between rows of an output that the caller gave."""
    assert given.shape == shape and given.dtype is dtype, "key/value must be [num_rows, heads, head_size] of %s" % dtype
    assert _C.rows_dense(given, given.stride(), row), "a row must be dense"
    assert shape[0] <= 1 or given.stride(0) >= shape[1] * shape[2], "rows must not overlap"
    return max(given.stride(0), shape[1] * shape[2])
