"""flash_attn_varlen_func over a paged KV cache on the gfx950 attention kernel, and the dense
entry points (flash_attention_forward / scaled_dot_product_attention) mapped onto the same kernel.

API shims: src/flag_gems/ops/attention.py:1118-1287 (varlen), :1028-1110 (flash_attention_forward),
:749-769 (scaled_dot_product_attention).  Host checks and parameter preparation: mha_varlan_fwd and
mha_fwd, src/flag_gems/ops/flash_api.py:230-569 and :26-227.
"""
import ctypes
import logging

import torch

from .. import _C

logger = logging.getLogger("flag_gems.ops.attention")


def maybe_contiguous(x):
    return x.contiguous() if x is not None and x.stride(-1) != 1 else x


# The reference's forward returns three tensors that only dropout gives a meaning (philox state, an unused slot, the
# attention probabilities).  Dropout is not part of this path, so they are placeholders: made once per device and
# handed out again, instead of three allocations on every call.
_placeholders = {}


def _dropout_placeholders(device):
    hit = _placeholders.get(device)
    if hit is None:
        hit = _placeholders[device] = (torch.empty((2,), dtype=torch.int64, device=device),
                                       torch.empty((), dtype=torch.int64, device=device),
                                       torch.empty((), device=device))
    return hit


def mha_varlan_fwd(
    q, k, v, out, cu_seqlens_q, cu_seqlens_k, seqused_k, leftpad_k, page_table, alibi_slopes,
    max_seqlen_q, max_seqlen_k, p_dropout, softmax_scale, zero_tensors, is_causal,
    window_size_left, window_size_right, softcap, return_softmax, gen,
):
    """Validation + launch.  Returns (out, q, k, v, lse, philox_args, unused, p) like the reference;
    the last three are placeholders because dropout is not part of the inference path."""
    assert q.is_cuda and k.is_cuda and v.is_cuda
    q_dtype = q.dtype
    assert q_dtype in (torch.float16, torch.bfloat16), "FlashAttention only support fp16 and bf16 data type"
    assert q_dtype == k.dtype
    assert q_dtype == v.dtype
    assert q.stride(-1) == 1, "Input tensor must have contiguous last dimension"
    assert k.stride(-1) == 1, "Input tensor must have contiguous last dimension"
    assert v.stride(-1) == 1, "Input tensor must have contiguous last dimension"
    assert cu_seqlens_q.dtype == torch.int32
    assert cu_seqlens_q.is_contiguous()
    assert cu_seqlens_k.dtype == torch.int32
    assert cu_seqlens_k.is_contiguous()
    assert page_table is not None
    assert page_table.dtype == torch.int32 and page_table.stride(-1) == 1

    total_q, num_heads, head_size = q.size()
    num_heads_k = k.size(2)
    batch_size = cu_seqlens_q.numel() - 1
    block_size = k.size(1)
    num_pages = k.size(0)

    assert k.size() == v.size()
    assert cu_seqlens_q.size() == (batch_size + 1,)
    assert cu_seqlens_k.size() == (batch_size + 1,)
    if out is not None:
        assert out.stride(-1) == 1
        assert out.dtype == q.dtype
        assert out.size() == (total_q, num_heads, head_size)
    assert seqused_k is not None, "the paged kernel takes key lengths from seqused_k"
    assert seqused_k.dtype == torch.int32
    assert seqused_k.is_contiguous()
    assert seqused_k.size() == (batch_size,)

    if max_seqlen_q == 1 and alibi_slopes is None:
        is_causal = False
    if is_causal:
        window_size_right = 0
    if window_size_left >= max_seqlen_k:
        window_size_left = -1
    if window_size_right >= max_seqlen_k:
        window_size_right = -1

    assert leftpad_k is None, "leftpad_k is not supported."
    assert head_size <= 256, "FlashAttention forward only supports head dimension at most 256"
    assert head_size % 8 == 0, "head_size must be a multiple of 8, this is ensured by padding!"
    assert num_heads % num_heads_k == 0, "Number of heads in key/value must divide number of heads in query"
    assert k.shape == (num_pages, block_size, num_heads_k, head_size)
    assert k.stride() == v.stride()
    assert p_dropout == 0, "dropout is not implemented on this path (inference only)"
    assert not return_softmax, "return_softmax needs dropout, which is not implemented"

    if alibi_slopes is not None:
        assert alibi_slopes.device == q.device
        assert alibi_slopes.dtype in (torch.float,)
        assert alibi_slopes.stride(-1) == 1
        assert alibi_slopes.shape == (num_heads,) or alibi_slopes.shape == (batch_size, num_heads)
        alibi_batch_stride = alibi_slopes.stride(0) if alibi_slopes.ndim == 2 else 0
    else:
        alibi_batch_stride = 0

    with _C.device_guard(q.device):
        if out is None:
            out = torch.empty_like(q, dtype=v.dtype)
        lse = torch.empty((num_heads, total_q), dtype=torch.float, device=q.device)
        if zero_tensors:
            out.zero_()
            lse.fill_(float("-inf"))
        if total_q > 0 and batch_size > 0:
            p = _C.FgFlashParams()
            p.q, p.k_cache, p.v_cache, p.out, p.lse = q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), lse.data_ptr()
            p.cu_seqlens_q = cu_seqlens_q.data_ptr()
            p.seqused_k = seqused_k.data_ptr()
            p.block_table = page_table.data_ptr()
            p.alibi_slopes = alibi_slopes.data_ptr() if alibi_slopes is not None else None
            p.q_row_stride, p.q_head_stride, _ = q.stride()
            p.o_row_stride, p.o_head_stride, _ = out.stride()
            p.k_page_stride, p.k_row_stride, p.k_head_stride, _ = k.stride()
            p.v_page_stride, p.v_row_stride, p.v_head_stride, _ = v.stride()
            p.block_table_stride = page_table.stride(0)
            p.alibi_batch_stride = alibi_batch_stride
            p.total_q = total_q
            p.batch, p.Hq, p.Hk, p.D, p.page_size = batch_size, num_heads, num_heads_k, head_size, block_size
            p.max_seqlen_q, p.max_seqlen_k = int(max_seqlen_q), int(max_seqlen_k)
            p.is_causal = 1 if is_causal else 0
            p.window_left, p.window_right = int(window_size_left), int(window_size_right)
            p.softmax_scale = float(softmax_scale)
            p.softcap = float(softcap)
            p.dtype = _C.dtype_id(q.dtype)
            # single-token queries: scratch for the partial results of split key ranges (the reference's
            # out_accum / softmax_lse_accum); the library says how much it wants, zero for prefill shapes
            ws_bytes = _C.lib().fg_flash_attn_workspace_bytes(ctypes.byref(p), q.device.index or 0)
            if ws_bytes > 0:
                ws = torch.empty(ws_bytes, dtype=torch.uint8, device=q.device)
                p.workspace, p.workspace_bytes = ws.data_ptr(), ws_bytes
            rc = _C.lib().fg_flash_attn_varlen_fwd(ctypes.byref(p), _C.current_stream(q.device))
            _C.check(rc, "fg_flash_attn_varlen_fwd")
        philox_args, unused, probs = _dropout_placeholders(q.device)
    return out, q, k, v, lse, philox_args, unused, probs


# Scratch sizes by everything they depend on: sizes, masks, the caches' layout and the device (one library call less for a shape seen before).
# Kept of calls that ran only: the library also answers 0 for parameters that it refuses, for reasons that are not in the key.
_cache_attn_scratch = {}
_INT32_MAX = 2 ** 31 - 1


def cache_attn_fwd(q, k, v, out, cu_seqlens_q, seqused_k, page_table, alibi_slopes, max_seqlen_q, max_seqlen_k,
                   softmax_scale, is_causal, window_size_left, window_size_right, softcap, num_sink_tokens, k_descale,
                   v_descale, return_lse=True):
    """Attention over an 8-bit paged cache, or under a window with sink tokens: validation + launch.  Returns (out, lse);
    lse is None where it is not asked for.  Takes scratch memory for the call, 1.05 GiB at most, and runs without if there is none."""
    assert q.is_cuda and k.is_cuda and v.is_cuda
    dtype, cache_dtype, index = q.dtype, k.dtype, q.get_device()
    assert dtype is torch.bfloat16 or dtype is torch.float16, "FlashAttention only support fp16 and bf16 data type"
    assert v.dtype is cache_dtype
    fmt = _C.cache_format(cache_dtype)
    assert fmt is not None or cache_dtype is dtype, "the cache must hold q's type or 8-bit floats"
    total_q, num_heads, head_size = q.shape
    num_pages, block_size, num_heads_k, cache_size = k.shape
    batch = cu_seqlens_q.size(0) - 1
    assert v.shape == k.shape and cache_size == head_size
    q_row, q_head, q_unit = q.stride()
    k_page, k_row, k_head, k_unit = k.stride()
    v_page, v_row, v_head, v_unit = v.stride()
    assert q_unit == k_unit == v_unit == 1, "Input tensor must have contiguous last dimension"
    assert page_table is not None and page_table.dtype is torch.int32 and page_table.dim() == 2
    table_rows, table_width = page_table.shape
    table_stride, table_unit = page_table.stride()
    assert table_rows >= batch and table_width > 0 and (table_unit == 1 or table_width == 1)
    assert cu_seqlens_q.dtype is torch.int32 and cu_seqlens_q.is_contiguous()
    assert seqused_k is not None, "the paged kernel takes key lengths from seqused_k"
    assert seqused_k.dtype is torch.int32 and seqused_k.is_contiguous() and seqused_k.shape == (batch,)
    assert num_heads % num_heads_k == 0, "Number of heads in key/value must divide number of heads in query"
    assert num_sink_tokens >= 0, "num_sink_tokens must not be negative"
    assert k.get_device() == v.get_device() == page_table.get_device() == cu_seqlens_q.get_device() == seqused_k.get_device() == index and (
        out is None or out.get_device() == index), "all tensors must be on one device"
    if alibi_slopes is not None:
        raise NotImplementedError("alibi_slopes are not supported with an 8-bit cache or sink tokens")
    if out is not None:
        o_row, o_head, o_unit = out.stride()
        assert o_unit == 1 and out.dtype is dtype and out.shape == (total_q, num_heads, head_size)
    else:
        o_row, o_head = num_heads * head_size, head_size
    if fmt is None:
        fmt, k_scale, v_scale = _C.CACHE_SAME, (0, 0, 0), (0, 0, 0)
    else:
        k_scale = _C.sequence_scale(k_descale, batch, num_heads_k, index, "k_descale")
        v_scale = _C.sequence_scale(v_descale, batch, num_heads_k, index, "v_descale")
    device = q.device
    with _C.device_guard(device):
        if out is None:
            out = torch.empty((total_q, num_heads, head_size), dtype=dtype, device=device)
        lse = torch.empty((num_heads, total_q), dtype=torch.float, device=device) if return_lse else None
        if total_q == 0 or batch == 0:
            return out, lse
        sizes = (batch, num_heads, num_heads_k, head_size, block_size, min(max_seqlen_q, _INT32_MAX), min(max_seqlen_k, _INT32_MAX),
                 1 if is_causal else 0, min(max(window_size_left, -1), _INT32_MAX), min(max(window_size_right, -1), _INT32_MAX))
        num_sink_tokens = min(num_sink_tokens, _INT32_MAX)

        def packed(ws, ws_bytes):
            return _C.CACHE_ATTN_FORMAT.pack(
                q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), 0 if lse is None else lse.data_ptr(),
                cu_seqlens_q.data_ptr(), seqused_k.data_ptr(), page_table.data_ptr(), 0,
                q_row, q_head, o_row, o_head, k_page, k_row, k_head, v_page, v_row, v_head, table_stride, 0, total_q,
                *sizes, softmax_scale, softcap, _C.dtype_id(dtype), ws, ws_bytes, fmt, num_sink_tokens, num_pages, table_width,
                k_scale[0], v_scale[0], k_scale[1], k_scale[2], v_scale[1], v_scale[2])

        key = (sizes, total_q, num_sink_tokens, fmt, index, num_pages, k_page, k_row, v_page, v_row)
        ws_bytes = _cache_attn_scratch.get(key)
        if ws_bytes is None:
            ws_bytes = _C.lib().fg_cache_attn_workspace_bytes(packed(0, 0), index)
        ws = None
        if ws_bytes > 0:
            try:
                ws = torch.empty(ws_bytes, dtype=torch.uint8, device=device)
            except torch.OutOfMemoryError:  # up to 1 GiB: the call runs without it, unsplit
                pass
        rc = _C.lib().fg_cache_attn_fwd(packed(0, 0) if ws is None else packed(ws.data_ptr(), ws_bytes), _C.current_stream(device))
        if rc:
            _C.check(rc, "fg_cache_attn_fwd")
        if key not in _cache_attn_scratch:
            if len(_cache_attn_scratch) >= 4096:
                _cache_attn_scratch.clear()
            _cache_attn_scratch[key] = ws_bytes
    return out, lse


def flash_attn_varlen_func(
    q,
    k,
    v,
    max_seqlen_q,
    cu_seqlens_q,
    max_seqlen_k,
    cu_seqlens_k=None,  # only used for non-paged prefill
    seqused_k=None,
    q_v=None,
    dropout_p=0.0,
    softmax_scale=None,
    causal=False,
    window_size=None,
    softcap=0.0,  # 0.0 means deactivated
    alibi_slopes=None,
    deterministic=False,
    return_attn_probs=False,
    block_table=None,
    return_softmax_lse=False,
    out=None,
    # Dummy FA3 arguments
    scheduler_metadata=None,
    q_descale=None,
    k_descale=None,
    v_descale=None,
    num_splits: int = 0,
    fa_version: int = 2,
    num_sink_tokens: int = 0,
):
    """Variable-length attention forward with FA2 semantics over a paged KV cache.

    q: (total_q, nheads, headdim); k, v: (num_pages, page_size, nheads_k, headdim);
    cu_seqlens_q: (batch + 1,) int32; seqused_k: (batch,) int32; block_table: (batch, pages) int32.
    The causal mask is aligned to the bottom right corner; GQA/MQA by head mapping
    (query head h reads KV head h // (nheads // nheads_k)); window_size = (left, right) gives
    sliding-window attention; softcap > 0 applies softcap * tanh(score / softcap); alibi_slopes
    (nheads,) or (batch, nheads) fp32 adds -slope * |i + seqlen_k - seqlen_q - j|.
    Returns out (total_q, nheads, headdim), and the fp32 log-sum-exp (nheads, total_q) as well
    when return_softmax_lse is set.  q_v, deterministic, return_attn_probs, scheduler_metadata
    and, for a cache of q's own type, the descale arguments are accepted and ignored, as in the reference.

    An 8-bit cache (k and v of torch.float8_e4m3fn or torch.float8_e5m2, head dim a multiple of 16; a cache of bytes is
    passed as a view of one of these types) stands for k * k_descale and v * v_descale: float32 tensors that expand to
    (batch, nheads_k), None for 1.  q stays in 16 bits (q_descale must be None).
    num_sink_tokens: the first keys of a sequence stay visible in front of a left window (key j is visible if it lies in the
    window or j < num_sink_tokens, and the causal or right bound admits it); pages outside both are not read and may be gone.
    Neither goes together with alibi_slopes.  A block table entry that is needed and names no page of the cache gives NaN.  An
    infinite or NaN value in V gives NaN or infinities to the queries that see its key and to others that share their block
    of rows; in K, NaN to the queries whose score it makes NaN or +infinity.
    """
    logger.debug("GEMS FLASH_ATTN_VARLEN_FUNC")
    assert cu_seqlens_k is not None or seqused_k is not None, "cu_seqlens_k or seqused_k must be provided"
    assert cu_seqlens_k is None or seqused_k is None, "cu_seqlens_k and seqused_k cannot be provided at the same time"
    assert block_table is None or seqused_k is not None, "seqused_k must be provided if block_table is provided"
    if softmax_scale is None:
        softmax_scale = q.shape[-1] ** (-0.5)
    if window_size is None:
        real_window_size = (-1, -1)
    else:
        assert len(window_size) == 2
        real_window_size = (window_size[0], window_size[1])
    q, k, v = maybe_contiguous(q), maybe_contiguous(k), maybe_contiguous(v)
    if fa_version != 2:
        raise RuntimeError("Only FA2 is implemented.")
    if num_splits > 0:
        raise RuntimeError("num_splits > 0 is not implemented in GEMS.")
    max_seqlen_q = max_seqlen_q.item() if hasattr(max_seqlen_q, "item") else max_seqlen_q
    max_seqlen_k = max_seqlen_k.item() if hasattr(max_seqlen_k, "item") else max_seqlen_k
    left, right = real_window_size
    if k.dtype in _C.CACHE_8BIT or (num_sink_tokens != 0 and left >= 0):
        assert dropout_p == 0, "dropout is not implemented on this path (inference only)"
        if k.dtype in _C.CACHE_8BIT and q_descale is not None:
            raise NotImplementedError("q_descale: the query is not quantized on this path")
        out, softmax_lse = cache_attn_fwd(q, k, v, out, cu_seqlens_q, seqused_k, block_table, alibi_slopes, max_seqlen_q,
                                          max_seqlen_k, softmax_scale, causal, left, right, softcap, num_sink_tokens,
                                          k_descale, v_descale, return_softmax_lse)
        return (out, softmax_lse) if return_softmax_lse else out
    assert num_sink_tokens >= 0, "num_sink_tokens must not be negative"
    out, q, k, v, softmax_lse, *_ = mha_varlan_fwd(
        q, k, v, out, cu_seqlens_q,
        # (the reference passes an uninitialised tensor shaped like cu_seqlens_q here; only its shape and dtype are
        # looked at, so cu_seqlens_q itself serves without an allocation)
        cu_seqlens_q if cu_seqlens_k is None else cu_seqlens_k,
        seqused_k, None, block_table, alibi_slopes, max_seqlen_q, max_seqlen_k, dropout_p,
        softmax_scale, False, causal, real_window_size[0], real_window_size[1], softcap,
        return_softmax_lse and dropout_p > 0, None,
    )
    return (out, softmax_lse) if return_softmax_lse else out


# ---- dense attention on the paged kernel ---------------------------------------------------------------
# A dense K (batch, seqlen_k, heads_k, head_dim) with arbitrary batch / row / head strides IS a paged cache:
# cut every sequence into virtual pages of `page` consecutive rows; page j of sequence b is page number
# b * pages_per_batch_stride + j of a cache whose page stride is page * row_stride.  No byte is copied; the
# kernel never reads a key row at or past seqlen_k, so a last, partial page is fine.  The page size is the
# largest power of two (16..256) that divides the batch stride measured in rows; when there is none
# (a sequence length like 1030) the whole sequence is one page, which the general kernel handles.
_dense_meta = {}


def _page_rows(k, batch):
    """Virtual page size for a dense K, or None when the batch stride is not a whole number of pages."""
    if batch == 1:
        return 64  # no batch stride to respect
    row_stride, batch_stride = k.stride(1), k.stride(0)
    if row_stride <= 0 or batch_stride % row_stride != 0:
        return None
    rows = batch_stride // row_stride
    for page in (256, 128, 64, 32, 16):
        if rows % page == 0:
            return page
    return None


def _dense_tables(device, batch, seqlen_q, seqlen_k, page, pages_per_batch):
    """cu_seqlens_q, seqused_k and the virtual block table of a dense batch (cached per shape)."""
    key = (device.index, batch, seqlen_q, seqlen_k, page, pages_per_batch)
    hit = _dense_meta.get(key)
    if hit is None:
        if len(_dense_meta) > 256:
            _dense_meta.clear()
        cu = torch.arange(batch + 1, dtype=torch.int32, device=device) * seqlen_q
        used = torch.full((batch,), seqlen_k, dtype=torch.int32, device=device)
        npages = max(1, (seqlen_k + page - 1) // page)
        table = (torch.arange(batch, dtype=torch.int32, device=device)[:, None] * pages_per_batch
                 + torch.arange(npages, dtype=torch.int32, device=device)[None, :]).contiguous()
        hit = (cu, used, table)
        _dense_meta[key] = hit
    return hit


def mha_fwd(q, k, v, out, alibi_slopes, p_dropout, softmax_scale, is_causal, window_size_left, window_size_right,
            softcap, return_softmax, disable_splitkv=False):
    """Dense forward, q (batch, seqlen_q, heads, d), k / v (batch, seqlen_k, heads_k, d), any strides with a
    contiguous last dimension (reference: mha_fwd, src/flag_gems/ops/flash_api.py:26-227).  Returns
    (out, q, k, v, lse (batch, heads, seqlen_q) fp32, philox_seed, philox_offset, p) with placeholders for the
    dropout outputs."""
    assert q.is_cuda and k.is_cuda and v.is_cuda
    assert q.dtype in (torch.float16, torch.bfloat16), "FlashAttention only support fp16 and bf16 data type"
    assert q.dtype == k.dtype and q.dtype == v.dtype
    assert q.stride(-1) == 1 and k.stride(-1) == 1 and v.stride(-1) == 1, "Input tensor must have contiguous last dimension"
    batch, seqlen_q, num_heads, head_size = q.shape
    seqlen_k, num_heads_k = k.shape[1], k.shape[2]
    assert k.shape == (batch, seqlen_k, num_heads_k, head_size) and v.shape == k.shape
    assert head_size <= 256 and head_size % 8 == 0, "head dimension must be a multiple of 8 and at most 256"
    assert num_heads % num_heads_k == 0, "Number of heads in key/value must divide number of heads in query"
    assert p_dropout == 0, "dropout is not implemented on this path (inference only)"
    assert not return_softmax, "return_softmax needs dropout, which is not implemented"
    if seqlen_q == 1 and alibi_slopes is None:
        is_causal = False
    if is_causal:
        window_size_right = 0
    if window_size_left >= seqlen_k:
        window_size_left = -1
    if window_size_right >= seqlen_k:
        window_size_right = -1
    if alibi_slopes is not None:
        assert alibi_slopes.dtype == torch.float and alibi_slopes.stride(-1) == 1
        assert alibi_slopes.shape == (num_heads,) or alibi_slopes.shape == (batch, num_heads)
    with _C.device_guard(q.device):
        # rows of q must be equally spaced over the whole batch (row b * seqlen_q + s)
        if batch > 1 and q.stride(0) != seqlen_q * q.stride(1):
            q = q.contiguous()
        # K and V share one virtual block table, so they must share their strides
        if k.stride() != v.stride():
            k, v = k.contiguous(), v.contiguous()
        page = _page_rows(k, batch)
        if page is None:
            page, pages_per_batch, page_stride = max(seqlen_k, 1), 1, k.stride(0)  # one page per sequence
        else:
            pages_per_batch = k.stride(0) // (page * k.stride(1)) if batch > 1 else 0
            page_stride = page * k.stride(1)
        cu, used, table = _dense_tables(q.device, batch, seqlen_q, seqlen_k, page, pages_per_batch)
        if out is None:
            out = torch.empty((batch, seqlen_q, num_heads, head_size), dtype=q.dtype, device=q.device)
        else:
            assert out.shape == (batch, seqlen_q, num_heads, head_size) and out.dtype == q.dtype and out.stride(-1) == 1
            assert batch == 1 or out.stride(0) == seqlen_q * out.stride(1), "out rows must be equally spaced over the batch"
        total_q = batch * seqlen_q
        lse = torch.empty((num_heads, total_q), dtype=torch.float, device=q.device)
        if total_q > 0 and seqlen_k >= 0:
            p = _C.FgFlashParams()
            p.q, p.k_cache, p.v_cache, p.out, p.lse = q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), lse.data_ptr()
            p.cu_seqlens_q, p.seqused_k, p.block_table = cu.data_ptr(), used.data_ptr(), table.data_ptr()
            p.alibi_slopes = alibi_slopes.data_ptr() if alibi_slopes is not None else None
            p.q_row_stride, p.q_head_stride = q.stride(1), q.stride(2)
            p.o_row_stride, p.o_head_stride = out.stride(1), out.stride(2)
            p.k_page_stride, p.k_row_stride, p.k_head_stride = page_stride, k.stride(1), k.stride(2)
            p.v_page_stride, p.v_row_stride, p.v_head_stride = page_stride, v.stride(1), v.stride(2)
            p.block_table_stride = table.stride(0)
            p.alibi_batch_stride = alibi_slopes.stride(0) if alibi_slopes is not None and alibi_slopes.ndim == 2 else 0
            p.total_q = total_q
            p.batch, p.Hq, p.Hk, p.D, p.page_size = batch, num_heads, num_heads_k, head_size, page
            p.max_seqlen_q, p.max_seqlen_k = seqlen_q, seqlen_k
            p.is_causal = 1 if is_causal else 0
            p.window_left, p.window_right = int(window_size_left), int(window_size_right)
            p.softmax_scale = float(softmax_scale)
            p.softcap = float(softcap)
            p.dtype = _C.dtype_id(q.dtype)
            ws_bytes = _C.lib().fg_flash_attn_workspace_bytes(ctypes.byref(p), q.device.index or 0)
            if ws_bytes > 0:
                ws = torch.empty(ws_bytes, dtype=torch.uint8, device=q.device)
                p.workspace, p.workspace_bytes = ws.data_ptr(), ws_bytes
            rc = _C.lib().fg_flash_attn_varlen_fwd(ctypes.byref(p), _C.current_stream(q.device))
            _C.check(rc, "fg_flash_attn_varlen_fwd")
        philox_seed = torch.empty((), dtype=torch.int64, device=q.device)
        philox_offset = torch.empty((), dtype=torch.int64, device=q.device)
        probs = torch.empty((), device=q.device)
    return out, q, k, v, lse.view(num_heads, batch, seqlen_q).permute(1, 0, 2), philox_seed, philox_offset, probs


def flash_attention_forward(
    query, key, value, cumulative_sequence_length_q, cumulative_sequence_length_k, max_q, max_k, dropout_p, is_causal,
    return_debug_mask, *, scale=None, softcap=0.0, window_size_left=None, window_size_right=None, seqused_k=None,
    alibi_slopes=None, disable_splitkv=False,
):
    """aten::_flash_attention_forward for dense batches: query (batch, seqlen_q, heads, d), key / value
    (batch, seqlen_k, heads_k, d); FA2 semantics (causal mask aligned to the bottom right corner).
    Returns (out, lse (batch, heads, seqlen_q), philox_seed, philox_offset, debug_mask)."""
    logger.debug("GEMS FLASH_ATTENTION_FORWARD")
    assert cumulative_sequence_length_q is None and cumulative_sequence_length_k is None, "varlen is not supported yet."
    head_dim_q, head_dim_k, head_dim_v = query.shape[-1], key.shape[-1], value.shape[-1]
    assert head_dim_q == head_dim_k and head_dim_k == head_dim_v
    assert head_dim_k in {16, 32, 64, 96, 128, 192, 256}
    softmax_scale = scale or 1.0 / (head_dim_k ** 0.5)
    left = window_size_left if window_size_left is not None else -1
    right = window_size_right if window_size_right is not None else -1
    out, _, _, _, lse, philox_seed, philox_offset, p = mha_fwd(
        query, key, value, None, alibi_slopes, dropout_p, softmax_scale, is_causal, left, right, softcap,
        return_debug_mask, disable_splitkv=disable_splitkv,
    )
    return out, lse, philox_seed, philox_offset, p


def scaled_dot_product_attention(query, key, value, attn_mask=None, dropout_p=0.0, is_causal=False, scale=None,
                                 enable_gqa=False):
    """torch.nn.functional.scaled_dot_product_attention for (batch, heads, seqlen, d) inputs, forward only.
    Calls with an attention mask, with inputs that require a gradient, or causal with seqlen_q != seqlen_k (where
    torch aligns the mask to the top left corner) go to torch's own implementation."""
    logger.debug("GEMS SCALED DOT PRODUCT ATTENTION")
    head_dim_q, head_dim_k, head_dim_v = query.shape[-1], key.shape[-1], value.shape[-1]
    assert head_dim_q == head_dim_k and head_dim_k == head_dim_v
    assert dropout_p == 0.0, "Currenty only support dropout_p=0.0"
    q_heads, kv_heads = query.shape[1], key.shape[1]
    assert enable_gqa or q_heads == kv_heads, (
        f"q_head_num {q_heads} != kv_head_num {kv_heads}, enable_gqa must be True to support different head numbers."
    )
    needs_grad = torch.is_grad_enabled() and (query.requires_grad or key.requires_grad or value.requires_grad)
    covered = (
        query.dim() == 4 and attn_mask is None and not needs_grad and query.dtype in (torch.float16, torch.bfloat16)
        and head_dim_k % 8 == 0 and head_dim_k <= 256 and (not is_causal or query.shape[2] == key.shape[2])
        and query.is_cuda
    )
    if not covered:
        return torch.nn.functional.scaled_dot_product_attention(
            query, key, value, attn_mask=attn_mask, dropout_p=dropout_p, is_causal=is_causal, scale=scale,
            enable_gqa=enable_gqa,
        )
    sm_scale = scale if scale is not None else 1.0 / (head_dim_k ** 0.5)
    q, k, v = (maybe_contiguous(x).transpose(1, 2) for x in (query, key, value))
    out, *_ = mha_fwd(q, k, v, None, None, 0.0, sm_scale, is_causal, -1, -1, 0.0, False)
    return out.transpose(1, 2)
