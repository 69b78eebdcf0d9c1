"""Calls of attention over a paged cache that earlier refused calls, very uneven batches or large caches could spoil: what scratch
the wrapper hands over and which launches the library makes.  No GPU; no kernel runs."""
import ctypes

import pytest
import torch

import flag_gems
from flaggems_amd import _C
from test_wrapper_bounds import Harness

E4M3, E5M2 = torch.float8_e4m3fn, torch.float8_e5m2


class Asked:
    """Stands in front of the recording library: sizes come from the real one, and so does the refusal of rows that are not
    16-byte aligned."""

    def __init__(self, recorder, real):
        self.recorder, self.real = recorder, real

    def fg_cache_attn_workspace_bytes(self, packed, index):
        return self.real.fg_cache_attn_workspace_bytes(packed, index)

    def fg_cache_attn_fwd(self, packed, stream):
        self.recorder.fg_cache_attn_fwd(packed, stream)
        return -2 if _C.FgCacheAttnParams.from_buffer_copy(packed).base.q % 16 else 0

    def __getattr__(self, name):
        return getattr(self.recorder, name)


@pytest.fixture
def asked(monkeypatch):
    from flaggems_amd.ops import attention

    real = _C.lib()
    harness = Harness(monkeypatch)
    both = Asked(harness.rec, real)
    monkeypatch.setattr(_C, "lib", lambda: both)
    monkeypatch.setattr(attention, "_cache_attn_scratch", {})
    return harness.rec


def scratch_of(rec):
    return [_C.FgCacheAttnParams.from_buffer_copy(a[0]).base.workspace_bytes for n, a in rec.calls if n == "fg_cache_attn_fwd"]


def test_a_refused_call_leaves_no_answer_behind(asked):
    """q half a piece off is refused; the same sizes, aligned, get the scratch that they would have had without that call."""
    kc, vc = torch.zeros(2, 6, 16, 8, 128).to(E4M3).unbind(0)
    cu, used = torch.arange(4, dtype=torch.int32), torch.full((3,), 50, dtype=torch.int32)
    table = torch.zeros(3, 8192, dtype=torch.int32)
    room = torch.randn(3 * 32 * 128 + 4).bfloat16()

    def attend(at):
        q = room[at:at + 3 * 32 * 128].view(3, 32, 128)
        return flag_gems.flash_attn_varlen_func(q, kc, vc, 1, cu, 131072, seqused_k=used, causal=True, block_table=table)

    assert room.data_ptr() % 16 == 0
    with pytest.raises(RuntimeError):
        attend(4)
    attend(0)
    attend(0)
    refused, first, second = scratch_of(asked)
    assert refused == 0 and first == second > 0


def sizes(total, batch, longest, keys, hq=32, hk=8, dim=128, window=-1, sinks=0, page=16, fmt=_C.CACHE_E4M3, **kw):
    """The parameters of a causal call, with addresses that no kernel will see."""
    c = _C.FgCacheAttnParams()
    p = c.base
    for f in ("q", "k_cache", "v_cache", "out", "cu_seqlens_q", "seqused_k", "block_table"):
        setattr(p, f, 256)
    p.total_q, p.batch, p.Hq, p.Hk, p.D, p.page_size, p.max_seqlen_q, p.max_seqlen_k = total, batch, hq, hk, dim, page, longest, keys
    p.q_row_stride = p.o_row_stride = hq * dim
    p.q_head_stride = p.o_head_stride = dim
    for n in "kv":
        setattr(p, n + "_page_stride", page * hk * dim), setattr(p, n + "_row_stride", hk * dim), setattr(p, n + "_head_stride", dim)
    p.dtype, p.window_left, p.window_right, p.is_causal, p.softmax_scale, p.block_table_stride = _C.FG_BF16, window, -1, 1, 0.1, -(-keys // page)
    c.cache_format, c.num_pages, c.table_width, c.num_sink_tokens = fmt, 1 << 20, -(-keys // page), sinks
    for name, value in kw.items():
        setattr(c if hasattr(c, name) else p, name, value)
    return c


@pytest.mark.parametrize("hq,hk,dim", [(32, 8, 128), (64, 8, 128), (128, 1, 64), (8, 8, 64), (32, 4, 256)])
def test_scratch_stays_small(hq, hk, dim):
    """1 GiB for the ranges of chunks and 52 MB for those of few tokens, whatever the batch: total * (DP + 2) * 4 bytes a range
    and query head."""
    most = 0
    for total in [1, 3, 40, 333, 1000, 2047, 4096, 5001, 8192, 8200, 12000, 16384, 33000, 33279, 100003]:
        for batch in (1, 2, 8, 63, 512):
            for keys in (1, 700, 8192, 131072, 1 << 20):
                for longest in {total, max(1, total // batch), min(total, 4096)}:
                    for window in (-1, 4095):
                        c = sizes(total, batch, longest, keys, hq, hk, dim, window, 4)
                        most = max(most, _C.lib().fg_cache_attn_workspace_bytes(ctypes.byref(c), 0))
    assert 0 < most <= (1 << 30) + 52_000_000


@pytest.fixture(scope="module")
def launched(tmp_path_factory):
    """launched([parameters, ...]): for each call (return code, message, launches), with the scratch that it asks for."""
    import json
    import os
    import subprocess
    import sys

    from flaggems_amd import _C

    where = str(tmp_path_factory.mktemp("recorded"))
    script = os.path.join(os.path.dirname(os.path.abspath(__file__)), "emu", "recorded.py")

    def record(calls):
        for c in calls:
            c.base.workspace_bytes = _C.lib().fg_cache_attn_workspace_bytes(ctypes.byref(c), 0)
            c.base.workspace = 1 << 20 if c.base.workspace_bytes else 0
        spec = [["fg_cache_attn_fwd", bytes(c).hex()] for c in calls]
        run = subprocess.run([sys.executable, script, _C.LIB_PATH, where], input=json.dumps(spec), stdout=subprocess.PIPE, text=True, check=True, timeout=300)
        return [(rc, text, [(name, grid, block, _C.FgCacheAttnParams.from_buffer_copy(bytes.fromhex(arg))) for name, grid, block, arg in launches])
                for rc, text, launches in json.loads(run.stdout)]

    return record


UNEVEN = [dict(total=longest + batch - 1, batch=batch, longest=longest, keys=keys, hq=hq, hk=hk, dim=dim)
          for hq, hk, dim in [(64, 8, 128), (8, 8, 64), (16, 1, 64), (32, 8, 128)] for batch in (1, 64, 512, 4096, 65535)
          for longest in (1000, 32768, 131072, 1 << 20) for keys in (1 << 14, 1 << 20)]


def test_one_long_chunk_among_many_sequences(launched):
    """Grids go by the number of sequences times the longest.  Where that is more than a launch holds, sequences are launched a
    few at a time: no call is refused, and every sequence is in one launch of each kernel that it may need."""
    calls = [sizes(k_scale=1 << 21, v_scale=1 << 22, k_scale_batch_stride=3, v_scale_batch_stride=5, **kw) for kw in UNEVEN]
    several = 0
    for kw, c, (rc, text, launches) in zip(UNEVEN, calls, launched(calls)):
        assert rc == 0, (kw, text)
        assert launches and all(g * b < 1 << 32 for _, grid, block, _ in launches for g, b in zip(grid, block)), kw
        tiles = [a for name, _, _, a in launches if "attn_tile_kernel" in name]
        several += len(tiles) > 1
        at = 0
        for a in tiles:
            assert (a.base.cu_seqlens_q, a.base.seqused_k) == (256 + 4 * at, 256 + 4 * at)
            assert a.base.block_table == 256 + 4 * at * c.base.block_table_stride
            assert (a.k_scale, a.v_scale) == ((1 << 21) + 12 * at, (1 << 22) + 20 * at)
            at += a.base.batch
        assert at == kw["batch"], kw
    assert several > 10


def test_refusals_come_before_any_launch(launched):
    """A single sequence with more row blocks than a launch holds: neither kernel runs."""
    (rc, text, launches), = launched([sizes(total=(1 << 29) + 1, batch=2, longest=1 << 29, keys=1 << 14)])
    assert rc == -2 and "too many" in text and not launches


def test_a_full_card_costs_the_ranges_only(asked, monkeypatch):
    """No memory for the scratch: the call runs without, and the next one of these sizes asks again."""
    from flaggems_amd.ops import attention

    class Full:
        full = True

        def empty(self, *size, **kw):
            if self.full and kw["dtype"] is torch.uint8:
                raise torch.OutOfMemoryError("no room")
            return torch.empty(*size, **kw)

        def __getattr__(self, name):
            return getattr(torch, name)

    card = Full()
    monkeypatch.setattr(attention, "torch", card)
    kc, vc = torch.zeros(2, 6, 16, 8, 128).to(E4M3).unbind(0)
    cu, used = torch.arange(4, dtype=torch.int32), torch.full((3,), 50, dtype=torch.int32)
    q = torch.randn(3, 32, 128).bfloat16()
    for card.full in (True, False, True):
        flag_gems.flash_attn_varlen_func(q, kc, vc, 1, cu, 131072, seqused_k=used, causal=True, block_table=torch.zeros(3, 8192, dtype=torch.int32))
    without, given, again = scratch_of(asked)
    assert without == again == 0 < given


@pytest.mark.parametrize("name", ["int8", "fp8_inc", "fp8_ds_mla", "e4m3", "FP8", "", None])
def test_names_of_no_format_are_refused(asked, name):
    """Not taken for what the cache's own type would be."""
    x, slots = torch.randn(7, 2, 64).half(), torch.arange(7)
    table, cu = torch.zeros(3, 4, dtype=torch.int32), torch.tensor([0, 5, 5, 30], dtype=torch.int32)
    for kind in (E4M3, E5M2, torch.uint8):
        c = torch.zeros(6, 16, 2, 64).to(kind)
        with pytest.raises(ValueError, match="kv_cache_dtype"):
            flag_gems.reshape_and_cache_flash(x, x, c, c.clone(), slots, name, None, None)
        with pytest.raises(ValueError, match="kv_cache_dtype"):
            flag_gems.gather_cache_flash(c, c, table, cu, 30, name)
    assert not asked.calls


@pytest.mark.parametrize("name", ["fp8_inc", "fp8_ds_mla", "fp8e4"])
@pytest.mark.parametrize("kind", [torch.uint8, E4M3])
def test_vllm_hook_refuses_caches_it_does_not_know(monkeypatch, name, kind):
    """kv_cache_dtype names that begin with fp8 and stand for another layout or number format: refused, nothing written."""
    import importlib
    import types

    from flaggems_amd.patches import patch_vllm_all

    seen = []
    monkeypatch.setattr(importlib.import_module("flaggems_amd.fused.reshape_and_cache_flash"), "reshape_and_cache_flash", lambda *a: seen.append(a))
    monkeypatch.setattr(importlib.import_module("flaggems_amd.ops.attention"), "flash_attn_varlen_func", lambda **kw: seen.append(kw))
    one = torch.ones(1)
    layer = types.SimpleNamespace(_q_scale=one, _k_scale=one, _v_scale=one)
    meta = types.SimpleNamespace(num_actual_tokens=3, slot_mapping=None, use_cascade=False, query_start_loc=torch.zeros(3), seq_lens=None,
                                 max_query_len=2, max_seq_len=9, block_table=None, scheduler_metadata=None)
    impl = types.SimpleNamespace(kv_cache_dtype=name, use_irope=False, scale=1.0, alibi_slopes=None, sliding_window=(-1, -1), logits_soft_cap=0)
    x = torch.zeros(3, 2, 64)
    with pytest.raises(NotImplementedError, match=name):
        patch_vllm_all.custom_gems_flash_attention_impl_forward(impl, layer, x, x, x, torch.zeros(2, 4, 16, 2, 64, dtype=torch.uint8).view(kind), meta, output=x)
    assert not seen


def test_the_type_of_either_given_output_decides(asked):
    """An 8-bit cache is read to the type of the outputs that are given, whichever is: bf16 only if none is."""
    c = torch.zeros(6, 16, 2, 64).to(E4M3)
    table, cu = torch.zeros(3, 4, dtype=torch.int32), torch.tensor([0, 5, 5, 30], dtype=torch.int32)
    room = torch.zeros(30, 2, 64)
    for given in (dict(key=room), dict(value=room), dict(key=room, value=room.clone())):
        k, v = flag_gems.gather_cache_flash(c, c, table, cu, 30, **given)
        assert k.dtype == v.dtype == torch.float32
    with pytest.raises(AssertionError, match="num_rows, heads"):
        flag_gems.gather_cache_flash(c, c, table, cu, 30, key=room, value=room.half())
    assert [a[-3] for n, a in asked.calls] == [_C.FG_F32] * 3


def test_offsets_beyond_32_bits_stay_with_64_bit_arithmetic(launched):
    """The chunk kernel counts 16-byte pieces inside a page, and between pages, in 32 bits; pages or strides beyond that (64 GiB)
    are attended over by the kernel that counts in 64."""
    def chunk(page, keys, **kw):
        return sizes(total=600, batch=1, longest=600, keys=keys, page=page, **kw)

    far = [chunk(1 << 26, 1 << 26, hk=16, num_pages=1), chunk((1 << 26) + 1, 1 << 26, num_pages=1), chunk(1 << 13, 1 << 16, k_row_stride=524353 * 16),
           chunk(1 << 13, 1 << 16, v_row_stride=1 << 24), chunk(16, 1 << 16, k_page_stride=1 << 36), chunk(16, 1 << 16, v_page_stride=1 << 37),
           chunk(1 << 12, 1 << 16, fmt=_C.CACHE_SAME, k_row_stride=1 << 24, window=700, sinks=4)]
    near = [chunk(1 << 26, 1 << 26, num_pages=1), chunk(1 << 13, 1 << 16, k_row_stride=524352 * 16), chunk(16, 1 << 16, k_page_stride=(1 << 36) - 16),
            chunk(1 << 12, 1 << 16, fmt=_C.CACHE_SAME, k_row_stride=1 << 23, window=700, sinks=4),
            chunk(16, 1 << 16, v_page_stride=1 << 37, num_pages=1), chunk(1, 1 << 16, k_row_stride=1 << 40)]
    answers = launched(far + near)
    kinds = []
    for i, (rc, text, launches) in enumerate(answers):
        assert rc == 0, (i, text)
        kinds.append({"tile" if "attn_tile" in name else "stream" for name, _, _, _ in launches if "attn_merge" not in name})
    assert kinds == [{"stream"}] * len(far) + [{"tile"}] * len(near)
