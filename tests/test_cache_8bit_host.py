"""Host side of the 8-bit paged cache, of reading it back and of attention over it or under a window with sink tokens: what the
entry points refuse, and what the wrappers hand over the C ABI.  No GPU, no kernel is launched."""
import ctypes
import types

import pytest
import torch

import flag_gems
from flaggems_amd import _C
from oracle import torch_ref as O
from test_wrapper_bounds import Harness

E4M3, E5M2 = torch.float8_e4m3fn, torch.float8_e5m2


class Calls(Harness):
    """Checks the footprints of the calls as the header describes them."""

    def chk_fg_reshape_and_cache_flash_8bit(self, key, value, kc, vc, slots, i64, n, H, D, bs, blocks, ks, vs, kbs, vbs, ksc, kss, vsc, vss, dtype, fmt, stream):
        e = {_C.FG_F16: 2, _C.FG_BF16: 2, _C.FG_F32: 4}[dtype]
        self.inside("key", key, e, [(n, ks), (H * D, 1)])
        self.inside("value", value, e, [(n, vs), (H * D, 1)])
        self.inside("key cache", kc, 1, [(blocks, kbs), (bs * H * D, 1)])
        self.inside("value cache", vc, 1, [(blocks, vbs), (bs * H * D, 1)])
        self.inside("slots", slots, 8 if i64 else 4, [(n, 1)])
        self.inside("k_scale", ksc, 4, [(H, kss)])
        self.inside("v_scale", vsc, 4, [(H, vss)])

    def chk_fg_gather_cache_flash(self, kc, vc, key, value, table, ts, width, cu, starts, batch, rows, H, D, ps, pages, kps, vps, ks, vs, ksc, kss, vsc, vss,
                                  dtype, fmt, stream):
        e = {_C.FG_F16: 2, _C.FG_BF16: 2, _C.FG_F32: 4}[dtype]
        c = e if fmt == _C.CACHE_SAME else 1
        self.inside("key cache", kc, c, [(pages, kps), (ps * H * D, 1)])
        self.inside("value cache", vc, c, [(pages, vps), (ps * H * D, 1)])
        self.inside("key", key, e, [(rows, ks), (H * D, 1)])
        self.inside("value", value, e, [(rows, vs), (H * D, 1)])
        self.inside("table", table, 4, [(batch, ts), (width, 1)])
        self.inside("cu", cu, 4, [(batch + 1, 1)])
        self.inside("starts", starts, 4, [(batch, 1)])
        self.inside("k_scale", ksc, 4, [(H, kss)])
        self.inside("v_scale", vsc, 4, [(H, vss)])

    def chk_fg_cache_attn_fwd(self, packed, stream):
        c = _C.FgCacheAttnParams.from_buffer_copy(packed)
        p = c.base
        e = 2 if c.cache_format == _C.CACHE_SAME else 1
        self.inside("q", p.q, 2, [(p.total_q, p.q_row_stride), (p.Hq, p.q_head_stride), (p.D, 1)])
        self.inside("out", p.out, 2, [(p.total_q, p.o_row_stride), (p.Hq, p.o_head_stride), (p.D, 1)])
        self.inside("lse", p.lse, 4, [(p.Hq * p.total_q, 1)])
        for name in "kv":
            self.inside(name, getattr(p, name + "_cache"), e, [(c.num_pages, getattr(p, name + "_page_stride")), (p.page_size, getattr(p, name + "_row_stride")),
                                                               (p.Hk, getattr(p, name + "_head_stride")), (p.D, 1)])
            self.inside(name + "_scale", getattr(c, name + "_scale"), 4, [(p.batch, getattr(c, name + "_scale_batch_stride")),
                                                                          (p.Hk, getattr(c, name + "_scale_head_stride"))])
        self.inside("table", p.block_table, 4, [(p.batch, p.block_table_stride), (c.table_width, 1)])
        self.inside("cu", p.cu_seqlens_q, 4, [(p.batch + 1, 1)])
        self.inside("used", p.seqused_k, 4, [(p.batch, 1)])


@pytest.fixture
def calls(monkeypatch):
    return Calls(monkeypatch)


def cache(fmt=E4M3, blocks=6, page=16, heads=2, dim=64):
    both = torch.zeros(blocks, 2, page, heads, dim).to(fmt)
    return both.unbind(1)


def test_write_hands_over_what_it_was_given(calls):
    kc, vc = cache()
    qkv = torch.randn(9, 3, 2, 64).half()
    slots = torch.arange(7)
    for s in (None, torch.tensor(0.5), torch.rand(1), torch.rand(2)):
        flag_gems.reshape_and_cache_flash(qkv[:, 1], qkv[:, 2], kc, vc, slots, "fp8", s, s)
    flag_gems.reshape_and_cache_flash(qkv[:, 1], qkv[:, 2], kc.view(torch.uint8), vc.view(torch.uint8), slots.int(), "fp8_e5m2", None, None)
    assert calls.check_all() == ["fg_reshape_and_cache_flash_8bit"] * 5
    assert calls.rec.calls[0][1][-2] == _C.CACHE_E4M3 and calls.rec.calls[-1][1][-2] == _C.CACHE_E5M2
    assert [c[1][16] for c in calls.rec.calls[:4]] == [0, 0, 0, 1]


def test_caches_of_the_rows_type_are_copied_as_before(calls):
    """kv_cache_dtype and scales are ignored there, whatever they are; so is an 8-bit cache that takes 8-bit rows."""
    kc = torch.zeros(6, 16, 2, 64).half()
    x = torch.randn(7, 2, 64).half()
    flag_gems.reshape_and_cache_flash(x, x, kc, kc.clone(), torch.arange(7), "fp8", 3.0, "no scale")
    flag_gems.reshape_and_cache_flash(x.to(E4M3), x.to(E4M3), kc.to(E4M3), kc.to(E4M3), torch.arange(7), "auto", None, None)
    assert [c[0] for c in calls.rec.calls] == ["fg_reshape_and_cache_flash"] * 2


def test_write_refusals(calls):
    kc, vc = cache()
    x, slots = torch.randn(7, 2, 64).half(), torch.arange(7)
    w = flag_gems.reshape_and_cache_flash
    with pytest.raises(ValueError, match="bytes needs kv_cache_dtype"):
        w(x, x, kc.view(torch.uint8), vc.view(torch.uint8), slots, "auto", None, None)
    with pytest.raises(ValueError, match="does not fit"):
        w(x, x, kc, vc, slots, "fp8_e5m2", None, None)
    with pytest.raises(AssertionError):
        w(x, x, kc, vc.to(E5M2), slots, "fp8", None, None)
    with pytest.raises(AssertionError):
        w(x, x.float(), kc, vc, slots, "fp8", None, None)
    with pytest.raises(AssertionError, match="cache shape"):
        w(x, x, kc[:, :, :1], vc, slots, "fp8", None, None)
    with pytest.raises(AssertionError, match="key/value shape"):
        w(x[:3], x, kc, vc, slots, "fp8", None, None)
    with pytest.raises(AssertionError, match="dense"):
        w(x.transpose(1, 2).contiguous().transpose(1, 2), x, kc, vc, slots, "fp8", None, None)
    with pytest.raises(AssertionError, match="page must be dense"):
        w(x, x, torch.zeros(6, 2, 16, 64).to(E4M3).transpose(1, 2), vc, slots, "fp8", None, None)
    with pytest.raises(AssertionError, match="slot_mapping"):
        w(x, x, kc, vc, slots.float(), "fp8", None, None)
    with pytest.raises(TypeError, match="float64"):
        w(x.double(), x.double(), kc, vc, slots, "fp8", None, None)
    with pytest.raises(TypeError, match="must be a tensor"):
        w(x, x, kc, vc, slots, "fp8", 0.5, None)
    with pytest.raises(ValueError, match="float32"):
        w(x, x, kc, vc, slots, "fp8", torch.ones(1).half(), None)
    with pytest.raises(ValueError, match="one number or"):
        w(x, x, kc, vc, slots, "fp8", None, torch.ones(3))
    assert not calls.rec.calls


def test_read_hands_over_what_it_was_given(calls):
    kc, vc = cache()
    table = torch.zeros(3, 9, dtype=torch.int32)[:, :4]
    cu = torch.tensor([0, 5, 5, 30], dtype=torch.int32)
    key = torch.zeros(33, 2, 2, 64)
    k, v = flag_gems.gather_cache_flash(kc, vc, table, cu, 33)
    assert k.dtype == v.dtype == torch.bfloat16 and k.shape == (33, 2, 64)
    k, v = flag_gems.gather_cache_flash(kc, vc, table, cu, 33, k_scale=torch.rand(2), seq_starts=cu[:3], key=key[:, 0], value=key[:, 1])
    assert v.dtype == torch.float32
    k, v = flag_gems.gather_cache_flash(kc.view(torch.uint8), vc.view(torch.uint8), table, cu, 33, "fp8_e5m2", dtype=torch.float16)
    half = torch.zeros(6, 16, 2, 64).half()
    k, v = flag_gems.gather_cache_flash(half, half, table, cu, 33, k_scale="ignored")
    assert k.dtype == torch.float16
    assert calls.check_all() == ["fg_gather_cache_flash"] * 4
    assert [c[1][-2] for c in calls.rec.calls] == [_C.CACHE_E4M3, _C.CACHE_E4M3, _C.CACHE_E5M2, _C.CACHE_SAME]
    flag_gems.gather_cache_flash(kc, vc, table, cu, 0)
    assert len(calls.rec.calls) == 4


def test_read_refusals(calls):
    kc, vc = cache()
    table, cu = torch.zeros(3, 4, dtype=torch.int32), torch.tensor([0, 5, 5, 30], dtype=torch.int32)
    r = flag_gems.gather_cache_flash
    with pytest.raises(ValueError, match="bytes needs"):
        r(kc.view(torch.uint8), vc.view(torch.uint8), table, cu, 30)
    with pytest.raises(AssertionError, match="read back as it is"):
        r(kc.half(), vc.half(), table, cu, 30, dtype=torch.float32)
    with pytest.raises(AssertionError, match="block_table"):
        r(kc, vc, table.long(), cu, 30)
    with pytest.raises(AssertionError, match="block_table"):
        r(kc, vc, table[:2], cu, 30)
    with pytest.raises(AssertionError, match="cu_seqlens"):
        r(kc, vc, table, cu.long(), 30)
    with pytest.raises(AssertionError, match="seq_starts"):
        r(kc, vc, table, cu, 30, seq_starts=cu)
    with pytest.raises(AssertionError, match="num_rows, heads"):
        r(kc, vc, table, cu, 30, key=torch.zeros(29, 2, 64))
    with pytest.raises(AssertionError, match="overlap"):
        r(kc, vc, table, cu, 30, key=torch.zeros(1, 2, 64).expand(30, 2, 64), value=torch.zeros(30, 2, 64))
    with pytest.raises(TypeError):
        r(kc, vc, table, cu, 30, dtype=torch.float64)
    with pytest.raises(AssertionError, match="match"):
        r(kc, vc.to(E5M2), table, cu, 30)
    assert not calls.rec.calls


def attend(kc, vc, **kw):
    q = kw.pop("q", torch.randn(5, 8, 64).bfloat16())
    cu, used = torch.tensor([0, 2, 5], dtype=torch.int32), torch.tensor([20, 33], dtype=torch.int32)
    table = kw.pop("table", torch.zeros(2, 3, dtype=torch.int32))
    return flag_gems.flash_attn_varlen_func(q, kc, vc, 3, cu, 33, seqused_k=used, causal=True, block_table=table, **kw)


def test_attention_hands_over_what_it_was_given(calls):
    kc, vc = cache()
    out, lse = attend(kc, vc, return_softmax_lse=True)
    assert out.shape == (5, 8, 64) and out.dtype == torch.bfloat16 and lse.shape == (8, 5)
    for s in (torch.tensor(0.5), torch.rand(2), torch.rand(2, 2), torch.rand(2, 1), torch.tensor(0.5).expand(2, 2)):
        attend(kc, vc, k_descale=s, v_descale=s)
    attend(kc.float().bfloat16(), vc.float().bfloat16(), window_size=(9, 0), num_sink_tokens=4, q_descale=1, k_descale="ignored")
    assert calls.check_all() == ["fg_cache_attn_fwd"] * 7
    last = _C.FgCacheAttnParams.from_buffer_copy([a for n, a in calls.rec.calls if n == "fg_cache_attn_fwd"][-1][0])
    assert (last.cache_format, last.num_sink_tokens, last.base.window_left, last.table_width, last.num_pages) == (_C.CACHE_SAME, 4, 9, 3, 6)
    assert last.k_scale is None
    before = len(calls.rec.calls)
    attend(kc.float().bfloat16(), vc.float().bfloat16(), num_sink_tokens=4)        # no left window: sinks change nothing
    attend(kc.float().bfloat16(), vc.float().bfloat16(), window_size=(9, 0))       # a window without sinks: as ever
    assert [n for n, _ in calls.rec.calls[before:] if n.endswith("fwd")] == ["fg_flash_attn_varlen_fwd"] * 2


def test_attention_refusals(calls):
    kc, vc = cache()
    with pytest.raises(ValueError, match="bytes needs"):
        attend(kc.view(torch.uint8), vc.view(torch.uint8))
    with pytest.raises(NotImplementedError, match="q_descale"):
        attend(kc, vc, q_descale=torch.ones(1))
    with pytest.raises(NotImplementedError, match="alibi"):
        attend(kc, vc, alibi_slopes=torch.ones(8))
    with pytest.raises(AssertionError, match="fp16 and bf16"):
        attend(kc, vc, q=torch.randn(5, 8, 64))
    with pytest.raises(AssertionError, match="fp16 and bf16"):
        attend(kc, vc, q=torch.randn(5, 8, 64).to(E4M3))
    with pytest.raises(AssertionError):
        attend(kc, vc.to(E5M2))
    with pytest.raises(AssertionError, match="negative"):
        attend(kc, vc, num_sink_tokens=-1)
    with pytest.raises(AssertionError, match="negative"):
        attend(kc.float().bfloat16(), vc.float().bfloat16(), num_sink_tokens=-1)
    with pytest.raises(AssertionError, match="must divide"):
        attend(kc, vc, q=torch.randn(5, 7, 64).bfloat16())
    with pytest.raises(AssertionError):
        attend(kc, vc, table=torch.zeros(1, 3, dtype=torch.int32))
    with pytest.raises(AssertionError):
        attend(kc.float().half(), vc.float().half(), window_size=(9, 0), num_sink_tokens=4)   # q is bf16
    with pytest.raises(ValueError, match="must expand"):
        attend(kc, vc, k_descale=torch.rand(3))
    with pytest.raises(ValueError, match="float32"):
        attend(kc, vc, v_descale=torch.rand(2).half())
    with pytest.raises(TypeError, match="must be a tensor"):
        attend(kc, vc, v_descale=0.5)
    with pytest.raises(AssertionError, match="dropout"):
        attend(kc, vc, dropout_p=0.1)
    assert not [n for n, _ in calls.rec.calls if n.endswith("fwd")]


def test_c_entry_points_refuse_on_the_host():
    lib, one = _C.lib(), ctypes.c_void_p(256)

    def write(n=4, H=2, D=64, bs=16, blocks=4, kbs=2048, vbs=2048, ptr=one, ss=0, dtype=_C.FG_F16, fmt=_C.CACHE_E4M3):
        return lib.fg_reshape_and_cache_flash_8bit(ptr, one, one, one, one, 1, n, H, D, bs, blocks, H * D, H * D, kbs, vbs, one, ss, None, 0, dtype, fmt, None)

    assert write(n=0) == 0 and write(blocks=0) == 0 and write(H=0) == 0
    for kw, word in (({"n": -1}, "negative"), ({"bs": 0}, "block_size"), ({"dtype": 9}, "dtype"), ({"fmt": 0}, "not e4m3"), ({"ptr": None}, "null"),
                     ({"kbs": 2047}, "block stride"), ({"vbs": 2047}, "block stride"), ({"ss": 2}, "scale")):
        assert write(**kw) == -1 and word in _C.last_error(), kw

    def read(batch=2, rows=4, H=2, D=64, ps=16, pages=4, kps=2048, ks=128, vs=128, ss=0, dtype=_C.FG_F16, fmt=_C.CACHE_E4M3, ptr=one):
        return lib.fg_gather_cache_flash(one, one, ptr, one, one, 4, 4, one, None, batch, rows, H, D, ps, pages, kps, 2048, ks, vs, one, ss, None, 0, dtype, fmt, None)

    assert read(rows=0) == 0 and read(batch=0) == 0
    for kw, word in (({"rows": -1}, "negative"), ({"ps": 0}, "page size"), ({"dtype": 9}, "dtype"), ({"fmt": 3}, "format"), ({"ptr": None}, "null"),
                     ({"kps": 2047}, "page stride"), ({"ks": 127}, "row stride"), ({"vs": 0}, "row stride"), ({"ss": 5}, "scale"),
                     ({"pages": 0}, "no pages")):
        assert read(**kw) == -1 and word in _C.last_error(), kw

    assert write(n=1 << 27) == -2 and "too large" in _C.last_error()
    assert read(rows=1 << 27) == -2 and "too large" in _C.last_error()

    def attn(**kw):
        c = _C.FgCacheAttnParams()
        p = c.base
        for f in ("q", "k_cache", "v_cache", "out", "cu_seqlens_q", "seqused_k", "block_table"):
            setattr(p, f, 256)
        p.total_q, p.batch, p.Hq, p.Hk, p.D, p.page_size, p.max_seqlen_q, p.max_seqlen_k = 4, 2, 8, 2, 64, 16, 2, 50
        p.q_row_stride, p.q_head_stride, p.o_row_stride, p.o_head_stride = 512, 64, 512, 64
        for n in "kv":
            setattr(p, n + "_page_stride", 2048), setattr(p, n + "_row_stride", 128), setattr(p, n + "_head_stride", 64)
        p.dtype, p.window_left, p.window_right = _C.FG_BF16, -1, -1
        c.cache_format, c.num_pages, c.table_width = _C.CACHE_E4M3, 6, 4
        for name, value in kw.items():
            setattr(c if hasattr(c, name) else p, name, value)
        return lib.fg_cache_attn_fwd(ctypes.byref(c), None)

    assert lib.fg_cache_attn_fwd(None, None) == -1
    assert attn(batch=0) == 0 and attn(total_q=0) == 0
    for kw, rc, word in (({"dtype": _C.FG_F32}, -1, "fp16 and bf16"), ({"cache_format": 7}, -1, "format"), ({"num_sink_tokens": -1}, -1, "negative"),
                         ({"q": None}, -1, "null"), ({"D": 72}, -1, "multiple of 16"), ({"D": 272}, -1, "at most 256"), ({"Hq": 7}, -1, "not a multiple"),
                         ({"page_size": 0}, -1, "page size"), ({"max_seqlen_q": 0}, -1, "max_seqlen_q"), ({"num_pages": 0}, -1, "pages"),
                         ({"alibi_slopes": 256}, -2, "alibi"), ({"k_cache": 264}, -2, "aligned"), ({"k_row_stride": 136}, -2, "aligned"),
                         ({"v_page_stride": 2056}, -2, "aligned"), ({"q_head_stride": 66}, -2, "aligned"), ({"batch": 65536}, -2, "grid"),
                         ({"table_width": 1 << 27}, -2, "spans"), ({"total_q": 1 << 30, "max_seqlen_q": 1 << 30}, -2, "too many"),
                         ({"total_q": 1 << 30, "max_seqlen_q": 1 << 30, "D": 256}, -2, "too many")):
        assert attn(**kw) == rc and word in _C.last_error(), (kw, _C.last_error())


def test_vllm_hook_passes_an_8bit_cache_on(monkeypatch):
    """kv_cache_dtype fp8: the cache of bytes is written and attended over as the format that the name stands for; the
    query keeps its 16 bits."""
    import importlib

    from flaggems_amd.patches import patch_vllm_all

    attention = importlib.import_module("flaggems_amd.ops.attention")
    fused = importlib.import_module("flaggems_amd.fused.reshape_and_cache_flash")
    seen = []
    monkeypatch.setattr(fused, "reshape_and_cache_flash", lambda *a: seen.append(a))
    monkeypatch.setattr(attention, "flash_attn_varlen_func", lambda **kw: seen.append(kw))
    one = torch.ones(1)
    layer = types.SimpleNamespace(_q_scale=one, _k_scale=one, _v_scale=one)
    meta = types.SimpleNamespace(num_actual_tokens=3, slot_mapping=None, use_cascade=False, query_start_loc=torch.zeros(3), seq_lens=None,
                                 max_query_len=2, max_seq_len=9, block_table=None, scheduler_metadata=None)
    for name, kind in (("fp8", E4M3), ("fp8_e4m3", E4M3), ("fp8_e5m2", E5M2)):
        impl = types.SimpleNamespace(kv_cache_dtype=name, use_irope=False, scale=1.0, alibi_slopes=None, sliding_window=(-1, -1), logits_soft_cap=0)
        x = torch.zeros(3, 2, 64)
        patch_vllm_all.custom_gems_flash_attention_impl_forward(impl, layer, x, x, x, torch.zeros(2, 4, 16, 2, 64, dtype=torch.uint8), meta, output=x)
        write, attn = seen[-2:]
        assert write[2].dtype == kind and write[5] == name and attn["k"].dtype == kind and attn["q_descale"] is None and attn["k_descale"].shape == (2, 2)


def test_struct_mirror_of_the_attention_parameters():
    import os
    import re

    text = open(os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include", "fg_mi355.h")).read()
    body = re.sub(r"/\*.*?\*/", "", text[text.index("typedef struct FgCacheAttnParams {"):text.index("} FgCacheAttnParams;")], flags=re.S)
    names = []
    for decl in body[body.index("{") + 1:].split(";"):
        parts = decl.replace("*", " ").split(",")
        if parts[0].split():
            names += [parts[0].split()[-1]] + [p.strip() for p in parts[1:]]
    assert names == [f[0] for f in _C.FgCacheAttnParams._fields_]


@pytest.mark.parametrize("fmt", ["e4m3", "e5m2"])
def test_oracle_rounding_is_the_formats(fmt):
    """Known answers: every finite value of the format is its own nearest, the middle of two neighbours goes to the one whose
    last bit is 0, other values to the nearer; torch's conversion agrees inside the range."""
    kind = {"e4m3": E4M3, "e5m2": E5M2}[fmt]
    codes = torch.arange(128, dtype=torch.uint8).view(kind).double()
    v = codes[torch.isfinite(codes)]                               # ascending, codes of neighbours differ by one
    assert torch.equal(O.round_to_8bit(v, fmt), v) and torch.equal(O.round_to_8bit(-v, fmt), -v)
    mid = (v[1:] + v[:-1]) / 2
    even = torch.where(torch.arange(len(mid)) % 2 == 0, v[:-1], v[1:])
    assert torch.equal(O.round_to_8bit(mid, fmt), even)
    x = torch.randn(4000, dtype=torch.float64) * v.max() / 8
    x = x[x.abs() <= v.max()].float()
    assert torch.equal(O.round_to_8bit(x.double(), fmt), x.to(kind).double())
    assert O.round_to_8bit(torch.tensor([1e9, float("inf"), float("-inf")]), fmt).tolist() == [v.max(), v.max(), -v.max()]


def test_oracle_attention_against_scalar_sums():
    """Known answers for the attention oracle: written out for single keys, with window, sinks, scales and empty rows."""
    import math

    torch.manual_seed(0)
    q = torch.randn(4, 2, 8).half()
    kc, vc = (torch.randn(5, 4, 1, 8).to(E4M3) for _ in range(2))
    table = torch.tensor([[3, 1, 0], [2, 4, 0]], dtype=torch.int32)
    cu, used = torch.tensor([0, 3, 4], dtype=torch.int32), torch.tensor([9, 1], dtype=torch.int32)
    ks, vs = torch.tensor([[0.5], [2.0]]), torch.tensor([0.25])
    r = O.cache_attention(q, kc, vc, cu, used, table, 0.3, True, (2, 0), 1, 0.0, ks, vs)
    for row, (b, pos) in enumerate([(0, 6), (0, 7), (0, 8), (1, 0)]):
        for h in range(2):
            num, den = [0.0] * 8, 0.0
            for j in range(pos + 1):
                if j >= pos - 2 or j < 1:
                    k = [float(x) * float(ks[b, 0]) for x in kc[table[b, j // 4], j % 4, 0].float()]
                    w = math.exp(0.3 * sum(float(x) * y for x, y in zip(q[row, h], k)))
                    den += w
                    num = [n + w * 0.25 * float(x) for n, x in zip(num, vc[table[b, j // 4], j % 4, 0].float())]
            assert abs(float(r["lse"][h, row]) - math.log(den)) < 1e-9
            assert max(abs(float(r["out"][row, h, i]) - num[i] / den) for i in range(8)) < 1e-9
    r = O.cache_attention(q, kc, vc, cu, torch.tensor([1, 0], dtype=torch.int32), table, 0.3)
    assert torch.isinf(r["lse"][:, [0, 1, 3]]).all() and (r["out"][[0, 1, 3]] == 0).all() and torch.isfinite(r["lse"][:, 2]).all()


def test_bounds_beyond_32_bits_are_cut(calls):
    """A window, a number of sinks or a length limit of any size is passed on as the largest that the parameters hold."""
    kc, vc = cache()
    attend(kc, vc, window_size=(1 << 40, 1 << 50), num_sink_tokens=1 << 33)
    attend(kc, vc, window_size=(-7, -5))
    a, b = (_C.FgCacheAttnParams.from_buffer_copy(c[0]) for n, c in calls.rec.calls if n == "fg_cache_attn_fwd")
    assert (a.base.window_left, a.base.window_right, a.num_sink_tokens) == (2 ** 31 - 1,) * 3
    assert (b.base.window_left, b.base.window_right, b.num_sink_tokens) == (-1, -1, 0)


def test_tensors_off_the_gpu_are_refused():
    kc, vc = cache()
    x = torch.randn(7, 2, 64).half()
    with pytest.raises(AssertionError, match="on a GPU"):
        flag_gems.reshape_and_cache_flash(x, x, kc, vc, torch.arange(7), "fp8", None, None)
    with pytest.raises(AssertionError, match="on a GPU"):
        flag_gems.gather_cache_flash(kc, vc, torch.zeros(1, 2, dtype=torch.int32), torch.tensor([0, 7], dtype=torch.int32), 7)
    with pytest.raises(AssertionError):
        attend(kc, vc)


def test_scratch_goes_by_the_tokens_that_are_there():
    """A bound on the sequences' length that is far above the number of tokens costs nothing."""
    def scratch(total, longest):
        c = _C.FgCacheAttnParams()
        p = c.base
        for f in ("q", "k_cache", "v_cache", "out", "cu_seqlens_q", "seqused_k", "block_table"):
            setattr(p, f, 256)
        p.total_q, p.batch, p.Hq, p.Hk, p.D, p.page_size, p.max_seqlen_q, p.max_seqlen_k = total, 1, 8, 2, 256, 16, longest, 20000
        for n in "kv":
            setattr(p, n + "_page_stride", 8192), setattr(p, n + "_row_stride", 512), setattr(p, n + "_head_stride", 256)
        p.dtype, p.window_left, p.window_right = _C.FG_BF16, -1, -1
        c.cache_format, c.num_pages, c.table_width = _C.CACHE_E4M3, 6, 1250
        return _C.lib().fg_cache_attn_workspace_bytes(ctypes.byref(c), 0)

    assert scratch(1, 1) > 0 and scratch(1, 2 ** 31 - 1) == scratch(1, 1)
