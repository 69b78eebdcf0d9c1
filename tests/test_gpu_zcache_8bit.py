"""GPU parity of the 8-bit paged cache: rows quantized as they are written, read back as packed rows, and a run of
write, attention and read-back together, against the 64-bit oracle."""
import random

import pytest
import torch

import flag_gems
from oracle import torch_ref as O

pytestmark = pytest.mark.gpu
FMT = {"e4m3": torch.float8_e4m3fn, "e5m2": torch.float8_e5m2}


def values(cache):
    return cache.cpu().float().double()


def dirty(shape, fmt, dev, seed=3):
    """A cache with something in every place."""
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * 20).to(FMT[fmt]).to(dev)


def check_written(key, value, kc, vc, before, slots, ks, vs, fmt):
    """Every written place holds the nearest value of the format to row / scale, every other place what it held.  The
    quotient is rounded to fp32 first (2^-24 of it): a place may differ from the nearest value of the exact quotient only
    where that quotient lies within that distance of the middle between two values."""
    for x, cache, old, s in ((key, kc, before[0], ks), (value, vc, before[1], vs)):
        want = O.cache_write_8bit(x, old.float(), slots, s, fmt)
        got = values(cache)
        near = got == want
        if not near.all():
            flat = torch.full((want.numel() // (want.shape[2] * want.shape[3]), want.shape[2], want.shape[3]), float("nan"), dtype=torch.float64)
            exact = x.cpu().double() / O.per_head(s, x.shape[1])
            for i, slot in enumerate(slots.tolist()):
                if 0 <= slot < flat.shape[0]:
                    flat[slot] = exact[i]
            q = flat.view(want.shape)[~near]
            mid = (got[~near] + want[~near]) / 2
            assert ((q - mid).abs() <= 2.0 ** -24 * q.abs()).all()


@pytest.mark.parametrize("fmt", ["e4m3", "e5m2"])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("heads,dim,page,scales", [(8, 128, 16, "one"), (3, 64, 16, "head"), (1, 16, 1, "none"), (5, 24, 7, "head"),
                                                   (2, 7, 5, "head"), (4, 256, 64, "one")])
def test_write_8bit(gpu, fmt, dtype, heads, dim, page, scales):
    torch.manual_seed(0); random.seed(0)
    tokens, blocks = 37, 41
    qkv = torch.randn(tokens + 2, 3, heads, dim, device=gpu).mul_(3).to(dtype)
    _, key, value = qkv.unbind(1)                                      # strided tokens, more rows than slots
    top = torch.finfo(FMT[fmt]).max
    key[3, 0, :4] = torch.tensor([0.0, 1e4, -1e4, 2.0 ** -20], device=gpu, dtype=dtype)   # zero, beyond the range, tiny
    ks, vs = {"none": (None, None), "one": (torch.tensor(0.037, device=gpu), torch.tensor([1.7], device=gpu)),
              "head": (torch.rand(heads, device=gpu) + 0.01, torch.rand(heads, device=gpu) * 8 / top + 1e-3)}[scales]
    both = torch.stack([dirty((blocks, page, heads, dim), fmt, gpu, s) for s in (3, 4)], 1)   # pages of K and V in turn
    kc, vc = both.unbind(1)
    before = (kc.clone(), vc.clone())
    slots = torch.tensor(random.sample(range(blocks * page), min(tokens, blocks * page)), device=gpu)
    slots[1] = -1
    slots[2] = blocks * page                                           # outside the cache: skipped
    flag_gems.reshape_and_cache_flash(key, value, kc, vc, slots, "fp8_" + fmt, ks, vs)
    n = len(slots)
    check_written(key[:n], value[:n], kc, vc, before, slots, ks, vs, fmt)
    # int32 slots and a cache of bytes: the same
    kc2, vc2 = before[0].clone(), before[1].clone()
    flag_gems.reshape_and_cache_flash(key, value, kc2.view(torch.uint8), vc2.view(torch.uint8), slots.int(), "fp8_" + fmt, ks, vs)
    assert torch.equal(kc2.view(torch.uint8), kc.view(torch.uint8)) and torch.equal(vc2.view(torch.uint8), vc.view(torch.uint8))


@pytest.mark.parametrize("fmt", ["e4m3", "e5m2"])
def test_write_8bit_every_value_and_ties(gpu, fmt):
    """Every finite value of the format, the middles between neighbours (to the even one), the largest value's surroundings,
    infinities and NaN; with a scale of 1 and with one that is no power of two, where the exact quotients are the same."""
    codes = torch.arange(256, dtype=torch.uint8).view(FMT[fmt]).float()
    v = torch.unique(codes[torch.isfinite(codes)])
    x = torch.cat([v, (v[1:] + v[:-1]) / 2, v * (1 + 2.0 ** -12), torch.tensor([v.max() * 1.01, v.max() * 8, float("inf"), float("-inf")])])
    x = torch.cat([x, torch.zeros(-x.numel() % 16)]).view(-1, 1, 16).to(gpu)
    slots = torch.arange(x.shape[0], device=gpu)
    for s in (1.0, 1.5):
        kc = torch.zeros(x.shape[0], 1, 1, 16, dtype=FMT[fmt], device=gpu); vc = torch.zeros_like(kc)
        flag_gems.reshape_and_cache_flash(x * s, x * s, kc, vc, slots, "fp8_" + fmt, torch.tensor(s, device=gpu), torch.tensor(s, device=gpu))
        want = O.round_to_8bit(x.cpu().double(), fmt)
        assert torch.equal(values(kc).view(-1), want.view(-1)) and torch.equal(values(vc).view(-1), want.view(-1))
    nan = torch.full((1, 1, 16), float("nan"), device=gpu, dtype=torch.bfloat16)
    flag_gems.reshape_and_cache_flash(nan, nan, kc, vc, slots[:1], "fp8_" + fmt, None, None)
    assert torch.isnan(values(kc)[0]).all() and not torch.isnan(values(kc)[1:]).any()


@pytest.mark.parametrize("fmt", ["e4m3", "e5m2"])
@pytest.mark.parametrize("scale", [1.375 * 2.0 ** -99, 1.375 * 2.0 ** -61, 1.375 * 2.0 ** -60, 1.375 * 2.0 ** 99, 1.375 * 2.0 ** 101])
def test_write_8bit_ties_at_extreme_scales(gpu, fmt, scale):
    """Middles between neighbours times a scale of four bits are fp32 numbers: their quotients are exact, and go to the even one."""
    codes = torch.arange(256, dtype=torch.uint8).view(FMT[fmt]).float()
    v = torch.unique(codes[torch.isfinite(codes)])
    x = torch.cat([v, (v[1:] + v[:-1]) / 2])
    x = torch.cat([x, torch.zeros(-x.numel() % 16)]).view(-1, 1, 16)
    scaled = (x.double() * scale).float()
    assert torch.equal(scaled.double(), x.double() * scale)
    kc = torch.zeros(x.shape[0], 1, 1, 16, dtype=FMT[fmt], device=gpu); vc = torch.zeros_like(kc)
    s = torch.tensor(scale, device=gpu)
    flag_gems.reshape_and_cache_flash(scaled.to(gpu), scaled.to(gpu), kc, vc, torch.arange(x.shape[0], device=gpu), "fp8_" + fmt, s, s)
    want = O.round_to_8bit(x.double(), fmt)
    assert torch.equal(values(kc).view(-1), want.view(-1)) and torch.equal(values(vc).view(-1), want.view(-1))


def test_write_8bit_nothing(gpu):
    kc = dirty((2, 4, 2, 16), "e4m3", gpu); vc = kc.clone(); old = kc.clone()
    x = torch.ones(0, 2, 16, device=gpu, dtype=torch.float16)
    flag_gems.reshape_and_cache_flash(x, x, kc, vc, torch.zeros(0, dtype=torch.long, device=gpu), "fp8", None, None)
    assert torch.equal(values(kc), values(old))


def read_oracle(cache, table, cu, starts, rows, scale, old):
    out = old.cpu().double().clone()
    page = cache.shape[1]
    vals, table, cu = values(cache) if cache.dtype in FMT.values() else cache.cpu().double(), table.cpu(), cu.tolist()
    for b in range(len(cu) - 1):
        for i in range(cu[b], min(cu[b + 1], rows)):
            pos = i - cu[b] + (0 if starts is None else int(starts[b]))
            at = int(table[b, pos // page]) if pos // page < table.shape[1] else -1
            out[i] = vals[at, pos % page] * O.per_head(scale, cache.shape[2]) if 0 <= at < cache.shape[0] else 0
    return out


@pytest.mark.parametrize("fmt,dtype", [("e4m3", torch.bfloat16), ("e4m3", torch.float32), ("e5m2", torch.float16), ("same", torch.float16),
                                       ("same", torch.bfloat16), ("same", torch.float32)])
@pytest.mark.parametrize("heads,dim,page", [(8, 128, 16), (2, 64, 48), (1, 16, 1), (5, 24, 7), (3, 7, 5)])
@pytest.mark.parametrize("scales", ["none", "one", "head"])
def test_read(gpu, fmt, dtype, heads, dim, page, scales):
    torch.manual_seed(1)
    lens = [0, 1, 33, 0, 50, 7]
    blocks = 70
    cache = [torch.randn(blocks, page, heads, dim, device=gpu).mul_(3).to(dtype if fmt == "same" else FMT[fmt]) for _ in range(2)]
    table = torch.randint(0, blocks, (len(lens), 128), dtype=torch.int32, device=gpu)[:, ::1]
    starts = torch.tensor([0, 3, 5, 0, 11, 2], dtype=torch.int32, device=gpu)
    cu = torch.tensor([2] + lens, dtype=torch.int32, device=gpu).cumsum(0, dtype=torch.int32)   # the first two rows belong to nobody
    rows = int(cu[-1]) + 4
    s = {"none": (None, None), "one": (torch.tensor([0.3], device=gpu), torch.tensor(2.5, device=gpu)),
         "head": (torch.rand(heads, device=gpu), torch.rand(heads, device=gpu))}[scales]
    table[2, 20 // page] = -1                                          # pages that are not there: zeros
    table[4, 30 // page] = blocks
    wide = torch.full((rows, 2, heads, dim), 7.0, dtype=dtype, device=gpu)
    key, value = wide.unbind(1)                                        # strided rows
    for st in (None, starts):
        wide.fill_(7.0)
        got = flag_gems.gather_cache_flash(cache[0], cache[1], table, cu, rows, k_scale=s[0], v_scale=s[1], seq_starts=st, key=key, value=value)
        assert got[0] is key and got[1] is value
        for x, c, sc in ((key, cache[0], s[0]), (value, cache[1], s[1])):
            want = read_oracle(c, table, cu, st, rows, None if fmt == "same" else sc, torch.full((rows, heads, dim), 7.0))
            if fmt == "same":
                assert torch.equal(x.cpu().double(), want)
            else:  # one product in fp32 and one rounding: half a step each
                u = torch.finfo(dtype).eps / 2
                assert ((x.cpu().double() - want).abs() <= (u + 2.0 ** -23) * want.abs() + torch.finfo(dtype).smallest_normal * u).all()


def test_read_many_sequences_and_short_table(gpu):
    """More sequences than one comparison of 64 takes, empty ones among them; positions behind a table's end give zeros."""
    torch.manual_seed(2)
    g = torch.Generator().manual_seed(5)
    lens = torch.randint(0, 4, (333,), generator=g)
    cache = torch.randn(50, 2, 2, 16, device=gpu).to(torch.float8_e4m3fn)
    table = torch.randint(0, 50, (333, 1), generator=g).int().to(gpu)
    cu = torch.cat([torch.zeros(1, dtype=torch.long), lens.cumsum(0)]).int().to(gpu)
    rows = int(cu[-1])
    k, v = flag_gems.gather_cache_flash(cache, cache, table, cu, rows, dtype=torch.float32)
    want = read_oracle(cache, table, cu, None, rows, None, torch.zeros(rows, 2, 16))
    assert torch.equal(k.cpu().double(), want) and torch.equal(v.cpu().double(), want)
    k, v = flag_gems.gather_cache_flash(cache, cache, table, cu[:1], 3)  # no sequence: nothing is written
    assert k.shape == (3, 2, 16) and k.dtype == torch.bfloat16


def test_cache_beyond_4_gib(gpu):
    """Offsets past 32 bits: pages at both ends of an 8-bit cache of 4.5 GiB, written, attended over and read back."""
    blocks, page, heads, dim = 147456, 16, 16, 128
    kc = torch.zeros(blocks, page, heads, dim, dtype=torch.uint8, device=gpu).view(torch.float8_e4m3fn)
    vc = torch.zeros(blocks, page, heads, dim, dtype=torch.uint8, device=gpu).view(torch.float8_e4m3fn)
    torch.manual_seed(3)
    n = 40
    key, value = (torch.randn(n, heads, dim, device=gpu).to(torch.bfloat16) for _ in range(2))
    table = torch.tensor([[blocks - 1, 0, blocks - 7]], dtype=torch.int32, device=gpu)
    pos = torch.arange(n, device=gpu)
    slots = table[0].long()[pos // page] * page + pos % page
    s = torch.tensor(0.01, device=gpu)
    flag_gems.reshape_and_cache_flash(key, value, kc, vc, slots, "fp8", s, s)
    cu = torch.tensor([0, n], dtype=torch.int32, device=gpu)
    k, v = flag_gems.gather_cache_flash(kc, vc, table, cu, n, k_scale=s, v_scale=s, dtype=torch.float32)
    for x, got in ((key, k), (value, v)):
        want = O.round_to_8bit(x.cpu().float().div(0.01).double(), "e4m3") * float(s)
        assert (got.cpu().double() - want).abs().max() <= 2.0 ** -3 * 0.1 * want.abs().max()  # the same rows (a step at most)
    used = torch.tensor([n], dtype=torch.int32, device=gpu)
    q = torch.randn(1, heads, dim, device=gpu).to(torch.bfloat16)
    one = torch.tensor([0, 1], dtype=torch.int32, device=gpu)
    out = flag_gems.flash_attn_varlen_func(q, kc, vc, 1, one, n, seqused_k=used, causal=True, block_table=table, k_descale=s, v_descale=s)
    t = torch.einsum("hd,khd->hk", q[0].cpu().double(), k.cpu().double()) * dim ** -0.5
    want = torch.einsum("hk,khd->hd", torch.softmax(t, 1), v.cpu().double())
    spread = torch.einsum("hk,khd->hd", torch.softmax(t, 1), v.cpu().double().abs())
    assert ((out[0].cpu().double() - want).abs() <= 2.0 ** -8 * (want.abs() + spread) + 1e-3 * spread).all()


def test_write_attend_read_together(gpu):
    """A few sequences that grow: each step writes new tokens into the 8-bit cache and attends over it, with the window and
    sinks of streaming generation; at the end the cache is read back.  Everything against the oracle on the values that the
    cache must hold."""
    from test_gpu_zattn_cache import assert_close

    torch.manual_seed(4); random.seed(4)
    batch, hq, hk, dim, page, blocks, dtype = 3, 8, 2, 64, 16, 40, torch.bfloat16
    kc = torch.zeros(blocks, page, hk, dim, dtype=torch.float8_e4m3fn, device=gpu); vc = torch.zeros_like(kc)
    order = random.sample(range(blocks), blocks)
    table = torch.tensor(order[:36], dtype=torch.int32, device=gpu).view(batch, 12)
    lens = [0, 0, 0]
    ks, vs = torch.tensor([0.02, 0.03], device=gpu), torch.tensor([0.015], device=gpu)
    for new in ([37, 5, 64], [1, 1, 1], [1, 1, 1], [30, 1, 2], [1, 1, 1]):
        pos = [torch.arange(l, l + n) for l, n in zip(lens, new)]
        lens = [l + n for l, n in zip(lens, new)]
        slots = torch.cat([table[b].cpu().long()[p // page] * page + p % page for b, p in enumerate(pos)]).to(gpu)
        q = torch.randn(sum(new), hq, dim, device=gpu).to(dtype)
        key, value = (torch.randn(sum(new), hk, dim, device=gpu).to(dtype) for _ in range(2))
        before = (kc.clone(), vc.clone())
        flag_gems.reshape_and_cache_flash(key, value, kc, vc, slots, "fp8_e4m3", ks, vs)
        # (a quotient next to the middle of two values may go to either: see check_written)
        check_written(key, value, kc, vc, tuple(x.float() for x in before), slots, ks, vs, "e4m3")
        cu = torch.tensor([0] + new, dtype=torch.int32, device=gpu).cumsum(0, dtype=torch.int32)
        used = torch.tensor(lens, dtype=torch.int32, device=gpu)
        out, lse = flag_gems.flash_attn_varlen_func(q, kc, vc, max(new), cu, max(lens), seqused_k=used, causal=True, block_table=table,
                                                    window_size=(20, 0), num_sink_tokens=4, k_descale=ks, v_descale=vs, return_softmax_lse=True)
        assert_close(out, lse, O.cache_attention(q, kc, vc, cu, used, table, dim ** -0.5, window=(20, 0), sinks=4, k_scale=ks, v_scale=vs), dtype, dim)
    cu = torch.tensor([0] + lens, dtype=torch.int32, device=gpu).cumsum(0, dtype=torch.int32)
    k, v = flag_gems.gather_cache_flash(kc, vc, table, cu, sum(lens), k_scale=ks, v_scale=vs, dtype=torch.float32)
    for b in range(batch):
        p = torch.arange(lens[b])
        at = table[b].cpu().long()[p // page], p % page
        want = values(kc)[at] * O.per_head(ks, hk)
        assert ((k[cu[b]:cu[b + 1]].cpu().double() - want).abs() <= 2.0 ** -23 * want.abs()).all()


def test_vllm_hook_with_an_8bit_cache(gpu):
    """FlashAttentionImpl.forward of the vLLM patch with kv_cache_dtype fp8: the cache arrives as bytes."""
    import types

    from flaggems_amd.patches import patch_vllm_all
    from test_gpu_zattn_cache import assert_close

    torch.manual_seed(6)
    hq, hk, d, page, n = 8, 2, 64, 16, 24
    kv = torch.zeros(2, 6, page, hk, d, dtype=torch.uint8, device=gpu)
    s = torch.tensor(0.02, device=gpu)
    layer = types.SimpleNamespace(_q_scale=torch.tensor(1.0, device=gpu), _k_scale=s, _v_scale=s * 2)
    impl = types.SimpleNamespace(kv_cache_dtype="fp8", use_irope=False, scale=d ** -0.5, alibi_slopes=None, sliding_window=(-1, -1), logits_soft_cap=0)
    table = torch.tensor([[4, 1]], dtype=torch.int32, device=gpu)
    pos = torch.arange(n, device=gpu)
    meta = types.SimpleNamespace(num_actual_tokens=n, slot_mapping=table[0].long()[pos // page] * page + pos % page, use_cascade=False,
                                 query_start_loc=torch.tensor([0, n], dtype=torch.int32, device=gpu), seq_lens=torch.tensor([n], dtype=torch.int32, device=gpu),
                                 max_query_len=n, max_seq_len=n, block_table=table, scheduler_metadata=None)
    q, k, v = (torch.randn(n, h, d, device=gpu).to(torch.bfloat16) for h in (hq, hk, hk))
    out = torch.zeros_like(q)
    patch_vllm_all.custom_gems_flash_attention_impl_forward(impl, layer, q, k, v, kv, meta, output=out)
    kc, vc = kv.view(torch.float8_e4m3fn).unbind(0)
    want = O.cache_attention(q, kc, vc, meta.query_start_loc, meta.seq_lens, table, d ** -0.5, k_scale=s, v_scale=s * 2)
    assert_close(out, None, want, torch.bfloat16, d)
    assert torch.equal(values(kc).view(-1, hk, d)[meta.slot_mapping.cpu()], O.round_to_8bit(k.cpu().float().div(s.cpu()).double(), "e4m3"))
