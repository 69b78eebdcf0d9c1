"""GPU parity of attention over an 8-bit paged cache and of sliding windows with sink tokens, against the 64-bit oracle."""
import importlib
import random

import pytest
import torch

import flag_gems
from oracle import torch_ref as O

pytestmark = pytest.mark.gpu
FMT = {"e4m3": torch.float8_e4m3fn, "e5m2": torch.float8_e5m2}


def assert_close(out, lse, ref, dtype, dim):
    """Bounds from the arithmetic, u = half a step of the type:
      scores: a product of `dim` terms summed in fp32, plus the scaling: |dt| <= (dim + 8) 2^-24 scale sum|q||k|;
      weights: exp of that (twice: numerator and sum), each rounded to the type once: u + 2 |dt| + 8 2^-24, relative;
               a weight in fp16's subnormal range is off by at most half of 2^-24 of a sum that is at least 1;
      output: sum of weights times |v|, plus one rounding of the result (fp16: at least half of 2^-24);
      log-sum-exp: |dt| + a sum of `seen` terms in fp32 + 4 roundings of the result."""
    u = torch.finfo(dtype).eps / 2
    dt = (dim + 8) * 2.0 ** -24 * ref["reach"]
    out = out.cpu().double()
    assert not torch.isnan(out).any()
    rel = (u + 2 * dt + (8 + ref["seen"]) * 2.0 ** -24).t()[:, :, None]
    tol = rel * ref["spread"] + u * ref["out"].abs() + (2.0 ** -25 * (1 + ref["total"]) if dtype == torch.float16 else 0) + 1e-30
    bad = (out - ref["out"]).abs() > tol
    assert not bad.any(), "%d of %d outputs are off, worst %.3g of the bound" % (bad.sum(), bad.numel(), ((out - ref["out"]).abs() / tol).max())
    if lse is not None:
        fin = torch.isfinite(ref["lse"])
        got = lse.cpu().double()
        assert torch.equal(got[~fin], ref["lse"][~fin])            # rows that see nothing: +inf
        tol = dt + (ref["seen"] + 8) * 2.0 ** -24 + 2.0 ** -22 * ref["lse"].abs()
        assert ((got - ref["lse"]).abs()[fin] <= tol[fin]).all()


def make(dev, lens, hq, hk, dim, page, dtype, fmt, seed=0, spare=5, scales="seq"):
    """Pages in random order; whatever no sequence holds, and the places behind a sequence's end, are NaN."""
    g = torch.Generator().manual_seed(seed)
    n = [-(-k // page) for _, k in lens]
    blocks = sum(n) + spare
    order = torch.randperm(blocks, generator=g)
    table = torch.full((len(lens), max(n + [1])), -1, dtype=torch.int32)
    caches = [torch.full((blocks, page, hk, dim), float("nan")) for _ in range(2)]
    at = 0
    for b, (_, k) in enumerate(lens):
        table[b, :n[b]] = order[at:at + n[b]].int()
        at += n[b]
        pos = torch.arange(k)
        for c in caches:
            c[table[b].long()[pos // page], pos % page] = torch.randn(k, hk, dim, generator=g)
    kc, vc = ((c * (1.0 if fmt == "same" else 20.0)).to(dtype if fmt == "same" else FMT[fmt]).to(dev) for c in caches)
    cu = torch.tensor([0] + [q for q, _ in lens]).cumsum(0).int().to(dev)
    used = torch.tensor([k for _, k in lens], dtype=torch.int32, device=dev)
    q = torch.randn(int(cu[-1]), hq, dim, generator=g).mul(1.5).to(dtype).to(dev)
    ks = vs = None
    if fmt != "same" and scales != "none":
        shape = {"one": (), "head": (hk,), "seq": (len(lens), hk), "column": (len(lens), 1)}[scales]
        ks, vs = ((torch.rand(shape, generator=g) * 0.04 + 0.03).to(dev) for _ in range(2))
    return q, kc, vc, cu, used, table.to(dev), ks, vs


def run_and_check(dev, lens, hq, hk, dim, page, dtype, fmt, causal=True, window=(-1, -1), sinks=0, softcap=0.0, seed=0, scales="seq"):
    q, kc, vc, cu, used, table, ks, vs = make(dev, lens, hq, hk, dim, page, dtype, fmt, seed, scales=scales)
    scale = dim ** -0.5
    out, lse = flag_gems.flash_attn_varlen_func(
        q, kc, vc, max(n for n, _ in lens), cu, max(k for _, k in lens), seqused_k=used, softmax_scale=scale, causal=causal, window_size=window,
        softcap=softcap, block_table=table, return_softmax_lse=True, k_descale=ks, v_descale=vs, num_sink_tokens=sinks)
    ref = O.cache_attention(q, kc, vc, cu, used, table, scale, causal, window, sinks, softcap, ks, vs)
    assert_close(out, lse, ref, dtype, dim)
    return out


TYPES = [(torch.bfloat16, "e4m3"), (torch.float16, "e4m3"), (torch.bfloat16, "e5m2"), (torch.float16, "e5m2")]
ALL = TYPES + [(torch.bfloat16, "same"), (torch.float16, "same")]


@pytest.mark.parametrize("dtype,fmt", TYPES)
@pytest.mark.parametrize("hq,hk", [(8, 8), (8, 2), (6, 2), (40, 8), (32, 1), (48, 1)])
@pytest.mark.parametrize("dim", [16, 64, 80, 128, 192, 256])
def test_single_tokens(gpu, dtype, fmt, hq, hk, dim):
    run_and_check(gpu, [(1, 1), (1, 31), (1, 32), (1, 33), (1, 700), (1, 129)], hq, hk, dim, 16, dtype, fmt)


@pytest.mark.parametrize("dtype,fmt", TYPES[:2])
@pytest.mark.parametrize("page", [1, 4, 8, 16, 24, 48, 64, 256, 100])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_page_sizes(gpu, dtype, fmt, page, dim):
    run_and_check(gpu, [(1, 333), (3, 90), (40, 257)], 8, 2, dim, page, dtype, fmt)


@pytest.mark.parametrize("dtype,fmt", TYPES)
@pytest.mark.parametrize("dim,page", [(64, 16), (128, 32), (96, 16), (256, 64), (128, 24)])
def test_chunks(gpu, dtype, fmt, dim, page):
    run_and_check(gpu, [(2, 2), (5, 18), (129, 463), (64, 64), (33, 1000), (1, 77), (0, 50), (200, 201)], 8, 2, dim, page, dtype, fmt)


@pytest.mark.parametrize("hq,hk", [(6, 2), (5, 5), (16, 1), (7, 1), (40, 8)])
@pytest.mark.parametrize("dtype,fmt", [ALL[0], ALL[5]])
def test_chunks_head_groups(gpu, hq, hk, dtype, fmt):
    run_and_check(gpu, [(70, 300), (130, 130), (17, 64)], hq, hk, 64, 16, dtype, fmt, window=(90, 0) if fmt == "same" else (-1, -1), sinks=3)


@pytest.mark.parametrize("dtype,fmt", ALL)
@pytest.mark.parametrize("window,sinks", [((0, 0), 0), ((0, 0), 1), ((5, 0), 4), ((31, 0), 32), ((100, 0), 33), ((64, 0), 1000), ((700, 0), 7), ((5000, 0), 4)])
@pytest.mark.parametrize("dim,page", [(128, 16), (64, 32)])
def test_windows_and_sinks(gpu, dtype, fmt, window, sinks, dim, page):
    if fmt == "same" and sinks == 0:
        sinks = 2
    run_and_check(gpu, [(1, 900), (1, 3), (7, 300), (130, 130), (65, 700)], 8, 2, dim, page, dtype, fmt, window=window, sinks=sinks)


@pytest.mark.parametrize("dtype,fmt", [ALL[0], ALL[3], ALL[4]])
@pytest.mark.parametrize("causal,window,sinks", [(False, (-1, -1), 0), (False, (20, 30), 5), (False, (20, -1), 3), (False, (-1, 10), 2), (False, (0, 0), 1),
                                                 (False, (40, 100), 70)])
def test_two_sided_windows(gpu, dtype, fmt, causal, window, sinks):
    if fmt == "same" and window[0] < 0:
        window = (3, window[1])
        sinks = 2
    run_and_check(gpu, [(1, 300), (9, 300), (130, 140), (64, 64)], 4, 2, 64, 16, dtype, fmt, causal=causal, window=window, sinks=sinks)


@pytest.mark.parametrize("dtype,fmt", [ALL[0], ALL[1], ALL[5]])
@pytest.mark.parametrize("softcap", [10.0, 50.0])
def test_softcap(gpu, dtype, fmt, softcap):
    run_and_check(gpu, [(1, 400), (3, 90), (150, 200)], 8, 2, 128, 16, dtype, fmt, softcap=softcap, window=(60, 0), sinks=4)


@pytest.mark.parametrize("scales", ["none", "one", "head", "column"])
def test_scales(gpu, scales):
    run_and_check(gpu, [(1, 400), (3, 90), (150, 200)], 8, 2, 128, 16, torch.bfloat16, "e4m3", scales=scales)


@pytest.mark.parametrize("dtype,fmt", [ALL[0], ALL[5]])
def test_rows_that_see_nothing(gpu, dtype, fmt):
    """More new tokens than keys, sequences without keys, sequences without tokens."""
    run_and_check(gpu, [(30, 10), (1, 0), (0, 0), (3, 0), (0, 20), (5, 1), (200, 100)], 4, 2, 64, 16, dtype, fmt, window=(50, 0), sinks=2)
    run_and_check(gpu, [(1, 0), (1, 5)], 4, 2, 64, 16, dtype, fmt, window=(50, 0), sinks=2)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("window,sinks", [((-1, -1), 0), ((3000, 0), 4)])
def test_long_sequences_split_over_workgroups(gpu, dim, window, sinks):
    out = run_and_check(gpu, [(1, 20011), (1, 37), (1, 5000)], 8, 2, dim, 16, torch.bfloat16, "e4m3", window=window, sinks=sinks)
    again = run_and_check(gpu, [(1, 20011), (1, 37), (1, 5000)], 8, 2, dim, 16, torch.bfloat16, "e4m3", window=window, sinks=sinks)
    assert torch.equal(out, again)                                    # no order of arrival in the sums
    run_and_check(gpu, [(4, 20011), (2, 37), (3, 5000)], 8, 2, dim, 16, torch.float16, "e5m2", window=window, sinks=sinks)


def test_without_a_workspace(gpu, monkeypatch):
    """The C entry point runs unsplit without scratch memory."""
    from flaggems_amd import _C

    class Stingy:
        def __getattr__(self, name):
            return (lambda *a: 0) if name == "fg_cache_attn_workspace_bytes" else getattr(real, name)

    real = _C.lib()
    monkeypatch.setattr(_C, "lib", lambda: Stingy())
    monkeypatch.setattr(importlib.import_module("flaggems_amd.ops.attention"), "_cache_attn_scratch", {})
    run_and_check(gpu, [(1, 9000), (1, 37)], 8, 2, 128, 16, torch.bfloat16, "e4m3")


@pytest.mark.parametrize("q_len", [1, 40])
def test_pages_outside_the_window_are_not_read(gpu, q_len):
    """Pages that neither window nor sinks need are gone: table entries that name no page, and NaN in what is left of the
    pages at the window's edges."""
    lens, page, window, sinks = [(q_len, 800), (q_len, 431)], 16, 100, 4
    q, kc, vc, cu, used, table, ks, vs = make(gpu, lens, 8, 2, 64, page, torch.bfloat16, "e4m3", seed=2)
    for b, (n, k) in enumerate(lens):
        low = k - n - window
        for j in range(sinks, low):
            if j // page > (sinks - 1) // page and (j // page + 1) * page <= low:
                table[b, j // page] = -1 if j % 2 else 1 << 30
            else:
                blk = int(table[b, j // page])
                for c in (kc, vc):
                    c.view(torch.uint8)[blk, j % page] = 0x7f
    out, lse = flag_gems.flash_attn_varlen_func(q, kc, vc, q_len, cu, 800, seqused_k=used, causal=True, window_size=(window, 0), block_table=table,
                                                return_softmax_lse=True, k_descale=ks, v_descale=vs, num_sink_tokens=sinks)
    assert_close(out, lse, O.cache_attention(q, kc, vc, cu, used, table, 64 ** -0.5, True, (window, 0), sinks, 0.0, ks, vs), torch.bfloat16, 64)


@pytest.mark.parametrize("q_len", [1, 50])
def test_bad_tables_give_nan_for_their_sequence_only(gpu, q_len):
    lens = [(q_len, 300), (q_len, 200), (q_len, 280)]
    q, kc, vc, cu, used, table, ks, vs = make(gpu, lens, 4, 2, 64, 16, torch.float16, "e4m3")
    want = O.cache_attention(q, kc, vc, cu, used, table, 0.125, k_scale=ks, v_scale=vs)
    table[0, 3] = kc.shape[0]                                          # names no page
    used[2] = 16 * table.shape[1] + 1                                  # longer than its row of the table
    out = flag_gems.flash_attn_varlen_func(q, kc, vc, q_len, cu, 400, seqused_k=used, causal=True, block_table=table, k_descale=ks, v_descale=vs)
    assert torch.isnan(out[:q_len][-1]).all() and torch.isnan(out[2 * q_len:]).all()
    mid = {k: (v[q_len:2 * q_len] if v.shape[0] == 3 * q_len else v[:, q_len:2 * q_len]) for k, v in want.items()}
    assert_close(out[q_len:2 * q_len], None, mid, torch.float16, 64)


def test_layouts(gpu):
    """q out of a fused projection, out with padded rows, pages of K and V in turn, table rows apart; rows behind the last
    sequence and between out's rows stay as they were."""
    lens, hq, hk, dim, page = [(1, 90), (5, 300), (70, 100)], 8, 2, 64, 16
    q, kc, vc, cu, used, table, ks, vs = make(gpu, lens, hq, hk, dim, page, torch.bfloat16, "e4m3", scales="head")
    ref = O.cache_attention(q, kc, vc, cu, used, table, dim ** -0.5, k_scale=ks, v_scale=vs)
    total = q.shape[0]
    fused = torch.randn(total + 3, hq + 2 * hk, dim, device=gpu).to(torch.bfloat16)
    fused[:total, :hq] = q
    both = torch.stack([kc.view(torch.uint8), vc.view(torch.uint8)], 1).view(torch.float8_e4m3fn)
    wide = torch.full((3, 64), -5, dtype=torch.int32, device=gpu)
    wide[:, :table.shape[1]] = table
    rows = torch.full((total + 3, hq + 1, dim + 8), 9.0, device=gpu, dtype=torch.bfloat16)
    out = rows[:, :hq, :dim]
    k2, v2 = both.unbind(1)
    got, lse = flag_gems.flash_attn_varlen_func(fused[:, :hq], k2, v2, 70, cu, 300, seqused_k=used, causal=True, block_table=wide[:, :table.shape[1]],
                                                out=out, k_descale=ks, v_descale=vs, return_softmax_lse=True)
    assert got is out
    assert_close(out[:total], lse[:, :total], ref, torch.bfloat16, dim)
    assert (rows[total:] == 9).all() and (rows[:, hq:] == 9).all() and (rows[:, :, dim:] == 9).all()


def test_masked_places_hold_the_types_extremes(gpu):
    """NaN and infinities in V and K of keys that a row's block of rows does not see, largest values in keys that it sees."""
    lens = [(1, 100)]
    q, kc, vc, cu, used, table, _, _ = make(gpu, lens, 4, 2, 64, 16, torch.float16, "e5m2", scales="none")
    for j in range(8, 60):
        blk = int(table[0, j // 16])
        vc.view(torch.uint8)[blk, j % 16] = 0x7c                       # +inf
        kc.view(torch.uint8)[blk, j % 16] = 0xfc
    kc.view(torch.uint8)[int(table[0, 70 // 16]), 70 % 16] = 0x7b      # 57344
    q = q * 0.01
    out, lse = flag_gems.flash_attn_varlen_func(q, kc, vc, 1, cu, 100, seqused_k=used, causal=True, window_size=(39, 0), num_sink_tokens=8,
                                                block_table=table, return_softmax_lse=True)
    assert_close(out, lse, O.cache_attention(q, kc, vc, cu, used, table, 0.125, True, (39, 0), 8), torch.float16, 64)


def test_nan_in_a_query_reaches_its_row(gpu):
    lens = [(1, 100), (1, 64)]
    q, kc, vc, cu, used, table, ks, vs = make(gpu, lens, 4, 2, 64, 16, torch.bfloat16, "e4m3")
    q[0, 1, 5] = float("nan")
    out = flag_gems.flash_attn_varlen_func(q, kc, vc, 1, cu, 100, seqused_k=used, causal=True, block_table=table, k_descale=ks, v_descale=vs)
    nan = torch.isnan(out).all(-1).cpu()
    assert nan[0, 1] and int(nan.sum()) == 1 and int(torch.isnan(out).any(-1).sum()) == 1


def test_another_stream_and_a_graph(gpu):
    """Captured once on a side stream with its scratch memory, replayed with new inputs: equal to eager execution, with eager
    calls and synchronizations between the replays."""
    lens = [(1, 5000), (1, 300), (1, 2500), (1, 1)]
    args = make(gpu, lens, 8, 2, 64, 16, torch.bfloat16, "e4m3", scales="head")
    q, kc, vc, cu, used, table, ks, vs = args
    key, value = (torch.randn(4, 2, 64, device=gpu).to(torch.bfloat16) for _ in range(2))
    slots = torch.tensor([int(table[b, 0]) * 16 for b in range(4)], device=gpu)

    def step():
        flag_gems.reshape_and_cache_flash(key, value, kc, vc, slots, "fp8", ks, vs)
        a = flag_gems.flash_attn_varlen_func(q, kc, vc, 1, cu, 5000, seqused_k=used, causal=True, block_table=table, k_descale=ks, v_descale=vs,
                                             window_size=(2000, 0), num_sink_tokens=4)
        b = flag_gems.flash_attn_varlen_func(q, kc, vc, 1, cu, 5000, seqused_k=used, causal=True, block_table=table, k_descale=ks, v_descale=vs)
        k, v = flag_gems.gather_cache_flash(kc, vc, table, cu, 4, k_scale=ks, v_scale=vs)
        return a, b, k, v

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            first = step()
    torch.cuda.current_stream().wait_stream(side)
    eager = step()
    assert all(torch.equal(x, y) for x, y in zip(first, eager))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kept = step()
    for n in range(4):
        g = torch.Generator().manual_seed(n)
        q.copy_(torch.randn(q.shape, generator=g)); key.copy_(torch.randn(key.shape, generator=g)); value.copy_(torch.randn(key.shape, generator=g))
        used.copy_(torch.tensor([5000 - 700 * n, 300 - n, 2500 - 800 * n, 1 + 0 * n], dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        got = [x.clone() for x in kept]
        want = step()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(got, want)), n


def test_large_batches_of_mixed_lengths(gpu):
    random.seed(7)
    lens = [(random.choice([1, 1, 1, 2, 4, 9, 33, 100]), random.randint(100, 700)) for _ in range(24)]
    run_and_check(gpu, lens, 8, 2, 128, 16, torch.bfloat16, "e4m3")
    run_and_check(gpu, lens, 4, 4, 64, 16, torch.float16, "same", window=(150, 0), sinks=4)


def test_custom_op_takes_an_8bit_cache(gpu):
    lens = [(1, 90), (5, 300)]
    q, kc, vc, cu, used, table, ks, vs = make(gpu, lens, 8, 2, 64, 16, torch.bfloat16, "e4m3")
    out, lse = torch.ops.flag_gems.flash_attn_varlen_func(q, kc, vc, 5, cu, 300, None, used, None, 0.0, 0.125, True, [-1, -1], 0.0, None, False,
                                                          False, table, True, None, None, None, ks, vs, 2)
    assert_close(out, lse, O.cache_attention(q, kc, vc, cu, used, table, 0.125, k_scale=ks, v_scale=vs), torch.bfloat16, 64)


def test_more_sequences_than_a_launch_holds(gpu):
    """65535 sequences, one of them a chunk: the chunk kernel takes them in two launches.  Checked against the oracle: the chunk, the
    sequences where the launches meet and the last ones, each a call of the oracle of its own."""
    batch, n, heads, dim = 65535, 520, 64, 64
    g = torch.Generator(device=gpu).manual_seed(3)
    keys = torch.ones(batch, dtype=torch.int32, device=gpu)
    new = torch.ones(batch, dtype=torch.int32, device=gpu)
    at = 40000
    keys[at], new[at] = 600, n
    cu = torch.cat([torch.zeros(1, dtype=torch.int32, device=gpu), new.cumsum(0, dtype=torch.int32)])
    kc, vc = (torch.randn(2048, 1, heads, dim, generator=g, device=gpu).mul(20).to(torch.float8_e4m3fn) for _ in range(2))
    table = torch.randint(0, 2048, (batch, 600), generator=g, device=gpu, dtype=torch.int32)
    q = torch.randn(int(cu[-1]), heads, dim, generator=g, device=gpu).to(torch.bfloat16)
    ks, vs = (torch.rand(batch, 1, generator=g, device=gpu) * 0.04 + 0.03 for _ in range(2))
    out, lse = flag_gems.flash_attn_varlen_func(q, kc, vc, n, cu, 600, seqused_k=keys, causal=True, block_table=table, return_softmax_lse=True,
                                                k_descale=ks, v_descale=vs)
    meet = ((1 << 24) - 1) // (5 * 8) * 8 // heads                    # sequences of the first launch
    assert 0 < meet < batch
    for first, last in ((0, 2), (at, at + 1), (meet - 2, meet + 2), (batch - 2, batch)):
        a, b = int(cu[first]), int(cu[last])
        ref = O.cache_attention(q[a:b], kc, vc, cu[first:last + 1] - a, keys[first:last], table[first:last], dim ** -0.5, k_scale=ks[first:last],
                                v_scale=vs[first:last])
        assert_close(out[a:b], lse[:, a:b], ref, torch.bfloat16, dim)
    assert not torch.isnan(out).any()
