"""GPU parity of attention under a window with sink tokens over 16-bit caches, at the head dims and page sizes that take loads,
paddings and page lookups of their own, and of chunks whose keys are cut into many ranges; against the 64-bit oracle."""
import importlib

import pytest
import torch

from test_gpu_zattn_cache import run_and_check

pytestmark = pytest.mark.gpu
TOKENS = [(1, 1), (1, 31), (1, 33), (1, 700), (3, 129)]
CHUNKS = [(2, 2), (129, 463), (33, 1000), (1, 77), (0, 50), (64, 64)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim", [8, 40, 64, 72, 80, 96, 128, 136, 192, 200, 256])
@pytest.mark.parametrize("lens", [TOKENS, CHUNKS], ids=["tokens", "chunks"])
def test_head_dims(gpu, dtype, dim, lens):
    """8-bit caches take multiples of 16 only; rows of 136 and more elements are loaded where they are used, in two parts."""
    run_and_check(gpu, lens, 8, 2, dim, 16, dtype, "same", window=(90, 0), sinks=3)


@pytest.mark.parametrize("page", [1, 4, 8, 24, 48, 100, 256])
@pytest.mark.parametrize("dim", [64, 128, 200, 256])
@pytest.mark.parametrize("dtype,lens", [(torch.float16, TOKENS), (torch.bfloat16, CHUNKS)], ids=["tokens", "chunks"])
def test_page_sizes(gpu, page, dim, dtype, lens):
    run_and_check(gpu, lens, 6, 2, dim, page, dtype, "same", window=(200, 0), sinks=9)


@pytest.mark.parametrize("dim,page", [(72, 48), (200, 100), (256, 24), (256, 4)])
@pytest.mark.parametrize("softcap,causal,window", [(30.0, True, (120, 0)), (0.0, False, (50, 60))])
def test_soft_cap_and_two_sided_windows(gpu, dim, page, softcap, causal, window):
    run_and_check(gpu, TOKENS[2:], 8, 8, dim, page, torch.bfloat16, "same", causal=causal, window=window, sinks=5, softcap=softcap)
    run_and_check(gpu, CHUNKS, 16, 1, dim, page, torch.float16, "same", causal=causal, window=window, sinks=5, softcap=softcap)


@pytest.mark.parametrize("dim", [200, 256])
@pytest.mark.parametrize("hq,hk", [(8, 2), (5, 5)])
def test_long_sequences_of_wide_heads(gpu, dim, hq, hk):
    """Few sequences over many keys: cut into ranges and merged."""
    run_and_check(gpu, [(1, 9001), (1, 37), (1, 5000)], hq, hk, dim, 16, torch.bfloat16, "same", window=(8000, 0), sinks=4)


@pytest.mark.parametrize("dtype,fmt,window,sinks", [(torch.bfloat16, "e4m3", (-1, -1), 0), (torch.float16, "e5m2", (15000, 0), 4),
                                                    (torch.bfloat16, "same", (15000, 0), 70)])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("lens", [[(40, 20011)], [(40, 20011), (33, 37), (39, 9000)]], ids=["one", "three"])
def test_chunks_in_more_than_eight_ranges(gpu, monkeypatch, dtype, fmt, window, sinks, dim, lens):
    """(A workgroup for each row merges them; up to eight ranges are merged by a wave.)"""
    kept = {}
    monkeypatch.setattr(importlib.import_module("flaggems_amd.ops.attention"), "_cache_attn_scratch", kept)
    out = run_and_check(gpu, lens, 8, 2, dim, 16, dtype, fmt, window=window, sinks=sinks)
    tokens = sum(n for n, _ in lens)
    assert list(kept.values())[0] > 8 * tokens * 8 * (dim + 2) * 4
    again = run_and_check(gpu, lens, 8, 2, dim, 16, dtype, fmt, window=window, sinks=sinks)
    assert torch.equal(out, again)


@pytest.mark.parametrize("lens", [[(1, 700), (1, 33)], [(90, 300), (2, 40)]], ids=["tokens", "chunks"])
@pytest.mark.parametrize("softmax_scale,k_scale,v_scale", [(-0.1, 0.05, 0.05), (0.1, -0.05, -0.04), (-0.1, -0.05, 0.04), (0.0, 0.05, 0.05), (0.1, 0.0, 0.04),
                                                           (0.1, 0.05, 0.0), (1e-3, 5.0, 1e-30), (1e20, 5e-22, 1e30)])
@pytest.mark.parametrize("softcap", [0.0, 20.0])
def test_signs_and_sizes_of_scales(gpu, lens, softmax_scale, k_scale, v_scale, softcap):
    """The kernels move the sign of the score's factor into the query, and a factor of 0 makes every visible key weigh the same."""
    import flag_gems
    from oracle import torch_ref as O
    from test_gpu_zattn_cache import assert_close, make

    q, kc, vc, cu, used, table, _, _ = make(gpu, lens, 8, 2, 64, 16, torch.bfloat16, "e4m3", scales="none")
    ks, vs = torch.tensor([k_scale], device=gpu), torch.tensor([v_scale], device=gpu)
    out, lse = flag_gems.flash_attn_varlen_func(q, kc, vc, max(n for n, _ in lens), cu, max(k for _, k in lens), seqused_k=used, causal=True, block_table=table,
                                                softmax_scale=softmax_scale, softcap=softcap, k_descale=ks, v_descale=vs, return_softmax_lse=True)
    ref = O.cache_attention(q, kc, vc, cu, used, table, softmax_scale, softcap=softcap, k_scale=ks, v_scale=vs)
    # (sum |q| |k| times the factor's size: the oracle's bound takes the factor with its sign)
    size = O.cache_attention(q.abs(), kc.view(torch.uint8).bitwise_and(127).view(kc.dtype), vc, cu, used, table, abs(softmax_scale), k_scale=ks.abs())
    assert_close(out, lse, dict(ref, reach=size["reach"].abs()), torch.bfloat16, 64)
