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
