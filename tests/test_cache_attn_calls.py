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
