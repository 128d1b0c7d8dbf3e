"""Packed attention in pieces with a workspace that is aligned to 16 bytes and no more, on the GPU."""

from __future__ import annotations

import ctypes

import pytest
import torch

from gemma4_posttrain_jax_amd import _lib, kernels
from gemma4_posttrain_jax_amd.kvcache import key_shape

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("D", [64, 128, 256, 512])
def test_a_workspace_of_16_byte_alignment(D, device):
    """The same bits as with the front end's workspace, and nothing written around it."""

    T, H, R, Sp = 1500, 1, 4, 1536
    g = torch.Generator(device=device).manual_seed(D)
    normal = lambda *s: torch.empty(s, dtype=torch.bfloat16, device=device).normal_(generator=g)  # noqa: E731
    q, k, vt = normal(T, H, R, D) * (2 / D ** 0.5), normal(*key_shape(1, H, Sp, D)), normal(1, H, Sp // 8, D, 8)
    starts = torch.zeros(T, dtype=torch.int32, device=device)
    want = kernels.packed_prefill_attention(q, k, vt, starts, longest=T)
    out = torch.full_like(q, float("nan"))
    a = _lib.G4PackedPrefillArgs(T, H, R, D, 0, Sp, T, starts.data_ptr(), q.data_ptr(), k.data_ptr(), vt.data_ptr(),
                                 out.data_ptr(), None, 0)
    need = _lib.lib().g4_packed_prefill_workspace_size(ctypes.byref(a))
    assert need > 0
    ws = torch.full((need + 128,), 0xA5, dtype=torch.uint8, device=device)
    at = 16 + (-ws.data_ptr()) % 64
    a.workspace, a.workspace_bytes = ws.data_ptr() + at, need
    assert a.workspace % 32 == 16
    torch.cuda.synchronize()
    assert _lib.lib().g4_packed_prefill_attention(ctypes.byref(a), torch.cuda.current_stream().cuda_stream) == _lib.G4_OK
    assert torch.equal(out, want)
    assert bool((ws[:at] == 0xA5).all()) and bool((ws[at + need:] == 0xA5).all())
