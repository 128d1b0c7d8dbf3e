"""The sizes that the verification's launches cannot take are refused before the first of them, on the CPU."""

from __future__ import annotations

import ctypes

import pytest

from gemma4_posttrain_jax_amd import _lib

AT = 1 << 12  # an address that no check before a launch reads


# one looked-up draft per row over 2^30 logits: the first launch takes 2^14 of them per workgroup, the race 2^12
@pytest.mark.parametrize("temperature", [0.7, 1.0])
@pytest.mark.parametrize("dtype", [_lib.G4_DTYPE_BF16, _lib.G4_DTYPE_F32])
def test_a_race_of_2_32_threads_is_refused(temperature, dtype):
    V = 1 << 30
    a = _lib.G4VerifyArgs(dtype=dtype, batch=64, drafts=1, vocab=V, logits=AT, batch_stride=2 * V, row_stride=V, draft_tokens=AT,
                          uniforms=AT, noise=AT, noise_stride=V, temperature=temperature, token_out=AT, count_out=AT, logp_out=AT,
                          workspace=AT, workspace_bytes=1 << 60)
    rc = _lib.lib().g4_verify_draft(ctypes.byref(a), None)
    text = _lib.lib().g4_last_error().decode()
    assert rc == _lib.G4_ERR_UNSUPPORTED and "too many logits" in text, (rc, text)
