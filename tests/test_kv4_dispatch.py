"""The 4-bit KV cache's entry points on the CPU: what they refuse, and what they launch
(tests/fake_hip.cpp stands in for the HIP runtime)."""
import ctypes

import pytest

from csed499ii_amd import _lib

NULL = ctypes.c_void_p(0)


def attention(lib, at, tokens, requests, q_heads, kv_heads, head_dim, max_q, max_kv, cu_q, groupsize=-1):
    """One call with operands at address ``at``, which is never read on the host."""
    p = ctypes.c_void_p(at)
    return lib.marlin_hip_kv4_attention(p, p, p, p, p if cu_q else NULL, p, NULL, tokens, requests, q_heads, kv_heads,
                                        head_dim, q_heads * head_dim, head_dim, 16, 1 << 16, 1 << 14, groupsize, max_q,
                                        max_kv, 1.0, 0, 0, ctypes.c_void_p(64))


def test_one_token_a_request_needs_as_many_tokens(built_lib):
    """Without cu_q request i is token i: fewer tokens than requests would be read past q."""
    assert attention(built_lib, 0, 3, 4, 8, 2, 128, 1, 64, False) == _lib.ERR_PROB_SHAPE
    assert "cu_q" in _lib.last_error()
