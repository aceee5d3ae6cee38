"""What the entry points around the 4-bit KV cache refuse for its size, without a GPU: kernels that go through
requests in steps count them in 32 bits."""
import ctypes

import pytest

from csed499ii_amd import _lib

NULL, PTRS = ctypes.c_void_p(0), (ctypes.c_void_p * 1)(0)


@pytest.mark.parametrize("requests", [2 ** 30 + 1, 2 ** 31 - 4096, 2 ** 31 - 1])
def test_more_requests_than_the_kernels_count(built_lib, requests):
    lib = built_lib
    for call in (lambda: lib.marlin_hip_kv4_free_pages(*[NULL] * 5, requests, 1, 16, 8, 0, NULL),
                 lambda: lib.marlin_hip_kv4_compact(PTRS, 1, *[NULL] * 5, requests, 1, 2, 128, 16, 8, -1, 0, NULL),
                 lambda: lib.marlin_hip_kv4_fork(PTRS, 1, *[NULL] * 8, requests, 1, 1, 1, 2, 128, 16, 8, -1, 0, NULL),
                 lambda: lib.marlin_hip_kv4_shared(*[NULL] * 5, requests, 1, 1, 16, 0, NULL)):
        assert call() == _lib.ERR_PROB_SHAPE and "2^30 requests" in _lib.last_error()
