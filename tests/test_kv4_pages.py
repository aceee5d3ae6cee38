"""Pages of the 4-bit KV cache without a GPU: what the entry points refuse before any launch."""
import ctypes

import pytest
import torch

from csed499ii_amd import _lib, marlin

NULL = ctypes.c_void_p(0)
PTRS = (ctypes.c_void_p * 1)(0)


def calls(lib, layers=1, requests=1, new=1, pairs=1, free=1, width=4, H=2, D=128, page=16, pages=8, g=-1):
    return {
        "free": lambda: lib.marlin_hip_kv4_free_pages(*[NULL] * 5, requests, width, page, pages, 0, NULL),
        "copy": lambda: lib.marlin_hip_kv4_copy_pages(PTRS, layers, NULL, NULL, pairs, H, D, page, pages, g, 0, NULL),
        "compact": lambda: lib.marlin_hip_kv4_compact(PTRS, layers, *[NULL] * 5, requests, width, H, D, page, pages, g, 0, NULL),
        "fork": lambda: lib.marlin_hip_kv4_fork(PTRS, layers, *[NULL] * 8, requests, new, free, width, H, D, page, pages, g, 0, NULL),
    }


@pytest.mark.parametrize("change,who,code", [
    ({"requests": -1}, "free compact fork", _lib.ERR_PROB_SHAPE), ({"width": -1}, "free compact fork", _lib.ERR_PROB_SHAPE),
    ({"width": 2 ** 27}, "free compact fork", _lib.ERR_PROB_SHAPE), ({"page": 24}, "free copy compact fork", _lib.ERR_PROB_SHAPE),
    ({"pages": 2 ** 28}, "free copy compact fork", _lib.ERR_PROB_SHAPE), ({"pages": 0}, "free compact fork", _lib.ERR_PROB_SHAPE),
    ({"layers": -1}, "copy compact fork", _lib.ERR_PROB_SHAPE), ({"pairs": -1}, "copy", _lib.ERR_PROB_SHAPE),
    ({"new": -1}, "fork", _lib.ERR_PROB_SHAPE), ({"free": -1}, "fork", _lib.ERR_PROB_SHAPE), ({"H": 0}, "copy compact fork", _lib.ERR_PROB_SHAPE),
    ({"H": 32768}, "fork", _lib.ERR_PROB_SHAPE), ({"new": 65537}, "fork", _lib.ERR_PROB_SHAPE),
    ({"H": 2 ** 20, "page": 256}, "copy compact fork", _lib.ERR_PROB_SHAPE), ({"D": 96}, "copy compact fork", _lib.ERR_KERN_SHAPE),
    ({"g": 16}, "copy compact fork", _lib.ERR_KERN_SHAPE), ({"pairs": 0}, "copy", _lib.OK), ({"layers": 0}, "copy", _lib.OK),
])
def test_codes(built_lib, change, who, code):
    for name in who.split():
        assert calls(built_lib, **change)[name]() == code, name


def test_shared_codes(built_lib):
    def call(requests=4, groups=2, width=4, page=16):
        return built_lib.marlin_hip_kv4_shared(*[NULL] * 5, requests, groups, width, page, 0, NULL)

    assert call(requests=0) == call(groups=0) == _lib.OK
    for change in ({"requests": -1}, {"groups": -1}, {"width": -1}, {"width": 2 ** 27}, {"page": 24}, {"groups": 2 ** 20 + 1}):
        assert call(**change) == _lib.ERR_PROB_SHAPE, change


def test_wrappers_refuse(built_lib):
    cache = marlin.kv4_cache(4, 2, 128, device="cpu")
    i = torch.zeros(1, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="no CPU implementation"):
        marlin.kv4_layers([cache], 128)
    with pytest.raises(RuntimeError, match="a cache at least"):
        marlin.kv4_layers([], 128)
    with pytest.raises(RuntimeError, match="no CPU implementation"):
        marlin.kv4_free_pages(i.view(1, 1), i, 4, 16)
    with pytest.raises(TypeError):
        marlin.kv4_copy_pages([cache], i, i)
