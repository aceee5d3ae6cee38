"""Rotary positions without a GPU: frequencies, and what the entry points refuse before any launch."""
import ctypes
import math

import pytest
import torch

from csed499ii_amd import _lib, marlin
from csed499ii_amd.marlin import _rotary

NULL = ctypes.c_void_p(0)


def test_frequencies_are_turns():
    f = marlin.rotary_frequencies(8, device="cpu")
    assert f.dtype == torch.int64 and f.shape == (4,)
    for i, x in enumerate(f.tolist()):
        assert abs((x % 2 ** 64) / 2 ** 64 - 10000.0 ** (-i / 4) / (2 * math.pi)) < 2 ** -52
    # a pair that makes many turns keeps its frequency, one that makes few is divided
    plain, parts = (marlin.rotary_frequencies(128, device="cpu", **k).double() for k in ({}, {"scale": 16.0, "original": 4096}))
    assert (parts[:10] == plain[:10]).all() and torch.allclose(parts[-10:], plain[-10:] / 16, rtol=1e-12)
    assert ((parts <= plain) & (parts >= plain / 16 * (1 - 1e-12))).all()


@pytest.mark.parametrize("kw", [{"rotary_dim": 3}, {"rotary_dim": 0}, {"rotary_dim": 8, "base": 0.0}, {"rotary_dim": 8, "scale": -1.0},
                                {"rotary_dim": 8, "scale": float("nan")},
                                {"rotary_dim": 256, "base": 1e-300}, {"rotary_dim": 8, "scale": 1e-308}, {"rotary_dim": 8, "original": 0},
                                {"rotary_dim": 8, "original": 4096, "slow": 4.0, "fast": 4.0}])
def test_frequencies_refuse(kw):
    with pytest.raises(RuntimeError):
        marlin.rotary_frequencies(device="cpu", **kw)


def rows(lib, tokens=2, heads=2, D=128, r=64, s=128, dtype=0):
    return lib.marlin_hip_rotary(NULL, NULL, NULL, tokens, heads, D, r, 256, s, 256, 128, 0, dtype, 0, NULL)


@pytest.mark.parametrize("change,code", [
    ({"tokens": 0}, _lib.OK), ({"heads": 0}, _lib.OK), ({"tokens": -1}, _lib.ERR_PROB_SHAPE), ({"D": 12, "r": 2}, _lib.ERR_PROB_SHAPE),
    ({"D": 1032}, _lib.ERR_PROB_SHAPE), ({"r": 130}, _lib.ERR_PROB_SHAPE), ({"r": 7}, _lib.ERR_PROB_SHAPE), ({"r": 0}, _lib.ERR_PROB_SHAPE),
    ({"s": 129}, _lib.ERR_PROB_SHAPE), ({"tokens": 2 ** 31 - 1, "heads": 64}, _lib.ERR_PROB_SHAPE), ({"dtype": 2}, _lib.ERR_KERN_SHAPE),
])
def test_row_codes(built_lib, change, code):
    assert rows(built_lib, **change) == code


def append(lib, tokens=2, Hq=4, H=2, D=128, r=64, s=128, page=16, g=-1, dtype=0):
    return lib.marlin_hip_kv4_append_rotary(*[NULL] * 7, tokens, Hq, H, D, r, s, *[128] * 7, page, 4, g, 0, dtype, 0, NULL)


@pytest.mark.parametrize("change,code", [
    ({"tokens": 0}, _lib.OK), ({"tokens": -1}, _lib.ERR_PROB_SHAPE), ({"Hq": -1}, _lib.ERR_PROB_SHAPE), ({"tokens": 2 ** 31 - 1}, _lib.ERR_PROB_SHAPE), ({"H": 0}, _lib.ERR_PROB_SHAPE),
    ({"r": 130}, _lib.ERR_PROB_SHAPE), ({"r": 5}, _lib.ERR_PROB_SHAPE), ({"s": 4}, _lib.ERR_PROB_SHAPE), ({"page": 17}, _lib.ERR_PROB_SHAPE),
    ({"D": 96}, _lib.ERR_KERN_SHAPE), ({"g": 8}, _lib.ERR_KERN_SHAPE), ({"dtype": 3}, _lib.ERR_KERN_SHAPE),
])
def test_append_codes(built_lib, change, code):
    assert append(built_lib, **change) == code


def test_angle_codes(built_lib):
    call = lambda n, p: built_lib.marlin_hip_rotary_angles(NULL, NULL, NULL, n, p, 1.0, 0, NULL)  # noqa: E731
    assert call(0, 4) == call(4, 0) == _lib.OK and call(-1, 4) == call(4, -1) == call(2 ** 26, 64) == _lib.ERR_PROB_SHAPE


def test_wrappers_refuse_cpu_tensors(built_lib):
    x, i = torch.zeros((1, 2, 128), dtype=torch.float16), torch.zeros(1, dtype=torch.int32)
    a, cache = torch.zeros((1, 64, 2), dtype=torch.float64), marlin.kv4_cache(2, 2, 128, device="cpu")
    for f in (lambda: marlin.rotary(x, a), lambda: marlin.rotary_angles(i, torch.zeros(4, dtype=torch.int64)),
              lambda: marlin.kv4_append_rotary(x, x, x, cache, i, a)):
        with pytest.raises(RuntimeError, match="no CPU implementation"):
            f()


def test_overlap_of_strided_rows():
    x = torch.zeros((4, 10, 64), dtype=torch.float16)
    q, k, v = x.split_with_sizes((6, 2, 2), 1)
    assert _rotary._apart(q, k) and _rotary._apart(k, q) and _rotary._apart(v, q)
    assert not _rotary._apart(q, x) and not _rotary._apart(q, q) and not _rotary._apart(x[:, 5:7], k)
    assert _rotary._apart(x[:2], x[2:]) and not _rotary._apart(x[:3], x[2:])
    assert _rotary._apart(x[1:2, 6:], q[:1]) and _rotary._apart(x[:0], x) and not _rotary._apart(x[1:2, :7], x[:, 6:8])
    assert not _rotary._apart(x.transpose(0, 1), x)
