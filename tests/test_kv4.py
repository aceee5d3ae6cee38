"""The 4-bit KV cache without a GPU: what the C entry points refuse before any launch, the
launch plan, and the plain implementation the GPU tests compare with."""
import ctypes

import numpy as np
import pytest
import torch

from csed499ii_amd import _lib, marlin
from tests import kv4_ref as ref

NULL = ctypes.c_void_p(0)


def _attention(lib, tokens=4, requests=4, Hq=8, H=2, D=128, qt=1024, qh=128, page=16, pages=8, width=4, g=-1, max_q=1,
               max_kv=64, scale=1.0, dtype=0):
    return lib.marlin_hip_kv4_attention(NULL, NULL, NULL, NULL, NULL, NULL, NULL, tokens, requests, Hq, H, D, qt, qh,
                                        page, pages, width, g, max_q, max_kv, scale, dtype, 0, NULL)


@pytest.mark.parametrize("change,code", [
    ({"tokens": 0}, _lib.OK), ({"requests": 0}, _lib.OK), ({"max_q": 0}, _lib.OK),
    ({"tokens": -1}, _lib.ERR_PROB_SHAPE), ({"Hq": 9}, _lib.ERR_PROB_SHAPE), ({"Hq": 0}, _lib.ERR_PROB_SHAPE),
    ({"H": 0}, _lib.ERR_PROB_SHAPE), ({"page": 24}, _lib.ERR_PROB_SHAPE), ({"page": 8}, _lib.ERR_PROB_SHAPE),
    ({"page": 512}, _lib.ERR_PROB_SHAPE), ({"pages": 0}, _lib.ERR_PROB_SHAPE),
    ({"pages": 2 ** 28}, _lib.ERR_PROB_SHAPE), ({"width": 2 ** 27}, _lib.ERR_PROB_SHAPE),
    ({"qt": 1001}, _lib.ERR_PROB_SHAPE), ({"scale": 0.0}, _lib.ERR_PROB_SHAPE), ({"scale": -1.0}, _lib.ERR_PROB_SHAPE),
    ({"scale": float("inf")}, _lib.ERR_PROB_SHAPE), ({"max_kv": -1}, _lib.ERR_PROB_SHAPE),
    ({"D": 96}, _lib.ERR_KERN_SHAPE), ({"g": 16}, _lib.ERR_KERN_SHAPE), ({"D": 64, "g": 128}, _lib.ERR_KERN_SHAPE),
    ({"dtype": 2}, _lib.ERR_KERN_SHAPE),
])
def test_attention_codes(built_lib, change, code):
    assert _attention(built_lib, **change) == code
    if code != _lib.OK:
        assert _lib.last_error()


def test_row_and_table_codes(built_lib):
    lib = built_lib
    rows = lambda **c: lib.marlin_hip_kv4_append(  # noqa: E731
        NULL, NULL, NULL, NULL, c.get("tokens", 0), c.get("H", 2), c.get("D", 128), c.get("s", 128), 128, 128, 128,
        c.get("page", 16), 4, c.get("g", -1), c.get("dtype", 0), 0, NULL)
    assert rows() == _lib.OK
    assert rows(tokens=-1) == rows(s=4) == rows(page=17) == rows(H=0) == _lib.ERR_PROB_SHAPE
    assert rows(D=32) == rows(g=8) == rows(dtype=5) == _lib.ERR_KERN_SHAPE
    gather = lambda n, d: lib.marlin_hip_kv4_gather(NULL, NULL, NULL, NULL, n, 2, d, 16, 4, -1, 0, 0, NULL)  # noqa: E731
    assert (gather(0, 128), gather(-1, 128), gather(0, 256)) == (_lib.OK, _lib.ERR_PROB_SHAPE, _lib.ERR_KERN_SHAPE)
    tab = lambda r, page: lib.marlin_hip_kv4_tables(*[NULL] * 8, r, 1, 1, page, 1, 0, NULL)  # noqa: E731
    assert tab(-1, 16) == tab(1, 20) == _lib.ERR_PROB_SHAPE


def test_wrappers_refuse_cpu_tensors(built_lib):
    x = torch.zeros((1, 2, 128), dtype=torch.float16)
    i = torch.zeros(1, dtype=torch.int32)
    cache = marlin.kv4_cache(2, 2, 128, device="cpu")
    for f in (lambda: marlin.kv4_append(x, x, cache, i), lambda: marlin.kv4_gather(cache, i, 128),
              lambda: marlin.kv4_attention(x, cache, i.view(1, 1), i),
              lambda: marlin.kv4_tables(i, i, i, i.view(1, 1), 1, 16)):
        with pytest.raises(RuntimeError, match="no CPU implementation"):
            f()


def test_plan(built_lib):
    """Two workgroups a compute unit where there is that much work, fewer for short caches of few
    heads, and no division (no scratch) where a tile has no step of 32 tokens for each wave."""
    assert marlin.plan_kv4_attention(1, 32, 32, 128, 1, 100) == {"workgroups": 32, "split": False}
    assert marlin.plan_kv4_attention(1, 64, 8, 128, 1, 131072, sms=256) == {"workgroups": 512, "split": True}
    assert marlin.plan_kv4_attention(4096, 64, 8, 128, 1, 131072)["workgroups"] == 512
    assert marlin.plan_kv4_attention(0, 64, 8, 128, 1, 1024)["workgroups"] == 0
    for kv in (1, 256, 257, 1000):
        p = marlin.plan_kv4_attention(1, 8, 8, 128, 1, kv)
        assert p["workgroups"] == 8 * -(-kv // 256) and p["split"] == (kv > 256)
    with pytest.raises(RuntimeError, match="multiple"):
        marlin.plan_kv4_attention(1, 9, 2, 128)


@pytest.mark.parametrize("D,g,T", [(128, -1, 16), (128, 32, 32), (64, 32, 16), (64, -1, 64)])
def test_reference_layout_round_trip(D, g, T):
    """The plain implementation's own layout: every nibble and scale of a block has one place,
    and what is written is read back."""
    G = ref.groups(D, g)
    k, v, ks, vs = ref.places(T, D, G)
    assert sorted(np.concatenate([k, v]).reshape(-1)) == list(range(2 * T * D))
    # (as fp16 places, the scales start after T * D bytes of codes)
    assert sorted(set(np.concatenate([ks, vs]).reshape(-1))) == list(range(T * D // 2, T * D // 2 + 2 * T * G))
    rng = np.random.default_rng(0)
    block = np.zeros(T * (D + 4 * G), np.uint8)
    x, y = rng.standard_normal((T, D)), rng.standard_normal((T, D))
    for o in range(T):
        ref.write_block(block, T, D, G, o, x[o], y[o])
    for got, want in zip(ref.read_block(block, T, D, G), (x, y)):
        c, s = ref.quantize(want, G)
        assert np.array_equal(got, (c - 8) * np.repeat(s, D // G, -1))
        assert np.abs(got - want).max() <= 0.51 * s.max() + 1e-3
