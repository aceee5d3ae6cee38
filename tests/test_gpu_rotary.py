"""Rotary positions on the GPU against 64-bit plain implementations.

A turned value is computed in fp64 (off by 2^-50 of its terms at most), rounded to fp32 and then
to the row's type: half a step of the type (2^-11, bf16 2^-8; fp16's subnormals 2^-25) and half a
step of fp32 (2^-24) beside it.  A frequency is off by the rounding of a power and a quotient in
fp64 (2^-51 of it, with room) and by 2^-64 of a turn, each times the position."""
import math

import numpy as np
import pytest
import torch

from csed499ii_amd import marlin
from tests.gpu_util import new_stream

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def ints(x):
    return torch.tensor(np.asarray(x), dtype=torch.int32, device=DEV)


def frequencies(r, base=10000.0, scale=1.0, original=None, slow=1.0, fast=32.0):
    f = np.longdouble(base) ** (-np.arange(0, r, 2, dtype=np.longdouble) / r)
    if original is None:
        return f / scale
    m = np.clip((original * f / (2 * np.pi) - slow) / (fast - slow), 0, 1)
    return f * (m + (1 - m) / scale)


def turned(x, angles, interleaved):
    """``x [N, H, D]`` and ``angles [N, pairs, 2]``, both float64 on the CPU."""
    out, r = x.clone(), 2 * angles.shape[1]
    cos, sin = angles[:, None, :, 0], angles[:, None, :, 1]
    lo = torch.arange(0, r, 2) if interleaved else torch.arange(r // 2)
    hi = lo + (1 if interleaved else r // 2)
    a, b = x[..., lo], x[..., hi]
    out[..., lo], out[..., hi] = a * cos - b * sin, b * cos + a * sin
    return out


def near(got, want, x, dtype):
    eps = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}[dtype] + 2.0 ** -24
    tiny = 2.0 ** -25 if dtype == torch.float16 else 2.0 ** -134
    tol = eps * want.abs() + tiny + 2.0 ** -50 * x.abs().amax(-1, keepdim=True) * 2
    err = (got.double().cpu() - want).abs()
    assert (err <= tol).all(), f"worst {(err / tol).max():.3f} of the bound"


@pytest.mark.parametrize("kw", [{}, {"base": 500000.0}, {"scale": 8.0}, {"scale": 16.0, "original": 4096},
                                {"scale": 8.0, "original": 8192, "slow": 1.0, "fast": 4.0}, {"base": 1.5, "scale": 0.01}])
@pytest.mark.parametrize("r", [2, 24, 128])
def test_angles(r, kw):
    pos = np.array([0, 1, 2, 63, 4095, 4096, 131071, 1 << 20, 2 ** 31 - 1, -1, -77, -2 ** 31])
    f = frequencies(r, **kw)
    got = marlin.rotary_angles(ints(pos), marlin.rotary_frequencies(r, device=DEV, **kw), 1.25).cpu().numpy()
    a = pos[:, None].astype(np.longdouble) * f
    bound = np.abs(pos[:, None]) * (f * 2.0 ** -51 + 2 * math.pi * 2.0 ** -64) + 2.0 ** -50
    assert got.shape == (len(pos), r // 2, 2)
    assert (np.abs(got[..., 0] / 1.25 - np.cos(a)) <= bound).all()
    assert (np.abs(got[..., 1] / 1.25 - np.sin(a)) <= bound).all()


def _angles(N, r, seed=0, top=1 << 20):
    rng = np.random.default_rng(seed)
    angles = marlin.rotary_angles(ints(rng.integers(0, top, N)), marlin.rotary_frequencies(r, device=DEV))
    return angles, angles.cpu()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("N,H,D,r", [
    (1, 1, 8, 2), (1, 32, 128, 128), (3, 5, 64, 64), (7, 2, 80, 32), (5, 3, 96, 24), (2, 64, 128, 96), (65, 9, 128, 6),
    (4, 1, 1024, 1024), (2, 3, 1024, 2), (130, 1, 16, 16), (9, 300, 64, 8), (1, 7, 256, 250), (1000, 8, 64, 16),
])
def test_rows(N, H, D, r, interleaved, dtype):
    gen = torch.Generator().manual_seed(N + D + r)
    wide = torch.randn((N, H + 3, D + 8), generator=gen).to(dtype)
    angles, cpu = _angles(N, r)
    on = wide.to(DEV)
    x = on[:, 1:H + 1, :D]  # a view, its rows apart
    want = turned(x.cpu().double(), cpu, interleaved)
    got = marlin.rotary(x, angles, interleaved)
    assert got.is_contiguous() and got.dtype == dtype
    near(got, want, x.cpu().double(), dtype)
    # in place, and into rows of another tensor: the same bits, and nothing beside them
    other = torch.zeros((N, H + 3, D + 8), dtype=dtype, device=DEV)
    assert torch.equal(marlin.rotary(x, angles, interleaved, out=other[:, 2:H + 2, 8:]), got)
    assert not other[:, :2].any() and not other[:, H + 2:].any() and not other[..., :8].any()
    same = marlin.rotary(x, angles, interleaved, out=x)
    assert same is x and torch.equal(x, got)
    wide[:, 1:H + 1, :D] = got.cpu()
    assert torch.equal(on.cpu(), wide)


def test_many_rounds_of_heads_keep_or_share_their_angles():
    """More tokens than the rule's border, so that a workgroup goes through several rounds of heads."""
    N, H, D = 1111, 70, 128
    x = torch.randn((N, H, D), generator=torch.Generator().manual_seed(1)).half()
    for interleaved in (False, True):
        angles, cpu = _angles(N, 64)
        got = marlin.rotary(x.to(DEV), angles, interleaved)
        near(got, turned(x.double(), cpu, interleaved), x.double(), torch.float16)


def test_rotation_back_and_empty():
    x = torch.randn((50, 4, 64), device=DEV).half()
    pos, f = torch.arange(50, device=DEV, dtype=torch.int32), marlin.rotary_frequencies(64, device=DEV)
    y = marlin.rotary(marlin.rotary(x, marlin.rotary_angles(pos, f)), marlin.rotary_angles(-pos, f))
    # two roundings: each 2^-11 of a value that is at most the pair's length
    pair = (x.double()[..., :32] ** 2 + x.double()[..., 32:] ** 2).sqrt().repeat(1, 1, 2)
    assert ((y.double() - x.double()).abs() <= 3 * 2.0 ** -11 * pair + 2.0 ** -24).all()
    assert marlin.rotary(x[:0], marlin.rotary_angles(pos[:0], f)).shape == (0, 4, 64)
    assert marlin.rotary(x[:, :0], marlin.rotary_angles(pos, f)).shape == (50, 0, 64)


def test_infinities_and_nan_stay_in_their_pairs():
    x = torch.ones((1, 1, 64), device=DEV).half()
    x[0, 0, 3], x[0, 0, 40] = float("nan"), float("inf")
    angles, _ = _angles(1, 64)
    y = marlin.rotary(x, angles)[0, 0]
    bad = ~torch.isfinite(y)
    assert sorted(bad.nonzero().flatten().tolist()) == [3, 8, 35, 40]


GEOMETRIES = [(128, -1, 16), (128, 64, 32), (128, 32, 64), (64, -1, 16), (64, 32, 128)]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("D,g,T", GEOMETRIES)
@pytest.mark.parametrize("N,Hq,Hkv,r", [(1, 1, 1, 64), (24, 8, 2, 64), (61, 5, 3, 24), (700, 16, 48, 32), (5, 70, 1, 2)])
def test_append_is_rotary_then_append(D, g, T, dtype, interleaved, N, Hq, Hkv, r):
    gen = torch.Generator().manual_seed(N + D + T)
    x = (torch.randn((N, Hq + 2 * Hkv, D), generator=gen) * torch.rand((N, 1, 1), generator=gen) * 30).to(dtype).to(DEV)
    q, k, v = x.split_with_sizes((Hq, Hkv, Hkv), 1)
    r = min(r * (D // 64), D)
    pages = -(-N // T) + 2
    slots = torch.randperm(pages * T, generator=gen)[:N].int()
    if N > 4:
        slots[3], slots[4] = -1, pages * T + 9
    slots, (angles, _) = slots.to(DEV), _angles(N, r, seed=N)
    before = torch.randint(0, 256, marlin.kv4_cache(pages, Hkv, D, T, g, "cpu").shape, generator=gen, dtype=torch.uint8).to(DEV)
    want, got = before.clone(), before.clone()
    kept = x.clone()
    q_want = marlin.rotary(q, angles, interleaved)
    marlin.kv4_append(marlin.rotary(k, angles, interleaved), v, want, slots, groupsize=g)
    q_got = marlin.kv4_append_rotary(q, k, v, got, slots, angles, groupsize=g, interleaved=interleaved)
    assert torch.equal(q_got, q_want) and torch.equal(got, want) and torch.equal(x, kept)
    # without q, and with q turned where it lies, between its neighbours
    got.copy_(before)
    assert marlin.kv4_append_rotary(None, k, v, got, slots, angles, groupsize=g, interleaved=interleaved) is None
    assert torch.equal(got, want)
    got.copy_(before)
    assert marlin.kv4_append_rotary(q, k, v, got, slots, angles, groupsize=g, interleaved=interleaved, out=q) is q
    assert torch.equal(got, want) and torch.equal(q, q_want) and torch.equal(x[:, Hq:], kept[:, Hq:])


def test_tables_give_the_positions():
    ctx, new, T = [5, 0, 31, 7], [3, 20, 2, 0], 16
    free, table = ints(range(40)), ints(np.full((4, 5), -1))
    got = marlin.kv4_tables(ints(ctx), ints(new), free, table, 30, T, return_positions=True)
    plain = marlin.kv4_tables(ints(ctx), ints(new), free, ints(np.full((4, 5), -1)), 30, T)
    assert len(got) == 5 and all(torch.equal(a, b) for a, b in zip(got, plain) if a.numel() != 30)
    assert got[4].tolist() == [c + i for c, n in zip(ctx, new) for i in range(n)] + [0] * 5


def test_graph_and_other_stream():
    """Replays with new contents, between eager calls, on a stream that is not the default one."""
    N, D = 17, 128
    x = torch.randn((N, 12, D), device=DEV).half()
    pos = torch.arange(N, device=DEV, dtype=torch.int32)
    f, slots = marlin.rotary_frequencies(D, device=DEV), torch.arange(N, device=DEV, dtype=torch.int32)
    cache = marlin.kv4_cache(4, 2, D, device=DEV)
    q, k, v = x.split_with_sizes((8, 2, 2), 1)

    def step():
        return marlin.kv4_append_rotary(q, k, v, cache, slots, marlin.rotary_angles(pos, f))

    side = new_stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        step()
        with torch.cuda.graph(graph, stream=side):
            out = step()
    torch.cuda.synchronize()
    for i in range(4):
        x.copy_(torch.randn_like(x))
        pos.add_(1000 * i)
        graph.replay()
        torch.cuda.synchronize()
        got, bytes_ = out.clone(), cache.clone()
        cache.zero_()
        assert torch.equal(step(), got) and torch.equal(cache, bytes_)
