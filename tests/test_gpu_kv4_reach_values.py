"""Attention, plain, through a window and behind shared prefixes, where scores and values span many orders of
magnitude, against 64 bits, in the kernel of few rows and in that of prompts.

The bound is that of tests/test_gpu_kv4.py, with what lies below fp16's range beside the row's largest p v: a
pass brings that to 2^7, so a token's p v is off by 2^-25 at most, 2^-32 of the largest.  A code is 8 at most."""
import numpy as np
import pytest
import torch

from csed499ii_amd import marlin
from tests import kv4_ref as ref
from tests.test_gpu_kv4 import DEV, _check, _problem, ints
from tests.test_gpu_kv4_edges import WIDE, _set_token
from tests.test_gpu_kv4_reach import attention

pytestmark = pytest.mark.gpu
KERNELS = [(3, 4, 2), (50, 34, 17)]  # new tokens, query and kv heads


def _run(p, g, T, form, window, sinks):
    q, cache, table, kv, cu, _ = p
    q, cache, table, kv, cu = q.to(DEV), torch.from_numpy(cache).to(DEV), ints(table), ints(kv), ints(cu)
    kw = dict(max_q=int(max(np.diff(p[4]))), max_kv=int(p[3].max()), groupsize=g, return_lse=True)
    if form != "shared":
        return marlin.kv4_attention(q, cache, table, kv, cu, **kw, **({"window": window, "sinks": sinks} if form == "window" else {}))
    ctx = ints(p[3] - np.diff(p[4]))
    s = marlin.kv4_shared(table, ctx, ints([0, len(p[3])]), T, cu, always=True)
    assert s.lens.item() > 0
    return marlin.kv4_attention(q, cache, table, kv, cu, context_lens=ctx, shared=s, **kw)


def _want(p, D, T, form, window, sinks):
    reach = (window, sinks) if form == "window" else ()
    return attention(p[0].double().numpy(), *p[1:5], D, p[5], T, *reach)


def _two(n, kv, pages, Hq, Hkv, D, g, T, dtype, seed, **kw):
    """Two requests of the same lengths that share their first pages."""
    p = list(_problem([n, n], [kv, kv], Hq, Hkv, D, g, T, dtype, seed, **kw))
    p[2][1, :pages] = p[2][0, :pages]
    return p


@pytest.mark.parametrize("n,Hq,Hkv", KERNELS)
@pytest.mark.parametrize("window,sinks", [(200, 4), (64, 0), (330, 70)])
@pytest.mark.parametrize("k_gain,v_gain", [(30.0, 1.0), (1.0, 1e-4), (1.0, 3000.0), (6.0, 1e-3), (0.0, 1.0), (1.0, 0.0)])
def test_window_peaked_flat_tiny_and_large(n, Hq, Hkv, window, sinks, k_gain, v_gain):
    D, g, T = 128, 64, 16
    p = _problem([n, n], [700, 90], Hq, Hkv, D, g, T, torch.float16, seed=5, k_gain=k_gain, v_gain=v_gain)
    _check(*_run(p, g, T, "window", window, sinks), _want(p, D, T, "window", window, sinks), torch.float16,
           f"gains {k_gain} {v_gain}", x_max=1000.0 * max(1.0, k_gain) / 30)


@pytest.mark.parametrize("form", ["window", "shared"])
@pytest.mark.parametrize("n,Hq,Hkv", KERNELS)
@pytest.mark.parametrize("order", ["rising", "falling"])
def test_maximum_and_values_that_move(form, n, Hq, Hkv, order):
    """Scores and value scales that rise (or fall) by orders of magnitude along the cache."""
    D, T, kv = 128, 16, 600
    p = _two(n, kv, 33, Hq, Hkv, D, -1, T, torch.float16, 9)
    pl = ref.places(T, D, 1)
    for r in range(2):
        for j in range(33 * r, -(-kv // T)):
            f = 2.0 ** (j * 0.375 - 7) if order == "rising" else 2.0 ** (7 - j * 0.375)
            halves = p[1][p[2][r, j]].view(np.float16)
            for o in range(min(T, kv - j * T)):
                halves[:, pl[2][o]] = np.float16(min(f, 4.0) * 0.3)
                halves[:, pl[3][o]] = np.float16(f)
    _check(*_run(p, -1, T, form, 400, 20), _want(p, D, T, form, 400, 20), torch.float16, order, x_max=400.0)


@pytest.mark.parametrize("n,Hq,Hkv", KERNELS)
@pytest.mark.parametrize("D,g", [(128, -1), (128, 32), (64, 32)])
@pytest.mark.parametrize("form", ["plain", "window", "shared"])
@pytest.mark.parametrize("case", WIDE + ["heavy sink", "weightless zeros first", "nothing but zeros first"])
def test_values_over_many_orders_of_magnitude(case, form, D, g, n, Hq, Hkv):
    T, kv, pages, window, sinks = 32, 400, 10, 330, 4
    p = _two(n, kv, pages, Hq, Hkv, D, g, T, torch.bfloat16, 211)
    p[0] = p[0].abs()  # a token whose codes are all alike has the same sign of score for every row
    q, cache, table, kvs, cu, G = p
    pl = ref.places(T, D, G)

    def scale(tokens, f):
        for t in tokens:
            for page in {table[0, t // T], table[1, t // T]}:
                cache[page].view(np.float16)[:, pl[3][t % T]] *= np.float16(f)

    unit = float(q.double().sum(-1).mean()) / np.sqrt(D)  # of a token of codes 1 and scale 1
    if case.startswith("outlier"):  # no weight (2^-60 or less), the largest scale; the others near the least
        scale(range(kv), 2.0 ** -17)
        _set_token(cache, table, T, D, G, {"first": 0, "inside": 170, "last": kv - n}[case.split()[1]], 0, 80 / (8 * unit), 60000.0)
    elif case == "sink of tiny v":
        _set_token(cache, table, T, D, G, 0, 15, 12 / (7 * unit), 2.0 ** -24)
    elif case == "heavy sink":  # takes nearly all weight, with v as the others'
        _set_token(cache, table, T, D, G, 0, 15, 12 / (7 * unit), 1.0)
    elif case == "zeros first":
        scale(range(150), 0.0)
        scale(range(150, 300), 2.0 ** -20)
        scale(range(300, kv), 3000.0)
    elif case.startswith("weightless zeros"):  # a token that takes nearly all weight and has no v
        _set_token(cache, table, T, D, G, kv - n if case.endswith("last") else 0, 15, 40 / (7 * unit), 0.0)
    elif case == "nothing but zeros first":  # ... and no v for many steps
        scale(range(150), 0.0)
        _set_token(cache, table, T, D, G, 0, 15, 40 / (7 * unit), 0.0)
    else:
        for t in range(kv):
            scale([t], 2.0 ** (-17 + t / 12.5))  # 2^-17 to 2^14.9
    w, ref_lse, weight = _want(p, D, T, form, window, sinks)
    out, lse = _run(p, g, T, form, window, sinks)
    o = out.double().cpu().numpy()
    top = weight.max(-1, keepdims=True)  # >= the largest w_j s_j: some code is not 8
    tol = (2.0 ** -11 + 2.0 ** -13) * weight + 2.0 ** -8 * np.abs(w) + kv * 8 * 2.0 ** -32 * top
    bad = ~(np.abs(o - w) <= tol)
    assert not bad.any(), f"{bad.sum()} of {bad.size} off, worst {np.nanmax(np.abs(o - w) / tol):.2f} of the bound"
    assert np.abs(lse.double().cpu().numpy() - ref_lse).max() <= 2.0 ** -16 * 100


@pytest.mark.parametrize("n,Hq,Hkv,gain", [(3, 4, 2, x) for x in (1.0, 1e4, 1e6, 1e7, 1e9, 1e20)] + [(50, 34, 17, x) for x in (1.0, 1e3)])
@pytest.mark.parametrize("D,g", [(128, -1), (128, 32), (64, 32)])
@pytest.mark.parametrize("form", ["plain", "window", "shared"])
def test_equal_scores_of_any_size(form, D, g, n, Hq, Hkv, gain):
    """Keys that are all alike, values of many sizes: every token that a row sees has the same weight, wherever its
    sums meet, however large the score (in the prompt kernel while fp32 has its fraction: past 10^4 a score's
    rounding shows)."""
    T, kv = 32, 600
    p = _two(n, kv, 10, Hq, Hkv, D, g, T, torch.bfloat16, 3, poison=False)
    k, _, k_at, v_at = ref.places(T, D, p[5])
    rng = np.random.default_rng(0)
    for page in np.unique(p[2][p[2] >= 0]):
        codes, halves = p[1][page], p[1][page].view(np.float16)
        nibbles = np.unique(k // 2)
        codes[:, nibbles] = 0x99  # both codes 1
        for o in range(T):
            halves[:, k_at[o]] = 1.0
            halves[:, v_at[o]] *= np.float16(2.0 ** rng.integers(-6, 6))
    p[0] = (p[0].double() * gain).to(torch.bfloat16)
    _check(*_run(p, g, T, form, 333, 5), _want(p, D, T, form, 333, 5), torch.bfloat16, f"gain {gain}", x_max=100.0 * gain)


@pytest.mark.parametrize("n,Hq,Hkv", KERNELS)
@pytest.mark.parametrize("D,g", [(128, -1), (128, 32), (64, 32)])
@pytest.mark.parametrize("form,pos", [("window", 2), ("window", 85), ("window", 200), ("window", 397), ("shared", 100), ("shared", 397)])
def test_nan_of_a_seen_row_without_weight_shows(form, pos, D, g, n, Hq, Hkv):
    """A NaN scale of V whose token's weight is zero in fp32, among the sinks, where windows begin, in the
    midst and at the end: the rows that see it are NaN, no others."""
    T, kv, window, sinks = 32, 399, 313, 4
    p = _two(n, kv, 10, Hq, Hkv, D, g, T, torch.float16, 221)
    p[0] = p[0].abs()
    unit = float(p[0].double().sum(-1).mean()) / np.sqrt(D)
    _set_token(p[1], p[2], T, D, p[5], pos, 0, 300 / (8 * unit), np.nan)
    out, _ = _run(p, g, T, form, window, sinks)
    nan = torch.isnan(out).flatten(1).cpu()
    at = torch.arange(kv - n, kv)
    seen = pos <= at
    if form == "window":
        seen &= (pos > at - window) | torch.tensor(pos < sinks)
    for r in range(2):  # (the second request has the first ten pages in common, or none of that token)
        mine, sees = nan[r * n:(r + 1) * n], seen & (r == 0 or pos < 320)
        assert mine[sees].all() and not mine[~sees].any(), r
