"""Attention over the 4-bit KV cache through a sliding window with sinks, and over prefixes that requests
share, against 64-bit plain implementations.

The bounds are those of tests/test_gpu_kv4.py: an output is off by 2^-11 of sum_j w_j |v_jd| (p v in fp16; 2^-13
more for fp32 sums, exp2 and the scores), and by its own rounding.  A shared prefix adds two products and a sum
in fp32 to that, of what both passes left: within the same 2^-13."""
import math

import numpy as np
import pytest
import torch

from csed499ii_amd import marlin
from tests import kv4_ref as ref
from tests.gpu_util import new_stream
from tests.test_gpu_kv4 import GEOMETRIES, _check, _problem

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def ints(x):
    return torch.tensor(np.asarray(x), dtype=torch.int32, device=DEV)


def attention(q, cache, table, kv_lens, cu, D, G, T, window=None, sinks=0, ctx=None):
    """As ``kv4_ref.attention``, with a window; positions start at ``ctx``."""
    N, Hq, _ = q.shape
    num_pages, H, _ = cache.shape
    out, weight = np.zeros((N, Hq, D)), np.zeros((N, Hq, D))
    lse = np.full((N, Hq), -np.inf)
    for i in range(len(kv_lens)):
        kv, n = min(int(kv_lens[i]), table.shape[1] * T), int(cu[i + 1] - cu[i])
        past = int(kv_lens[i]) - n if ctx is None else int(ctx[i])
        blocks = [ref.read_block(cache[p, :].reshape(H, -1)[h], T, D, G) if 0 <= p < num_pages else None
                  for h in range(H) for p in table[i, :-(-kv // T)]]
        for h in range(H):
            mine = blocks[h * (len(blocks) // H):(h + 1) * (len(blocks) // H)]
            there = np.repeat([b is not None for b in mine], T)[:kv].astype(bool) if mine else np.zeros(0, bool)
            zero = np.zeros((T, D))
            k = np.concatenate([zero if b is None else b[0] for b in mine])[:kv] if mine else np.zeros((0, D))
            v = np.concatenate([zero if b is None else b[1] for b in mine])[:kv] if mine else np.zeros((0, D))
            j = np.arange(kv)
            for t in range(n):
                p = past + t
                seen = there & (j <= p)
                if window is not None:
                    seen &= (j > p - window) | (j < sinks)
                if not seen.any():
                    continue
                for hq in range(h * Hq // H, (h + 1) * Hq // H):
                    x = k[seen] @ q[cu[i] + t, hq] / math.sqrt(D)
                    m = x.max()
                    w = np.exp(x - m)
                    out[cu[i] + t, hq] = w @ v[seen] / w.sum()
                    weight[cu[i] + t, hq] = w @ np.abs(v[seen]) / w.sum()
                    lse[cu[i] + t, hq] = m + math.log(w.sum())
    return out, lse, weight


# ---- windows ----


def _window(p, g, window, sinks, one=False, **kw):
    q, cache, table, kv, cu, G = p
    kw.setdefault("max_q", int(max(np.diff(cu), default=1)))
    kw.setdefault("max_kv", int(kv.max(initial=0)))
    return marlin.kv4_attention(q.to(DEV), torch.from_numpy(cache).to(DEV), ints(table), ints(kv), None if one else ints(cu),
                                groupsize=g, return_lse=True, window=window, sinks=sinks, **kw)


WINDOWS = [(1, 0), (1, 1), (5, 3), (31, 32), (32, 0), (33, 4), (64, 33), (65, 70), (128, 4), (500, 64), (5000, 1), (2 ** 31, 2 ** 31)]
ONE = [([1], [1], 1, 1), ([1] * 4, [31, 32, 33, 0], 8, 1), ([1] * 3, [700, 1, 97], 20, 2), ([1] * 2, [513, 1025], 34, 2)]


@pytest.mark.parametrize("window,sinks", WINDOWS)
@pytest.mark.parametrize("D,g,T", GEOMETRIES)
def test_window_single_tokens(D, g, T, window, sinks):
    for q_lens, kv_lens, Hq, Hkv in ONE:
        dtype = torch.bfloat16 if len(kv_lens) == 2 else torch.float16
        p = _problem(q_lens, kv_lens, Hq, Hkv, D, g, T, dtype, seed=sum(kv_lens) + D)
        want = attention(p[0].double().numpy(), *p[1:5], D, p[5], T, window, sinks)
        _check(*_window(p, g, window, sinks, one=True), want, dtype, f"D={D} g={g} T={T} kv={kv_lens} window={window} sinks={sinks}")


MANY = [([3, 1, 5], [3, 40, 70], 4, 2), ([17, 0, 1], [33, 5, 64], 2, 1), ([5] * 2, [330, 7], 8, 1),
        ([7, 2], [4, 300], 2, 2),  # more new tokens than are cached: rows that see nothing, or only sinks
        ([64, 1, 3], [200, 513, 3], 4, 4), ([97, 40], [97, 600], 3, 1)]


@pytest.mark.parametrize("window,sinks", [(1, 0), (4, 2), (33, 4), (64, 0), (100, 70), (300, 1), (2 ** 31, 5)])
@pytest.mark.parametrize("D,g,T", GEOMETRIES)
def test_window_several_tokens(D, g, T, window, sinks):
    for q_lens, kv_lens, Hq, Hkv in MANY:
        dtype = torch.bfloat16 if len(kv_lens) == 2 else torch.float16
        p = _problem(q_lens, kv_lens, Hq, Hkv, D, g, T, dtype, seed=sum(kv_lens) + D)
        want = attention(p[0].double().numpy(), *p[1:5], D, p[5], T, window, sinks)
        _check(*_window(p, g, window, sinks), want, dtype, f"D={D} g={g} T={T} q={q_lens} kv={kv_lens} window={window} sinks={sinks}")


@pytest.mark.parametrize("window,sinks", [(1, 0), (30, 4), (64, 64), (200, 0), (257, 5), (5000, 3)])
@pytest.mark.parametrize("D,g,T", [(128, -1, 16), (128, 32, 64), (64, 32, 128), (64, -1, 16)])
@pytest.mark.parametrize("q_lens,kv_lens,Hq,Hkv", [([300], [300], 2, 2), ([170, 1, 257], [900, 300, 257], 3, 1), ([40, 300], [1300, 500], 8, 1)])
def test_window_prompts(D, g, T, q_lens, kv_lens, Hq, Hkv, window, sinks):
    dtype = torch.bfloat16 if len(kv_lens) == 2 else torch.float16
    p = _problem(q_lens, kv_lens, Hq, Hkv, D, g, T, dtype, seed=sum(kv_lens) + D)
    want = attention(p[0].double().numpy(), *p[1:5], D, p[5], T, window, sinks)
    _check(*_window(p, g, window, sinks), want, dtype, f"window={window} sinks={sinks}")


@pytest.mark.parametrize("n", [1, 40, 200])
def test_window_reads_no_page_outside(n):
    """Pages that no row's window reaches may be gone: entries of -1, or pages of NaN."""
    D, T, kv, window, sinks = 128, 16, 1500, 100, 20
    p = list(_problem([n], [kv], 4, 2, D, -1, T, torch.float16, seed=n))
    want = attention(p[0].double().numpy(), *p[1:5], D, 1, T, window, sinks)
    first = kv - n - window + 1
    gone = [j for j in range(-(-kv // T)) if j * T >= sinks and (j + 1) * T <= first]
    assert len(gone) > 60
    p[2][0, gone[::2]] = -1
    for j in gone[1::2]:
        p[1][p[2][0, j]].view(np.float16)[:] = np.nan
    _check(*_window(p, -1, window, sinks), want, torch.float16, "gone")


def test_window_positions_past_the_table():
    """The table is full: new tokens have no page, and see what lies in their window and the sinks."""
    D, T = 64, 16
    p = list(_problem([20, 5], [64, 64], 4, 2, D, -1, T, torch.float16, seed=3, poison=False))
    ctx = np.array([60, 200])
    kv = np.minimum(ctx + [20, 5], 64)
    for window, sinks in ((30, 3), (10, 0), (1, 64), (150, 2)):
        want = attention(p[0].double().numpy(), p[1], p[2], kv, p[4], D, 1, T, window, sinks, ctx=ctx)
        got = marlin.kv4_attention(p[0].to(DEV), torch.from_numpy(p[1]).to(DEV), ints(p[2]), ints(kv), ints(p[4]), 20, 64,
                                   return_lse=True, window=window, sinks=sinks, context_lens=ints(ctx))
        _check(*got, want, torch.float16, f"window={window} sinks={sinks}")


@pytest.mark.parametrize("q_lens,kv_lens", [([1] * 3, [9000, 3000, 20]), ([5] * 2, [9000, 6000]), ([300], [6000])])
def test_wide_window_is_plain_attention(q_lens, kv_lens):
    """A window as wide as all positions: the same, within the order of sums."""
    D, T = 128, 16
    p = _problem(q_lens, kv_lens, 8, 1, D, -1, T, torch.float16, seed=8)
    a, la = _window(p, -1, 10 ** 6, 0)
    b, lb = marlin.kv4_attention(p[0].to(DEV), torch.from_numpy(p[1]).to(DEV), ints(p[2]), ints(p[3]), ints(p[4]),
                                 max_q=max(q_lens), max_kv=max(kv_lens), return_lse=True)
    assert (a.float() - b.float()).abs().max() <= 2 ** -9 * b.float().abs().max() and (la - lb).abs().max() < 1e-4
    for _ in range(3):
        assert torch.equal(_window(p, -1, 10 ** 6, 0)[0], a)


def test_window_of_many_requests():
    """More than a launch takes; a window across which divided tiles meet."""
    D, T, R = 64, 16, 1100
    rng = np.random.default_rng(0)
    kv_lens = rng.integers(0, 120, R).tolist()
    p = _problem([1] * R, kv_lens, 2, 1, D, -1, T, torch.float16, seed=1)
    want = attention(p[0].double().numpy(), *p[1:5], D, 1, T, 40, 4)
    _check(*_window(p, -1, 40, 4, one=True), want, torch.float16, "many")
    q = np.ones(R, int)
    q[::100] = 90
    kv_lens = np.maximum(kv_lens, q).tolist()
    p = _problem(q.tolist(), kv_lens, 2, 1, D, -1, T, torch.float16, seed=2)
    want = attention(p[0].double().numpy(), *p[1:5], D, 1, T, 40, 4)
    _check(*_window(p, -1, 40, 4), want, torch.float16, "many, some long")


# ---- shared prefixes ----


def _forked(groups, tails, q_lens, Hq, Hkv, D, g, T, dtype, seed):
    """Requests in groups (of so many) behind prefixes of whole pages: ``groups`` [(prefix pages, requests)], own
    tokens and new tokens of each request."""
    kv_lens, common = [], []
    for pages, n in groups:
        for _ in range(n):
            kv_lens.append(pages * T + tails[len(kv_lens)])
            common.append(pages)
    p = list(_problem(q_lens, kv_lens, Hq, Hkv, D, g, T, dtype, seed))
    i = 0
    for pages, n in groups:
        for r in range(i + 1, i + n):
            m = min(pages, p[2].shape[1])
            p[2][r, :m] = p[2][i, :m]
        i += n
    cu_groups = np.concatenate([[0], np.cumsum([n for _, n in groups])])
    return p, cu_groups


def _shared(p, cu_groups, g, T, one=False, ctx=None, **kw):
    q, cache, table, kv, cu, G = p
    ctx = ints(kv - np.diff(cu) if ctx is None else ctx)
    cu = None if one else ints(cu)
    table, kv_ = ints(table), ints(kv)
    s = marlin.kv4_shared(table, ctx, ints(cu_groups), T, cu, always=True)  # (two passes of the smallest, too)
    kw.setdefault("max_q", int(max(np.diff(p[4]), default=1)))
    kw.setdefault("max_kv", int(kv.max(initial=0)))
    return s, marlin.kv4_attention(q.to(DEV), torch.from_numpy(cache).to(DEV), table, kv_, cu, groupsize=g, return_lse=True,
                                   context_lens=ctx, shared=s, **kw)


@pytest.mark.parametrize("D,g,T", GEOMETRIES)
@pytest.mark.parametrize("Hq,Hkv", [(4, 2), (9, 1)])
def test_shared_single_tokens(D, g, T, Hq, Hkv):
    scale = max(1, 64 // T)
    groups = [(3 * scale, 4), (0, 2), (1, 1), (2, 3)]
    tails = [1, 20, 2 * T, T + 1, 5, 40, 7, T, 1, 130]
    p, cu_groups = _forked(groups, tails, [1] * 10, Hq, Hkv, D, g, T, torch.float16, seed=D + T)
    want = attention(p[0].double().numpy(), *p[1:5], D, p[5], T)
    s, (out, lse) = _shared(p, cu_groups, g, T, one=True)
    _check(out, lse, want, torch.float16, f"D={D} g={g} T={T}")
    assert s.lens.tolist() == [3 * scale * T, 0, 0, 2 * T]


@pytest.mark.parametrize("D,g,T", GEOMETRIES)
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_shared_several_tokens(D, g, T, dtype):
    groups = [(2, 3), (300 // T + 1, 2), (1, 2)]
    q_lens = [3, 1, 5, 40, 2, 0, 9]
    tails = [3, 11, T + 5, 60, 2, 0, 9]
    p, cu_groups = _forked(groups, tails, q_lens, 4, 2, D, g, T, dtype, seed=D + T)
    want = attention(p[0].double().numpy(), *p[1:5], D, p[5], T)
    s, (out, lse) = _shared(p, cu_groups, g, T)
    _check(out, lse, want, dtype, f"D={D} g={g} T={T}")
    assert s.lens.tolist() == [2 * T, (300 // T + 1) * T, 0]  # (of the last group one request has no new tokens)


@pytest.mark.parametrize("groups,n,Hq,Hkv,q", [([(70, 40)], 40, 8, 1, 1), ([(40, 150)], 150, 4, 2, 2), ([(20, 2), (30, 3)], 5, 6, 2, 90),
                                              ([(64, 20), (1, 20), (33, 24)], 64, 8, 2, 1)])
@pytest.mark.parametrize("D,g", [(128, -1), (128, 32), (64, 32)])
def test_shared_many_rows(groups, n, Hq, Hkv, q, D, g):
    """Groups whose rows go to the prompt kernel, and passes that divide their tokens."""
    T = 16
    rng = np.random.default_rng(n)
    q_lens = [int(x) for x in rng.integers(1, q + 1, n)]
    tails = [a + int(x) for a, x in zip(q_lens, rng.integers(0, 60, n))]
    p, cu_groups = _forked(groups, tails, q_lens, Hq, Hkv, D, g, T, torch.float16, seed=n + D)
    want = attention(p[0].double().numpy(), *p[1:5], D, p[5], T)
    s, (out, lse) = _shared(p, cu_groups, g, T, one=q == 1)
    _check(out, lse, want, torch.float16, f"{groups}")
    assert (s.lens > 0).all()
    for _ in range(3):
        assert torch.equal(_shared(p, cu_groups, g, T, one=q == 1)[1][0], out)


def test_shared_what_is_shared():
    """Groups that share less than they say, rows that differ, empty and padded requests, borders past the requests."""
    T, P = 16, 8
    table = np.arange(12 * P, dtype=np.int32).reshape(12, P)
    table[1, :5] = table[0, :5]
    table[2, :3] = table[0, :3]
    table[3, 1:] = table[0, 1:]  # the first page differs: shares nothing
    table[6, :] = table[5, :]
    table[7, :] = table[5, :]
    table[9, :2] = table[8, :2] = -1
    ctx = [100, 90, 90, 100, 50, 128, 40, 0, 64, 64, 16, 15]
    find = lambda cu_groups, cu=None: marlin.kv4_shared(ints(table), ints(ctx), ints(cu_groups), T, None if cu is None else ints(cu))  # noqa: E731
    s = find([0, 4, 5, 8, 12])
    assert s.lens.tolist() == [48, 0, 32, 32]
    assert s.plan[13:].tolist() == [48, 48, 48, 0, 0, 32, 32, 0, 32, 32, 0, 0]
    s = find([0, 2, 2, 50])
    assert s.lens.tolist() == [80, 0, 0] and s.plan[10:12].tolist() == [80, 80]
    s = find([5, 7])
    assert s.lens.tolist() == [32] and s.plan[4:].tolist() == [0] * 5 + [32, 32] + [0] * 5
    cu = np.concatenate([[0], np.cumsum([1, 0, 2, 1] + [1] * 8)])
    s = find([0, 4, 12], cu)
    assert s.lens.tolist() == [48, 0] and s.plan[7:11].tolist() == [48, 0, 48, 0]
    assert s.plan[4:7].tolist() == [0, 4, 12]
    assert find([0]).lens.numel() == 0


@pytest.mark.parametrize("n", [1, 3, 30])
def test_far_pages(n):
    """Pages whose byte offset passes 32 bits, through a window and behind a prefix, turned as they are written."""
    D, T, H, G, R = 128, 256, 8, 2, 4
    pages = 17000  # 4.6 GB
    cache = torch.zeros((pages, H, T * (D + 4)), dtype=torch.uint8, device=DEV)
    assert cache.numel() > 2 ** 32
    gen = torch.Generator().manual_seed(n)
    k, v = (torch.randn((7 * T, H, D), generator=gen).half().to(DEV) for _ in range(2))
    angles = marlin.rotary_angles(torch.arange(7 * T, dtype=torch.int32, device=DEV), marlin.rotary_frequencies(D, device=DEV))
    marlin.kv4_append_rotary(None, k, v, cache, ints(np.arange(7 * T) + (pages - 7) * T), angles)
    small = cache[-7:].cpu().numpy()
    want_small = marlin.kv4_cache(7, H, D, T, device=DEV)
    marlin.kv4_append(marlin.rotary(k, angles), v, want_small, ints(np.arange(7 * T)))
    assert torch.equal(cache[-7:], want_small)
    table = np.array([[0, 1, 2, 3 + r] for r in range(R)])  # three pages shared, the last one each request's own
    kv, cu = np.array([3 * T + 9 + 60 * r + n for r in range(R)]), np.arange(R + 1) * n
    q = torch.randn((R * n, G * H, D), generator=gen).half()
    far = ints(table + pages - 7)
    kw = dict(cu_q=ints(cu), max_q=n, max_kv=int(kv.max()), return_lse=True, context_lens=ints(kv - n))
    want = attention(q.double().numpy(), small, table, kv, cu, D, 1, T)
    s = marlin.kv4_shared(far, ints(kv - n), ints([0, R]), T, ints(cu), always=True)
    assert s.lens.tolist() == [3 * T]
    _check(*marlin.kv4_attention(q.to(DEV), cache, far, ints(kv), shared=s, **kw), want, torch.float16, f"{n} tokens, shared")
    want = attention(q.double().numpy(), small, table, kv, cu, D, 1, T, 100, 5)
    _check(*marlin.kv4_attention(q.to(DEV), cache, far, ints(kv), window=100, sinks=5, **kw), want, torch.float16, f"{n} tokens, window")


@pytest.mark.parametrize("form", ["shared", "window"])
@pytest.mark.parametrize("n", [4, 40])
def test_strided_rows_and_tokens_past_max_q(form, n):
    """q a slice of wider rows, out given; a request's tokens past max_q keep what out held."""
    D, T, R, Hq, H = 128, 16, 12, 8, 2
    p, cu_groups = _forked([(20, R)], [n + 3 + i for i in range(R)], [n] * R, Hq, H, D, -1, T, torch.float16, seed=n)
    q, cache, table, kv, cu = p[0].to(DEV), torch.from_numpy(p[1]).to(DEV), ints(p[2]), ints(p[3]), ints(p[4])
    wide = torch.randn((R * n, Hq + 5, D + 8), device=DEV).half()
    wide[:, 2:2 + Hq, :D] = q
    reach = {"window": 50, "sinks": 3} if form == "window" else {"shared": marlin.kv4_shared(table, kv - n, ints(cu_groups), T, cu, always=True)}
    want = attention(p[0].double().numpy(), *p[1:5], D, 1, T, *((50, 3) if form == "window" else ()))
    out = torch.full((R * n, Hq, D), 7.0, dtype=torch.float16, device=DEV)
    most = n - 1
    got, lse = marlin.kv4_attention(wide[:, 2:2 + Hq, :D], cache, table, kv, cu, max_q=most, max_kv=int(p[3].max()), out=out,
                                    return_lse=True, context_lens=kv - n, **reach)
    assert got.data_ptr() == out.data_ptr()
    rows = torch.tensor([t % n < most for t in range(R * n)])
    assert (out[~rows] == 7.0).all()
    _check(got[rows], lse[rows], [x[rows.numpy()] for x in want], torch.float16, f"{form}, {n} tokens")


def test_shared_of_nothing():
    cache = marlin.kv4_cache(4, 2, 128, device=DEV)
    table, none, q = torch.zeros((0, 3), dtype=torch.int32, device=DEV), ints([]), torch.zeros((0, 4, 128), dtype=torch.float16, device=DEV)
    for cu_groups in ([0], [0, 0]):
        s = marlin.kv4_shared(table, none, ints(cu_groups), 16, always=True)
        assert marlin.kv4_attention(q, cache, table, none, context_lens=none, shared=s).shape == q.shape


def test_shared_in_one_pass_where_two_do_not_pay():
    """Few samples: the bits of a call without the prefix.  Many: two passes, other sums of the same."""
    D, T = 128, 16
    for R, H, same in ((4, 2, True), (64, 32, False)):
        p, cu_groups = _forked([(80, R)], [1 + i % 30 for i in range(R)], [1] * R, H, H, D, -1, T, torch.float16, seed=8)
        q, cache, table, kv = p[0].to(DEV), torch.from_numpy(p[1]).to(DEV), ints(p[2]), ints(p[3])
        kw = dict(max_kv=int(p[3].max()), context_lens=kv - 1, return_lse=True)
        plain = marlin.kv4_attention(q, cache, table, kv, **kw)
        s = marlin.kv4_shared(table, kv - 1, ints(cu_groups), T)
        assert s.lens.tolist() == [1280]
        got = marlin.kv4_attention(q, cache, table, kv, shared=s, **kw)
        assert all(torch.equal(a, b) for a, b in zip(plain, got)) == same
        always = marlin.kv4_attention(q, cache, table, kv, shared=s._replace(always=True), **kw)
        assert same or all(torch.equal(a, b) for a, b in zip(always, got))
        want = attention(p[0].double().numpy(), *p[1:5], D, 1, T)
        for out, lse in (got, always):
            _check(out, lse, want, torch.float16, f"{R} requests")


def test_shared_prefix_of_many_requests():
    """Several rounds of requests of one group, and more groups than a launch of attention takes."""
    T, D, R = 16, 64, 2300
    for cu_groups in ([0, R], list(range(0, R + 1, 2))):
        p, _ = _forked([(2, R)], [1 + i % 5 for i in range(R)], [1] * R, 1, 1, D, -1, T, torch.float16, seed=1)
        want = attention(p[0].double().numpy(), *p[1:5], D, 1, T)
        s, (out, lse) = _shared(p, cu_groups, -1, T, one=True)
        _check(out, lse, want, torch.float16, "many")
        assert (s.lens == 32).all()


@pytest.mark.parametrize("one", [True, False])
def test_shared_missing_pages_padding_and_nan(one):
    """Shared pages that are none, a padded request, a NaN in the prefix, rows of no request left alone."""
    T, D = 16, 128
    n = [1] * 5 if one else [3, 1, 4, 1, 2]
    p, cu_groups = _forked([(6, 5)], [x + 9 for x in n], n, 4, 2, D, -1, T, torch.float16, seed=5)
    p[2][:, 2], p[2][:, 4] = -1, 10 ** 6
    want = attention(p[0].double().numpy(), *p[1:5], D, 1, T)
    s, (out, lse) = _shared(p, cu_groups, -1, T, one=one)
    assert s.lens.tolist() == [96]
    _check(out, lse, want, torch.float16, "missing")
    p[3][3] = 0  # a padded request: sees nothing
    ctx = p[3] - n
    ctx[3] = 0
    want = attention(p[0].double().numpy(), p[1], p[2], p[3], p[4], D, 1, T, ctx=ctx)
    _check(*_shared(p, cu_groups, -1, T, one=one, ctx=ctx)[1], want, torch.float16, "padding")
    pl = ref.places(T, D, 1)
    p[1][p[2][0, 1], 0].view(np.float16)[pl[3][7]] = np.nan  # a seen NaN of V, head 0
    out, _ = _shared(p, cu_groups, -1, T, one=one, ctx=ctx)[1]
    rows = [t for r in range(5) if r != 3 for t in range(p[4][r], p[4][r + 1])]
    assert torch.isnan(out[rows][:, :2]).all() and not torch.isnan(out[:, 2:]).any()
    if not one:
        wide = torch.cat([p[0], p[0][:3]]).to(DEV)  # three rows behind the last request
        out = torch.full(wide.shape, 7.0, dtype=torch.float16, device=DEV)
        table, kv, cu, ctx = ints(p[2]), ints(p[3]), ints(p[4]), ints(ctx)
        s = marlin.kv4_shared(table, ctx, ints(cu_groups), T, cu, always=True)
        marlin.kv4_attention(wide, torch.from_numpy(p[1]).to(DEV), table, kv, cu, max_q=4, context_lens=ctx, shared=s, out=out)
        assert (out[-3:] == 7.0).all()


@pytest.mark.parametrize("k_gain,v_gain", [(30.0, 1.0), (1.0, 1e-4), (1.0, 3000.0), (0.0, 1.0)])
def test_shared_peaked_flat_tiny_and_large(k_gain, v_gain):
    D, T = 128, 16
    p = list(_problem([1] * 40, [20 * T + 5] * 40, 8, 1, D, 64, T, torch.float16, seed=4, k_gain=k_gain, v_gain=v_gain))
    p[2][1:, :20] = p[2][:1, :20]
    want = attention(p[0].double().numpy(), *p[1:5], D, 2, T)
    s, (out, lse) = _shared(p, [0, 40], 64, T, one=True)
    assert s.lens.tolist() == [320]
    _check(out, lse, want, torch.float16, f"gains {k_gain} {v_gain}", x_max=1000.0 * max(1.0, k_gain) / 30)


def test_shared_and_window_in_graphs_and_refusals():
    D, T = 128, 16
    p, cu_groups = _forked([(40, 6)], [9] * 6, [1] * 6, 8, 2, D, -1, T, torch.float16, seed=6)
    q, cache, table, kv = p[0].to(DEV), torch.from_numpy(p[1]).to(DEV), ints(p[2]), ints(p[3])
    ctx, groups = kv - 1, ints(cu_groups)

    def step():
        s = marlin.kv4_shared(table, ctx, groups, T, always=True)
        return (marlin.kv4_attention(q, cache, table, kv, context_lens=ctx, shared=s, max_kv=700),
                marlin.kv4_attention(q, cache, table, kv, context_lens=ctx, window=70, sinks=4, max_kv=700))

    side = new_stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        step()
        with torch.cuda.graph(graph, stream=side):
            out = step()
    torch.cuda.synchronize()
    for i in range(4):
        q.copy_(torch.randn_like(q))
        kv.fill_(649 - 3 * i), ctx.fill_(648 - 3 * i)
        graph.replay()
        torch.cuda.synchronize()
        got = [x.clone() for x in out]
        with torch.cuda.stream(side):
            again = step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, again))
    s = marlin.kv4_shared(table, ctx, groups, T)
    call = lambda **kw: marlin.kv4_attention(q, cache, table, kv, **kw)  # noqa: E731
    for kw, what in (({"shared": s}, "context_lens"), ({"shared": s, "context_lens": ctx, "window": 5}, "not both"), ({"shared": s, "context_lens": ctx, "sinks": 2}, "not both"), ({"window": 0}, "window"),
                     ({"window": 4, "sinks": -1}, "sinks"), ({"sinks": 4}, "sinks")):
        with pytest.raises(RuntimeError, match=what):
            call(**kw)
    with pytest.raises(RuntimeError, match="shared is of"):
        marlin.kv4_attention(q[:5], cache, table[:5].contiguous(), kv[:5], context_lens=ctx[:5], shared=s)
    with pytest.raises(TypeError):
        call(shared=ctx, context_lens=ctx)
    for a in ((table, ctx[:3], groups, T), (table, ctx, groups[:0], T), (table, ctx, groups, 24), (table.long(), ctx, groups, T)):
        with pytest.raises(RuntimeError):
            marlin.kv4_shared(*a)
