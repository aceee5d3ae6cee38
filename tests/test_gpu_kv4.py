"""The 4-bit KV cache on the GPU against 64-bit plain implementations (tests/kv4_ref.py).

Attention's bound per output: the second product's operand p v is rounded to fp16, so an
output is off by at most 2^-11 sum_j w_j |v_jd| (w: softmax) beside its own rounding (2^-11,
bf16 2^-8); fp32 sums, exp2 and the scores' own error get another 2^-13 of that sum for scores up to
some tens.  Codes, scales, slots and tables are exact."""
import numpy as np
import pytest
import torch

from csed499ii_amd import marlin
from tests import kv4_ref as ref

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
GEOMETRIES = [(128, -1, 16), (128, 64, 32), (128, 32, 64), (64, -1, 16), (64, 32, 128), (128, -1, 256)]


def ints(x):
    return torch.tensor(np.asarray(x), dtype=torch.int32, device=DEV)


# ---- tables ----


@pytest.mark.parametrize("ctx,new,num_free,P,T,pad", [
    ([0], [1], 4, 3, 16, 0),
    ([0], [0], 4, 3, 16, 2),
    ([15, 16, 17, 0], [1, 1, 1, 1], 8, 4, 16, 0),
    ([5, 0, 31, 32], [40, 0, 1, 33], 16, 6, 16, 3),
    ([5, 0, 31, 32], [40, 0, 1, 33], 3, 6, 16, 0),       # the free list runs out
    ([30, 70], [50, 10], 16, 4, 16, 5),                  # past the table's width
    ([-3, 4], [-2, 5], 8, 2, 32, 0),                     # negative lengths count as zero
    ([7], [300], 32, 8, 64, 0),
    ([100, 200], [9, 9], 8, 0, 16, 0),                   # a table of no pages
    ([3, 3], [20, 20], 0, 4, 16, 0),                     # no free page at all
])
def test_tables_small(ctx, new, num_free, P, T, pad):
    rng = np.random.default_rng(len(ctx) + P)
    free = rng.permutation(1000)[:num_free].astype(np.int32)
    table = rng.integers(1000, 2000, (len(ctx), P)).astype(np.int32)
    N = sum(max(n, 0) for n in new) + pad
    want = ref.tables(ctx, new, free, table, N, T)
    t = ints(table)
    got = marlin.kv4_tables(ints(ctx), ints(new), ints(free), t, N, T)
    for name, g, w in zip(("slots", "cu", "kv", "used", "table"), (*got, t), want):
        assert np.array_equal(g.cpu().numpy(), w), name


@pytest.mark.parametrize("R,most,T", [(1, 9000, 16), (1023, 7, 16), (1024, 9, 32), (1025, 1, 16), (2500, 40, 64),
                                      (3000, 1, 16)])
def test_tables_many(R, most, T):
    """Several rounds of requests, several workgroups of tokens, requests without new tokens."""
    rng = np.random.default_rng(R)
    ctx, new = rng.integers(0, 500, R), rng.integers(0, most + 1, R)
    new[R // 3:R // 3 + 40] = 0
    P = -(-(500 + most) // T)
    free = rng.permutation(1 << 20)[:int(new.sum()) // T + 2 * R].astype(np.int32)
    table = rng.integers(0, 1 << 20, (R, P)).astype(np.int32)
    N = int(new.sum())
    want = ref.tables(ctx, new, free, table, N, T)
    t = ints(table)
    got = marlin.kv4_tables(ints(ctx), ints(new), ints(free), t, N, T)
    for name, g, w in zip(("slots", "cu", "kv", "used", "table"), (*got, t), want):
        assert np.array_equal(g.cpu().numpy(), w), name


def test_tables_fewer_slots_than_tokens_and_no_request():
    t = ints(np.full((2, 4), -1))
    slots, cu, kv, used = marlin.kv4_tables(ints([0, 0]), ints([20, 20]), ints(range(8)), t, 25, 16)
    assert slots.cpu().tolist() == list(range(20)) + [32, 33, 34, 35, 36]
    assert cu.cpu().tolist() == [0, 20, 40] and used.item() == 4
    assert t.cpu().tolist() == [[0, 1, -1, -1], [2, -1, -1, -1]]  # the page past the map is not written
    empty = torch.empty(0, dtype=torch.int32, device=DEV)
    slots, cu, kv, used = marlin.kv4_tables(empty, empty, empty, torch.empty((0, 3), dtype=torch.int32, device=DEV), 3, 16)
    assert slots.cpu().tolist() == [-1] * 3 and cu.cpu().tolist() == [0] and kv.numel() == 0 and used.item() == 0


# ---- rows in and out ----


def _rows(N, H, D, dtype, gen):
    """k and v as views of a fused projection's output, with zeros, ties, tiny and large groups."""
    x = torch.randn((N, 3 * H + 1, D), generator=gen)
    x[:, 1::7] *= 1e-4
    x[:, 2::5] *= 300
    x[0::3, 3::4] = 0
    x[1::4, :, : D // 2] = torch.randint(-15, 16, (x[1::4].shape[0], x.shape[1], D // 2), generator=gen) * 0.5  # ties
    x = x.to(dtype).to(DEV)
    return x[:, 1:H + 1], x[:, 2 * H + 1:]


@pytest.mark.parametrize("D,g,T", GEOMETRIES)
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("N,H", [(1, 1), (7, 3), (61, 2)])
def test_append_and_gather_exact(D, g, T, dtype, N, H):
    gen = torch.Generator().manual_seed(N + D + T)
    G, pages = ref.groups(D, g), -(-N // T) + 3
    k, v = _rows(N, H, D, dtype, gen)
    slots = torch.randperm(pages * T, generator=gen)[:N].int()
    slots[N // 2] = -1 if N > 1 else slots[0]
    if N > 4:
        slots[3] = pages * T + 5  # past the last page
    cache = torch.randint(0, 256, (pages, H, T * (D + 4 * G)), generator=gen, dtype=torch.uint8)
    want = cache.numpy().copy()
    kn, vn = k.double().cpu().numpy(), v.double().cpu().numpy()
    for t in range(N):
        s = int(slots[t])
        if 0 <= s < pages * T:
            for h in range(H):
                ref.write_block(want[s // T, h], T, D, G, s % T, kn[t, h], vn[t, h])
    dev_cache = cache.to(DEV)
    marlin.kv4_append(k, v, dev_cache, slots.to(DEV), groupsize=g)
    got = dev_cache.cpu().numpy()
    assert np.array_equal(got, want), "cache bytes"
    gk, gv = marlin.kv4_gather(dev_cache, slots.to(DEV), D, groupsize=g, dtype=dtype)
    for t in range(N):
        s = int(slots[t])
        for h in range(H):
            rk = rv = np.zeros((T, D))
            if 0 <= s < pages * T:
                rk, rv = ref.read_block(want[s // T, h], T, D, G)
            for got_row, r in ((gk[t, h], rk), (gv[t, h], rv)):
                w = torch.from_numpy(r[s % T].copy()).to(dtype)
                assert torch.equal(got_row.cpu(), w), (t, h)


def test_append_infinities_and_nan():
    """Scales saturate, an infinity takes the largest code, a NaN stays in its group."""
    D, T = 128, 16
    k = torch.ones((3, 1, D), dtype=torch.float16)
    k[0, 0, 5], k[0, 0, 6] = float("inf"), float("-inf")
    k[1, 0, 70] = float("nan")
    v = torch.ones((3, 1, D)).bfloat16()
    v[0, 0, 0] = 3e38
    for x in (k, v.clone()):
        x = x.to(DEV)
        cache = marlin.kv4_cache(1, 1, D, T, 64, device=DEV)
        marlin.kv4_append(x, x, cache, ints([0, 1, 2]), groupsize=64)
        for out in marlin.kv4_gather(cache, ints([0, 1, 2]), D, groupsize=64, dtype=torch.bfloat16):
            out = out.float().cpu()[:, 0]
            if x.dtype == torch.float16:
                assert out[0, 5] == torch.tensor(7 * 65504.0).bfloat16().float() and out[0, 6] == torch.tensor(-8 * 65504.0).bfloat16().float()
                assert torch.isnan(out[1, 64:]).all() and torch.isfinite(out[1, :64]).all()
            else:
                assert out[0, 0] == torch.tensor(7 * 65504.0).bfloat16().float() and (out[0, 1:64] == 0).all()
            assert (out[2] == out[2, 0]).all() and abs(out[2, 0] - 1) < 0.07


# ---- attention ----


def _problem(q_lens, kv_lens, Hq, Hkv, D, g, T, dtype, seed, k_gain=1.0, v_gain=1.0, poison=True):
    gen = torch.Generator().manual_seed(seed)
    G, R, N = ref.groups(D, g), len(q_lens), sum(q_lens)
    pages = [-(-n // T) for n in kv_lens]
    size = sum(pages) + 3
    cache = ref.random_cache(size, Hkv, T, D, G, gen, k_gain, v_gain)
    order, at = torch.randperm(size, generator=gen).tolist(), 0
    table = np.full((R, max(pages + [1])), -1, np.int32)
    pl = ref.places(T, D, G)
    for i, n in enumerate(pages):
        table[i, :n] = order[at:at + n]
        at += n
        if poison and kv_lens[i] % T:  # slots past the last token: scales NaN and infinite
            halves = cache[table[i, n - 1]].view(np.float16)
            for o in range(kv_lens[i] % T, T):
                halves[:, pl[2][o]] = np.nan if o % 2 else np.inf
                halves[:, pl[3][o]] = np.inf if o % 3 else np.nan
    q = torch.randn((N, Hq + 2, D), generator=gen).to(dtype)[:, 1:Hq + 1]
    cu = np.concatenate([[0], np.cumsum(q_lens)])
    return q, cache, table, np.asarray(kv_lens), cu, G


def _check(got, lse, want, dtype, what, x_max=40.0):
    out, ref_lse, weight = want
    o = got.double().cpu().numpy()
    own = 2.0 ** -11 if dtype == torch.float16 else 2.0 ** -8
    tol = (2.0 ** -11 + 2.0 ** -13) * weight + own * np.abs(out) + 2.0 ** -24
    bad = ~(np.abs(o - out) <= tol)
    assert not bad.any(), f"{what}: {bad.sum()} of {bad.size} off, worst {np.nanmax(np.abs(o - out) / tol):.2f} of the bound"
    if lse is not None:
        m = lse.double().cpu().numpy()
        none = np.isinf(ref_lse)
        assert np.array_equal(np.isneginf(m), none), f"{what}: rows that see nothing"
        # scores: 128 products summed in fp32, exp2's argument at up to x_max log2 units
        assert np.abs(m[~none] - ref_lse[~none]).max(initial=0.0) <= 2.0 ** -16 * (1 + x_max), f"{what}: lse"


def _run(p, g, dtype, **kw):
    q, cache, table, kv, cu, G = p
    one = kw.pop("one", False)
    kw.setdefault("max_q", int(max(np.diff(cu), default=1)))
    kw.setdefault("max_kv", int(kv.max(initial=0)))
    return marlin.kv4_attention(q.to(DEV), torch.from_numpy(cache).to(DEV), ints(table), ints(kv),
                                None if one else ints(cu), groupsize=g, return_lse=True, **kw)


DECODE = [
    ([1], [1], 1, 1), ([1], [2], 4, 4), ([1] * 3, [15, 16, 17], 4, 2), ([1] * 4, [31, 32, 33, 0], 8, 1),
    ([1] * 2, [127, 129], 3, 1), ([1] * 2, [700, 1], 20, 2), ([1], [1337], 16, 1), ([1] * 2, [513, 1025], 34, 2),
]


@pytest.mark.parametrize("D,g,T", GEOMETRIES)
@pytest.mark.parametrize("q_lens,kv_lens,Hq,Hkv", DECODE)
def test_single_tokens(D, g, T, q_lens, kv_lens, Hq, Hkv):
    dtype = torch.bfloat16 if len(kv_lens) == 2 else torch.float16
    p = _problem(q_lens, kv_lens, Hq, Hkv, D, g, T, dtype, seed=sum(kv_lens) + D)
    want = ref.attention(p[0].double().numpy(), *p[1:5], D, p[5], T)
    out, lse = _run(p, g, dtype, one=True)
    _check(out, lse, want, dtype, f"D={D} g={g} T={T} kv={kv_lens}")


SEVERAL = [
    ([2], [2], 1, 1), ([3, 1, 5], [3, 40, 70], 4, 2), ([17, 0, 1], [33, 5, 64], 2, 1), ([5] * 2, [130, 7], 8, 1),
    ([33], [33], 6, 3), ([7, 2], [4, 300], 2, 2),  # seven new tokens of which four are cached: rows that see nothing
    ([64, 1, 3], [200, 513, 3], 4, 4), ([130], [259], 2, 1), ([97, 40], [97, 900], 3, 1),
]


@pytest.mark.parametrize("D,g,T", GEOMETRIES)
@pytest.mark.parametrize("q_lens,kv_lens,Hq,Hkv", SEVERAL)
def test_several_tokens(D, g, T, q_lens, kv_lens, Hq, Hkv):
    dtype = torch.bfloat16 if len(kv_lens) == 2 else torch.float16
    p = _problem(q_lens, kv_lens, Hq, Hkv, D, g, T, dtype, seed=sum(kv_lens) + D)
    want = ref.attention(p[0].double().numpy(), *p[1:5], D, p[5], T)
    out, lse = _run(p, g, dtype)
    _check(out, lse, want, dtype, f"D={D} g={g} T={T} q={q_lens} kv={kv_lens}")


@pytest.mark.parametrize("q_lens,kv_lens", [([1, 1], [1200, 300]), ([40, 200], [1200, 300])])
@pytest.mark.parametrize("k_gain,v_gain", [(30.0, 1.0), (1.0, 1e-4), (1.0, 3000.0), (6.0, 1e-3), (0.0, 1.0), (1.0, 0.0)])
def test_peaked_flat_tiny_and_large(q_lens, kv_lens, k_gain, v_gain):
    """Scores up to hundreds (one token takes all), flat ones, values near fp16's limits."""
    D, g, T = 128, 64, 16
    p = _problem(q_lens, kv_lens, 4, 2, D, g, T, torch.float16, seed=5, k_gain=k_gain, v_gain=v_gain)
    want = ref.attention(p[0].double().numpy(), *p[1:5], D, p[5], T)
    out, lse = _run(p, g, torch.float16)
    _check(out, lse, want, torch.float16, f"gains {k_gain} {v_gain}", x_max=1000.0 * max(1.0, k_gain) / 30)


@pytest.mark.parametrize("n", [1, 30])
@pytest.mark.parametrize("order", ["rising", "falling"])
def test_maximum_and_values_that_move(n, order):
    """Scores and value scales that rise (or fall) by orders of magnitude along the cache, so
    that every step changes the reference."""
    D, T, kv = 128, 16, 900
    p = list(_problem([n], [kv], 2, 1, D, -1, T, torch.float16, seed=9))
    table, cache = p[2], p[1]
    pl = ref.places(T, D, 1)
    for j in range(-(-kv // T)):
        f = 2.0 ** (j / 4 - 7) if order == "rising" else 2.0 ** (7 - j / 4)
        halves = cache[table[0, j]].view(np.float16)
        for o in range(min(T, kv - j * T)):
            halves[:, pl[2][o]] = np.float16(min(f, 4.0) * 0.3)
            halves[:, pl[3][o]] = np.float16(f)
    want = ref.attention(p[0].double().numpy(), *p[1:5], D, 1, T)
    out, lse = _run(p, -1, torch.float16)
    _check(out, lse, want, torch.float16, order, x_max=400.0)


@pytest.mark.parametrize("q_lens", [[1, 1, 1], [20, 3, 33]])
def test_missing_pages_are_left_out(q_lens):
    """Entries that are no page (negative, past the pool) anywhere in the table, one request
    without any page: as if the tokens were not there."""
    D, T = 128, 16
    p = list(_problem(q_lens, [200, 90, 64], 4, 2, D, -1, T, torch.float16, seed=3))
    p[2][0, 3], p[2][0, 7], p[2][1, 0] = -1, 10 ** 6, -7
    p[2][2, :] = -1
    want = ref.attention(p[0].double().numpy(), *p[1:5], D, 1, T)
    assert np.isneginf(want[1][-1]).all()
    out, lse = _run(p, -1, torch.float16)
    _check(out, lse, want, torch.float16, "missing pages")


@pytest.mark.parametrize("max_kv", [1, 100, 5000, 1 << 20])
@pytest.mark.parametrize("n", [1, 40])
def test_any_plan_computes_the_same(max_kv, n):
    """The planned length only decides the split, whatever the real lengths are."""
    D, T = 128, 32
    p = _problem([n, n], [1500, 90], 4, 2, D, -1, T, torch.float16, seed=21)
    want = ref.attention(p[0].double().numpy(), *p[1:5], D, 1, T)
    out, lse = _run(p, -1, torch.float16, max_kv=max_kv)
    _check(out, lse, want, torch.float16, f"max_kv={max_kv}")


def test_scale_out_and_lengths_past_the_table():
    D, T = 64, 16
    p = list(_problem([1, 1], [48, 32], 2, 2, D, -1, T, torch.float16, seed=31, poison=False))
    want = ref.attention(p[0].double().numpy(), *p[1:5], D, 1, T, scale=0.5)
    q = p[0].to(DEV)
    out = torch.full(q.shape, float("nan"), dtype=torch.float16, device=DEV)
    kv = p[3].copy()
    kv[0] = 10 ** 9  # the table covers 48: cut there
    got = marlin.kv4_attention(q, torch.from_numpy(p[1]).to(DEV), ints(p[2]), ints(kv), scale=0.5, out=out)
    assert got is out
    _check(out, None, want, torch.float16, "scale")


def test_same_bits_run_to_run_and_row_by_row():
    """A split call's result does not depend on the order in which workgroups arrive, and a
    request's rows do not depend on the others of the batch (one plan)."""
    D, T = 128, 16
    p = _problem([1] * 3, [4000, 700, 2900], 8, 1, D, -1, T, torch.float16, seed=41)
    first, lse = _run(p, -1, torch.float16, one=True)
    assert marlin.plan_kv4_attention(3, 8, 1, D, 1, 4000)["split"]
    for _ in range(5):
        again, lse2 = _run(p, -1, torch.float16, one=True)
        assert torch.equal(first, again) and torch.equal(lse, lse2)


def test_nan_of_a_seen_row_shows_and_stays_where_it_is():
    """A NaN scale reaches the rows that see its token and no others."""
    D, T = 128, 16
    p = _problem([6], [40], 2, 1, D, -1, T, torch.float16, seed=51)
    pl = ref.places(T, D, 1)
    page, o = p[2][0, 36 // T], 36 % T  # position 36: tokens 2 .. 5 of the six see it
    p[1][page].view(np.float16)[:, pl[3][o]] = np.nan
    out, _ = _run(p, -1, torch.float16)
    nan = torch.isnan(out).flatten(1)
    assert nan[2:].all() and not nan[:2].any()


def test_far_pages_of_a_long_cache():
    """Pages whose byte offset passes 32 bits: written, read back and attended to."""
    D, T, H = 128, 256, 8
    pages = 17000  # 4.6 GB
    cache = torch.zeros((pages, H, T * (D + 4)), dtype=torch.uint8, device=DEV)
    assert cache.numel() > 2 ** 32
    gen = torch.Generator().manual_seed(61)
    k, v = (torch.randn((300, H, D), generator=gen).half().to(DEV) for _ in range(2))
    table = ints([[pages - 1, pages - 2]])
    slots = torch.cat([torch.arange(256) + (pages - 1) * T, torch.arange(44) + (pages - 2) * T]).int().to(DEV)
    marlin.kv4_append(k, v, cache, slots)
    gk, gv = marlin.kv4_gather(cache, slots, D)
    small = cache[-2:].cpu().numpy()
    for i, (page, at) in enumerate(((1, 0), (0, 256))):
        rk, rv = ref.read_block(small[page, 5], T, D, 1)
        m = min(256, 300 - at)
        assert np.array_equal(gk[at:at + m, 5].double().cpu().numpy(), rk[:m].astype(np.float16).astype(np.float64))
    for n in (1, 60):
        q = torch.randn((n, 16, D), generator=gen).half()
        want = ref.attention(q.double().numpy(), small, np.array([[1, 0]]), [300], [0, n], D, 1, T)
        out, lse = marlin.kv4_attention(q.to(DEV), cache, table, ints([300]), ints([0, n]), max_q=n, return_lse=True)
        _check(out, lse, want, torch.float16, f"far pages, {n} rows")


def test_a_step_in_a_graph_and_on_another_stream():
    """Tables, append and attention of a step captured on a side stream, replayed between
    eager work, equal the eager results; the stream's scratch is sized by an eager call."""
    D, T, H, Hq, R = 128, 16, 2, 8, 3
    gen = torch.Generator().manual_seed(71)
    ctx, new = ints([600, 31, 0]), ints([1, 1, 1])
    free, size = ints(range(40, 60)), 64
    cache0 = torch.from_numpy(ref.random_cache(size, H, T, D, 1, gen)).to(DEV)
    table0 = torch.full((R, 40), -1, dtype=torch.int32)
    table0[0, :38], table0[1, :2] = torch.arange(38), torch.tensor([38, 39])
    table0 = table0.to(DEV)
    q, k, v = (torch.randn((R, h, D), generator=gen).half().to(DEV) for h in (Hq, H, H))
    cache, table = cache0.clone(), table0.clone()

    def step():
        slots, cu, kv, used = marlin.kv4_tables(ctx, new, free, table, R, T)
        marlin.kv4_append(k, v, cache, slots)
        return marlin.kv4_attention(q, cache, table, kv, cu, max_q=1, max_kv=640)

    want = step().clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        eager = step()
    side.synchronize()
    assert torch.equal(eager, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        out = step()
    for _ in range(4):
        cache.copy_(cache0)
        table.copy_(table0)
        out.fill_(float("nan"))
        marlin.kv4_attention(q, cache0, table0, ctx)  # eager work of another length in between
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
    # a stream without scratch: captured unsplit, the same product
    fresh = torch.cuda.Stream()
    graph2 = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph2, stream=fresh):
        out2 = step()
    graph2.replay()
    torch.cuda.synchronize()
    assert (out2.float() - want.float()).abs().max() <= 2.0 ** -9 * want.float().abs().max()


def test_empty_calls():
    D, T = 128, 16
    cache = marlin.kv4_cache(4, 2, D, T, device=DEV)
    none = torch.empty((0, 2, D), dtype=torch.float16, device=DEV)
    marlin.kv4_append(none, none, cache, ints([]))
    assert marlin.kv4_gather(cache, ints([]), D)[0].shape == (0, 2, D)
    out = marlin.kv4_attention(none, cache, torch.empty((0, 3), dtype=torch.int32, device=DEV), ints([]))
    assert out.shape == (0, 2, D)
    q = torch.ones((2, 2, D), dtype=torch.float16, device=DEV)
    out, lse = marlin.kv4_attention(q, cache, torch.empty((2, 0), dtype=torch.int32, device=DEV), ints([5, 0]),
                                    return_lse=True)
    assert (out == 0).all() and torch.isneginf(lse).all()


def test_refusals():
    D, T = 128, 16
    cache = marlin.kv4_cache(4, 2, D, T, device=DEV)
    rows = torch.zeros((3, 2, D), dtype=torch.float16, device=DEV)
    slots, table, kv = ints([0, 1, 2]), ints([[0], [1], [2]]), ints([3, 3, 3])

    def no(match, f, *a, **kw):
        with pytest.raises((RuntimeError, TypeError), match=match):
            f(*a, **kw)

    no("page_size", marlin.kv4_cache, 4, 2, D, 24, device=DEV)
    no("kernels for", marlin.kv4_cache, 4, 2, 96, T, device=DEV)
    no("kernels for", marlin.kv4_cache, 4, 2, 64, T, 128, device=DEV)
    no("GPU tensor", marlin.kv4_append, rows.cpu(), rows, cache, slots)
    no("fp16 or bf16", marlin.kv4_append, rows.float(), rows.float(), cache, slots)
    no("heads", marlin.kv4_append, rows[:, :1], rows[:, :1], cache, slots)
    no("whole page", marlin.kv4_append, rows, rows, cache, slots, groupsize=32)
    no("slots has", marlin.kv4_append, rows, rows, cache, slots[:2])
    no("int32", marlin.kv4_append, rows, rows, cache, slots.long())
    no("k is", marlin.kv4_append, rows, rows[:2], cache, slots)
    no("contiguous rows", marlin.kv4_append, rows.transpose(1, 2).contiguous().transpose(1, 2), rows, cache, slots)
    no("contiguous rows", marlin.kv4_append, torch.zeros((3, 2, D + 4), dtype=torch.float16, device=DEV)[..., 4:], rows, cache, slots)
    no("uint8", marlin.kv4_append, rows, rows, cache.int(), slots)
    no("dtype", marlin.kv4_gather, cache, slots, D, dtype=torch.float32)
    no("pass cu_q", marlin.kv4_attention, rows[:2], cache, table, kv)
    no("cu_q has", marlin.kv4_attention, rows, cache, table, kv, ints([0, 1]))
    no("block_table", marlin.kv4_attention, rows, cache, table[:2], kv)
    no("multiple", marlin.kv4_attention, torch.zeros((3, 3, D), dtype=torch.float16, device=DEV), cache, table, kv)
    no("positive", marlin.kv4_attention, rows, cache, table, kv, scale=0.0)
    no("positive", marlin.kv4_attention, rows, cache, table, kv, scale=float("nan"))
    no("out must be", marlin.kv4_attention, rows, cache, table, kv, out=rows.float())
    no("requests", marlin.kv4_tables, kv, kv[:2], slots, table, 3, T)
    no("page_size", marlin.kv4_tables, kv, kv, slots, table, 3, 20)
    no("negative", marlin.kv4_tables, kv, kv, slots, table, -1, T)


# ---- many rows: the prompt kernel (more rows a head than the split kernel's, more than a few heads) ----


PROMPTS = [
    ([170, 1, 3], [200, 513, 3], 6, 6),          # beside requests that are the split kernel's
    ([300, 170, 290], [300, 330, 290], 6, 6),    # no short request: one launch
    ([200, 2], [190, 700], 18, 9),               # rows that see nothing
    ([41], [1200], 68, 17),                      # one block of rows, divided over its tokens
    ([90, 0, 1, 90], [400, 0, 70, 90], 10, 5),
]


@pytest.mark.parametrize("D,g,T", GEOMETRIES)
@pytest.mark.parametrize("q_lens,kv_lens,Hq,Hkv", PROMPTS)
def test_prompts(D, g, T, q_lens, kv_lens, Hq, Hkv):
    dtype = torch.bfloat16 if len(kv_lens) == 3 else torch.float16
    p = _problem(q_lens, kv_lens, Hq, Hkv, D, g, T, dtype, seed=sum(kv_lens) + D)
    want = ref.attention(p[0].double().numpy(), *p[1:5], D, p[5], T)
    out, lse = _run(p, g, dtype)
    _check(out, lse, want, dtype, f"D={D} g={g} T={T} q={q_lens} kv={kv_lens}")


@pytest.mark.parametrize("k_gain,v_gain", [(30.0, 1.0), (1.0, 1e-4), (1.0, 3000.0), (6.0, 1e-3), (0.0, 1.0), (1.0, 0.0)])
def test_prompts_peaked_flat_tiny_and_large(k_gain, v_gain):
    D, g, T = 128, 64, 16
    p = _problem([90, 170], [500, 300], 10, 10, D, g, T, torch.float16, seed=6, k_gain=k_gain, v_gain=v_gain)
    want = ref.attention(p[0].double().numpy(), *p[1:5], D, p[5], T)
    out, lse = _run(p, g, torch.float16)
    _check(out, lse, want, torch.float16, f"gains {k_gain} {v_gain}", x_max=1000.0 * max(1.0, k_gain) / 30)


def test_prompts_with_missing_pages_and_nan():
    D, T = 128, 16
    p = list(_problem([170, 3, 180], [260, 90, 200], 6, 6, D, -1, T, torch.float16, seed=4))
    p[2][0, 3], p[2][0, 7], p[2][1, 0] = -1, 10 ** 6, -7
    p[2][2, :] = -1
    want = ref.attention(p[0].double().numpy(), *p[1:5], D, 1, T)
    assert np.isneginf(want[1][-180:]).all()
    out, lse = _run(p, -1, torch.float16)
    _check(out, lse, want, torch.float16, "missing pages")
    # a NaN scale of V at position 200 reaches the rows that see it and no others
    p = _problem([170], [260], 17, 17, D, -1, T, torch.float16, seed=52)
    p[1][p[2][0, 200 // T]].view(np.float16)[:, ref.places(T, D, 1)[3][200 % T]] = np.nan
    out, _ = _run(p, -1, torch.float16)
    nan = torch.isnan(out).flatten(1)
    first = 200 - (260 - 170)
    assert nan[first:].all() and not nan[:first].any()


def test_divided_prompt_same_bits_and_in_a_graph():
    """A divided block of rows gives the same bits from run to run and on replays between eager
    work; captured on a stream without scratch it stays whole, the same product."""
    D, T = 128, 16
    q, cache, table, kv, cu, _ = _problem([41], [1200], 68, 17, D, -1, T, torch.float16, seed=42)
    q, cache, table, kv, cu = q.to(DEV), torch.from_numpy(cache).to(DEV), ints(table), ints(kv), ints(cu)
    call = lambda: marlin.kv4_attention(q, cache, table, kv, cu, max_q=41, max_kv=1200, return_lse=True)  # noqa: E731
    want, want_lse = call()
    for _ in range(4):
        out, lse = call()
        assert torch.equal(out, want) and torch.equal(lse, want_lse)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        out, lse = call()
    for _ in range(4):
        out.fill_(float("nan"))
        call()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(lse, want_lse)
    fresh, graph2 = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph2, stream=fresh):
        out2, _ = call()
    graph2.replay()
    torch.cuda.synchronize()
    assert (out2.float() - want.float()).abs().max() <= 2.0 ** -9 * want.float().abs().max()


@pytest.mark.parametrize("long", [0, 3, 170])
def test_more_requests_than_one_launch_takes(long):
    """1100 requests of 0 to 40 tokens; the last but fifty with ``long`` new tokens (0: no cu_q)."""
    D, T, R = 64, 16, 1100
    q_lens = [1] * R
    kv_lens = [(7 * i) % 41 for i in range(R)]
    if long:
        q_lens[R - 50], kv_lens[R - 50], kv_lens[R - 51] = long, long + 5, 20
    p = _problem(q_lens, kv_lens, 2, 1, D, -1, T, torch.float16, seed=81)
    want = ref.attention(p[0].double().numpy(), *p[1:5], D, 1, T)
    out, lse = _run(p, -1, torch.float16, one=not long)
    _check(out, lse, want, torch.float16, f"{R} requests, {long}")


# ---- the example: projections, tables, append, attention and read-back in one path ----


@pytest.mark.parametrize("args", [[], ["--head-dim", "64", "--groupsize", "32", "--page", "64", "--prompt", "70"],
                                  ["--requests", "3", "--heads", "8", "--kv-heads", "8", "--prompt", "33", "--steps", "40"]])
def test_example(args, capsys):
    """Off by fp16's rounding of p v and of the output (2^-11 each, of sums no larger than
    twice the largest output) at most."""
    import importlib.util
    import pathlib
    path = pathlib.Path(__file__).resolve().parents[1] / "examples" / "kv4_decode.py"
    spec = importlib.util.spec_from_file_location("kv4_decode", path)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    assert module.main(["--check", *args]) <= 4 * 2.0 ** -11
    assert "tokens/s" in capsys.readouterr().out


@pytest.mark.parametrize("q_lens,kv_lens,H,most", [([5, 2, 9], [40, 70, 9], 2, 3), ([700, 3, 400], [700, 90, 600], 6, 300),
                                                   ([700, 300, 400], [700, 300, 600], 6, 300), ([40, 700], [40, 700], 9, 4)])
def test_more_new_tokens_than_max_q(q_lens, kv_lens, H, most):
    """The first max_q tokens of every request are computed, and no other row is touched."""
    D, T = 64, 16
    p = _problem(q_lens, kv_lens, H, H, D, -1, T, torch.float16, seed=91)
    want = ref.attention(p[0].double().numpy(), *p[1:5], D, 1, T)
    buf = torch.full(p[0].shape, 7.0, dtype=torch.float16, device=DEV)
    out, lse = _run(p, -1, torch.float16, max_q=most, out=buf)
    keep = np.concatenate([np.arange(n) < most for n in q_lens])
    _check(out[torch.from_numpy(keep).to(DEV)], lse[torch.from_numpy(keep).to(DEV)], [w[keep] for w in want], torch.float16, "first")
    assert (out[torch.from_numpy(~keep).to(DEV)] == 7).all()


@pytest.mark.parametrize("gain", [1e-39, 1e-36, 1e-20, 1e20, 1e30])
@pytest.mark.parametrize("q_lens,kv_lens,H", [([1, 1], [300, 40], 2), ([170, 90], [260, 90], 9)])
def test_tiny_and_huge_bf16_queries(q_lens, kv_lens, H, gain):
    """Queries near the type's limits: scores that are all zero, or one token that takes all."""
    D, g, T = 128, 64, 16
    p = list(_problem(q_lens, kv_lens, H, H, D, g, T, torch.bfloat16, seed=101))
    p[0] = (p[0].double() * gain).to(torch.bfloat16)
    want = ref.attention(p[0].double().numpy(), *p[1:5], D, p[5], T)
    out, _ = _run(p, g, torch.bfloat16)
    _check(out, None, want, torch.bfloat16, f"q times {gain}")


@pytest.mark.parametrize("q_lens,kv_lens,H", [([1, 1], [700, 40], 2), ([5], [300], 4), ([170, 90], [260, 90], 9)])
def test_scores_at_fp16_limits(q_lens, kv_lens, H):
    """Queries and keys of tens of thousands, values of hundreds: scores of 10^11, one token takes all."""
    D, T = 128, 16
    p = _problem(q_lens, kv_lens, H, H, D, -1, T, torch.float16, seed=102, k_gain=1e4, v_gain=300.0)
    p = (p[0] * 1e4, *p[1:])
    want = ref.attention(p[0].double().numpy(), *p[1:5], D, 1, T)
    out, lse = _run(p, -1, torch.float16)
    _check(out, lse, want, torch.float16, "limits", x_max=1e12)


@pytest.mark.parametrize("D,g,T", [(128, -1, 16), (128, 32, 32), (64, 64, 16)])
def test_more_blocks_of_rows_than_compute_units(D, g, T):
    """Whole blocks for every unit and a few more, which are divided over their tokens: the
    rows of the first and the last request against 64 bits, all of them run to run."""
    H, R, n, kv = 64, 5, 90, 700  # 320 blocks of 90 rows
    p = _problem([n] * R, [kv] * R, H, H, D, g, T, torch.float16, seed=111)
    first, lse = _run(p, g, torch.float16)
    q, cache, table, kvs, cu, G = p
    for i, h in ((0, 0), (0, 63), (4, 0), (4, 31), (4, 63)):
        sl = slice(n * i, n * (i + 1))
        want = ref.attention(q[sl, h:h + 1].double().numpy(), cache[:, h:h + 1], table[i:i + 1], kvs[i:i + 1], [0, n], D, G, T)
        _check(first[sl, h:h + 1], lse[sl, h:h + 1], want, torch.float16, f"request {i} head {h}")
    for _ in range(3):
        again, lse2 = _run(p, g, torch.float16)
        assert torch.equal(first, again) and torch.equal(lse, lse2)
