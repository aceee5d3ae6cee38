"""The 4-bit KV cache's attention where lengths, tables and q do not fit each other, and where
values span many orders of magnitude, against tests/kv4_ref.py.  Bounds as in test_gpu_kv4.py."""
import ctypes

import numpy as np
import pytest
import torch

from csed499ii_amd import marlin
from tests import kv4_ref as ref
from tests.test_gpu_kv4 import DEV, _check, _problem, ints

pytestmark = pytest.mark.gpu

# query and kv heads: rows for the kernel of few rows, and for that of prompts
KERNELS = [(4, 2), (34, 17)]


def _wider(table, pages):
    """The table with ``pages`` entries a row, those added no page: for the reference, which
    knows no width."""
    return np.pad(table, ((0, 0), (0, pages - table.shape[1])), constant_values=-1)


@pytest.mark.parametrize("Hq,Hkv", KERNELS)
@pytest.mark.parametrize("D,g", [(128, -1), (64, 32)])
def test_new_tokens_past_the_table_keep_their_positions(Hq, Hkv, D, g):
    """A table of 64 tokens for requests of 80, 64, 200 and 20: the tokens that it covers see
    what lies up to them, those past it all that it covers."""
    T, new, kv = 16, [50, 3, 60, 20], [80, 64, 200, 20]
    q, cache, table, cut, cu, G = _problem(new, [min(n, 64) for n in kv], Hq, Hkv, D, g, T, torch.float16, seed=201)
    want = ref.attention(q.double().numpy(), cache, _wider(table, 13), kv, cu, D, G, T)
    out, lse = marlin.kv4_attention(q.to(DEV), torch.from_numpy(cache).to(DEV), ints(table), ints(kv), ints(cu),
                                    max_q=60, max_kv=200, groupsize=g, return_lse=True)
    _check(out, lse, want, torch.float16, "cut by the table")


@pytest.mark.parametrize("Hq,Hkv", KERNELS)
def test_fewer_rows_of_q_than_new_tokens(Hq, Hkv):
    """cu_q counts 90 new tokens, q has the first 65: each at its own position."""
    T, D, new, kv = 16, 128, [20, 70], [33, 90]
    q, cache, table, kvs, cu, G = _problem(new, kv, Hq, Hkv, D, -1, T, torch.float16, seed=202)
    want = [x[:65] for x in ref.attention(q.double().numpy(), cache, table, kv, cu, D, G, T)]
    out, lse = marlin.kv4_attention(q[:65].to(DEV), torch.from_numpy(cache).to(DEV), ints(table), ints(kv), ints(cu),
                                    max_q=70, max_kv=90, return_lse=True)
    _check(out, lse, want, torch.float16, "cut by q")


def _step(Hq, Hkv, ctx, new, P, rows, seed):
    """Tables, append and attention of a step over a cache that holds the contexts and, in every
    other slot, NaN scales: the outputs, and those in 64 bits at the true positions."""
    T, D, R = 16, 128, len(ctx)
    gen = torch.Generator().manual_seed(seed)
    have = [min(-(-c // T), P) for c in ctx]
    size = R * P + 8
    order = torch.randperm(size, generator=gen).tolist()
    table, at = np.full((R, P), size + 5, np.int32), 0  # (stale entries: no page)
    cache = np.full((size, Hkv, T * (D + 4)), 0xFF, np.uint8)
    filled = ref.random_cache(size, Hkv, T, D, 1, gen)
    scales = ref.places(T, D, 1)[2:]
    for i, n in enumerate(have):
        table[i, :n] = order[at:at + n]
        at += n
        for j in range(n):
            cache[table[i, j]] = filled[table[i, j]]
            for o in range(ctx[i] - j * T, T):
                for s in scales:
                    cache[table[i, j]].view(np.float16)[:, s[o]] = np.nan
    free = ints(order[at:])
    q, k, v = (torch.randn((sum(new), h, D), generator=gen).half() for h in (Hq, Hkv, Hkv))
    dev_table, dev_cache = ints(table), torch.from_numpy(cache).to(DEV)
    slots, cu, kv, _ = marlin.kv4_tables(ints(ctx), ints(new), free, dev_table, rows, T)
    marlin.kv4_append(k[:rows].to(DEV), v[:rows].to(DEV), dev_cache, slots)
    out, lse = marlin.kv4_attention(q[:rows].to(DEV), dev_cache, dev_table, kv, cu, max_q=max(new), max_kv=P * T,
                                    return_lse=True, context_lens=ints(ctx))
    total = [c + n for c, n in zip(ctx, new)]
    want = ref.attention(q.double().numpy(), dev_cache.cpu().numpy(), _wider(dev_table.cpu().numpy(), P + max(total) // T + 1),
                         total, cu.cpu().numpy(), D, 1, T)
    return out, lse, [w[:rows] for w in want], slots


@pytest.mark.parametrize("Hq,Hkv", KERNELS)
def test_step_that_fills_its_tables(Hq, Hkv):
    """Requests that pass their tables' 64 tokens in this step, had passed them before, and fit."""
    out, lse, want, slots = _step(Hq, Hkv, [30, 70, 5, 0], [50, 40, 3, 64], 4, 157, 203)
    assert (slots[:34] >= 0).all() and (slots[34:90] == -1).all() and (slots[90:] >= 0).all()
    _check(out, lse, want, torch.float16, "full tables")


@pytest.mark.parametrize("Hq,Hkv", KERNELS)
def test_step_with_fewer_slots_than_new_tokens(Hq, Hkv):
    """A slot map that ends inside the second request: its tokens see those before them only."""
    out, lse, want, slots = _step(Hq, Hkv, [0, 9], [40, 40], 8, 65, 204)
    assert (slots >= 0).all()
    _check(out, lse, want, torch.float16, "short map")


def test_context_lens_are_checked():
    D, T = 128, 16
    cache = marlin.kv4_cache(4, 2, D, T, device=DEV)
    q, table, kv = torch.zeros((2, 2, D), dtype=torch.float16, device=DEV), ints([[0], [1]]), ints([3, 3])
    for bad in (ints([1]), ints([1, 2]).long(), ints([1, 2]).cpu()):
        with pytest.raises(RuntimeError, match="context_lens"):
            marlin.kv4_attention(q, cache, table, kv, context_lens=bad)


# ---- values over many orders of magnitude ----


def _set_token(cache, table, T, D, G, pos, code, ks, vs):
    """Position ``pos`` of request 0: every code of K ``code``, scales of K and V."""
    page, o = table[0, pos // T], pos % T
    k, _, k_at, v_at = ref.places(T, D, G)
    for n in k[o]:
        b = cache[page][:, n // 2]
        cache[page][:, n // 2] = (b & 0xF0) | code if n % 2 == 0 else (b & 0x0F) | code << 4
    halves = cache[page].view(np.float16)
    halves[:, k_at[o]], halves[:, v_at[o]] = ks, vs


WIDE = ["outlier first", "outlier inside", "outlier last", "sink of tiny v", "zeros first", "weightless zeros last",
        "rising"]


@pytest.mark.parametrize("n,Hq,Hkv", [(3, 4, 2), (50, 34, 17)])
@pytest.mark.parametrize("D,g", [(128, -1), (128, 64), (128, 32), (64, 32)])
@pytest.mark.parametrize("case", WIDE)
def test_values_over_many_orders_of_magnitude(case, D, g, n, Hq, Hkv):
    """Scales of V from fp16's least to its largest in one row.  p v is rounded to fp16 around a
    power of two that follows the row's largest p v, not its largest v: 2^-11 of sum_j w_j |v_jd|
    holds whatever v a token of little weight has, but for what lies 2^-32 a token below the
    row's largest w_j s_j (a code is 8 at most).  bf16, so that no output is below the type's range."""
    T, kv = 32, 400
    q, cache, table, kvs, cu, G = _problem([n], [kv], Hq, Hkv, D, g, T, torch.bfloat16, seed=211)
    q = q.abs()  # a token whose codes are all alike has the same sign of score for every row
    pl = ref.places(T, D, G)
    at = {p: (table[0, p // T], p % T) for p in range(kv)}

    def scale(tokens, f):
        for p in tokens:
            cache[at[p][0]].view(np.float16)[:, pl[3][at[p][1]]] *= np.float16(f)

    unit = float(q.double().sum(-1).mean()) / np.sqrt(D)  # of a token of codes 1 and scale 1
    if case.startswith("outlier"):  # no weight (2^-60 or less), the largest scale; the others near the least
        scale(range(kv), 2.0 ** -17)
        _set_token(cache, table, T, D, G, {"first": 0, "inside": 170, "last": kv - n}[case.split()[1]], 0,
                   80 / (8 * unit), 60000.0)
    elif case == "sink of tiny v":
        _set_token(cache, table, T, D, G, 0, 15, 12 / (7 * unit), 2.0 ** -24)
    elif case == "zeros first":
        scale(range(150), 0.0)
        scale(range(150, 300), 2.0 ** -20)
        scale(range(300, kv), 3000.0)
    elif case == "weightless zeros last":  # a token that takes nearly all weight and has no v
        _set_token(cache, table, T, D, G, kv - n, 15, 40 / (7 * unit), 0.0)
    else:
        for p in range(kv):
            scale([p], 2.0 ** (-17 + p / 12.5))  # 2^-17 to 2^14.9
    want = ref.attention(q.double().numpy(), cache, table, kvs, cu, D, G, T)
    out, lse = marlin.kv4_attention(q.to(DEV), torch.from_numpy(cache).to(DEV), ints(table), ints(kvs), ints(cu),
                                    max_q=n, max_kv=kv, groupsize=g, return_lse=True)
    o, (w, ref_lse, weight) = out.double().cpu().numpy(), want
    top = weight.max(-1, keepdims=True)  # >= the largest w_j s_j: some code is not 8
    tol = (2.0 ** -11 + 2.0 ** -13) * weight + 2.0 ** -8 * np.abs(w) + kv * 8 * 2.0 ** -32 * top
    bad = ~(np.abs(o - w) <= tol)
    assert not bad.any(), f"{bad.sum()} of {bad.size} off, worst {np.nanmax(np.abs(o - w) / tol):.2f} of the bound"
    assert np.abs(lse.double().cpu().numpy() - ref_lse).max() <= 2.0 ** -16 * 100


@pytest.mark.parametrize("n,Hq,Hkv", [(3, 4, 2), (50, 34, 17)])
@pytest.mark.parametrize("D,g", [(128, -1), (128, 64), (128, 32), (64, 32)])
@pytest.mark.parametrize("pos", [100, 396])
def test_nan_of_a_seen_row_without_weight_shows(pos, D, g, n, Hq, Hkv):
    """A NaN scale of V whose token's weight is zero in fp32, among tokens that all rows see and
    among those that some do not: the rows that see it are NaN, no others."""
    T, kv = 32, 399
    q, cache, table, kvs, cu, G = _problem([n], [kv], Hq, Hkv, D, g, T, torch.float16, seed=221)
    q = q.abs()
    unit = float(q.double().sum(-1).mean()) / np.sqrt(D)
    _set_token(cache, table, T, D, G, pos, 0, 300 / (8 * unit), np.nan)
    out = marlin.kv4_attention(q.to(DEV), torch.from_numpy(cache).to(DEV), ints(table), ints(kvs), ints(cu), max_q=n,
                               max_kv=kv, groupsize=g)
    nan, first = torch.isnan(out).flatten(1), max(pos - (kv - n), 0)
    assert nan[first:].all() and not nan[:first].any()


@pytest.mark.parametrize("q_lens,kv_lens,Hq,Hkv", [([1, 3], [300, 40], 4, 2), ([60, 90], [100, 90], 34, 17),
                                                   ([1, 200], [50, 200], 6, 6), ([1] * 1100, [3] * 1100, 2, 1), ([0, 0], [9, 9], 4, 2)])
@pytest.mark.parametrize("D,before,after", [(128, 0, 37), (64, 5, 1)])
def test_rows_of_no_request_are_left_alone(q_lens, kv_lens, Hq, Hkv, D, before, after):
    """Rows of q before the first request and after the last one, as in a step padded to a fixed
    size, hold NaN and change nothing; ``out`` keeps what it had there.  In the kernel of few
    rows, of prompts, both, and over several launches."""
    T = 16
    q, cache, table, kv, cu, G = _problem(q_lens, kv_lens, Hq, Hkv, D, -1, T, torch.float16, seed=231)
    want = ref.attention(q.double().numpy(), cache, table, kv, cu, D, G, T)
    q = torch.from_numpy(np.pad(q.numpy(), ((before, after), (0, 0), (0, 0)), constant_values=np.nan)).to(DEV)
    out = torch.full(q.shape, 7.0, dtype=torch.float16, device=DEV)
    _, lse = marlin.kv4_attention(q, torch.from_numpy(cache).to(DEV), ints(table), ints(kv), ints(cu + before),
                                  max_q=max(max(q_lens), 1), max_kv=max(kv_lens), return_lse=True, out=out)
    mine = slice(before, before + sum(q_lens))
    _check(out[mine], lse[mine], want, torch.float16, "between the padding")
    assert (out[:before] == 7).all() and (out[before + sum(q_lens):] == 7).all()


def test_an_output_over_q_is_refused():
    """Rows are written while others of q are still read."""
    D, T = 128, 16
    cache = marlin.kv4_cache(4, 2, D, T, device=DEV)
    buf = torch.zeros((3, 8, D), dtype=torch.float16, device=DEV)
    table, kv = ints([[0], [1], [2]]), ints([3, 3, 3])
    flat = buf.view(-1)
    for q, out in ((buf, buf), (buf[:, :4], buf.view(6, 4, D)[:3]), (buf[:, 2:6], flat[-3 * 4 * D:].view(3, 4, D)),
                   (buf.view(6, 4, D)[:3], buf.view(6, 4, D)[2:5])):
        with pytest.raises(RuntimeError, match="overlap"):
            marlin.kv4_attention(q, cache, table, kv, out=out)
    halves = buf.view(6, 4, D)
    marlin.kv4_attention(halves[:3], cache, table, kv, out=halves[3:])  # side by side


def _new_stream():
    """A stream of its own, kept for good: torch hands out a pool's in turn, and other tests count
    on getting one that no call has used."""
    hip, handle = ctypes.CDLL("libamdhip64.so"), ctypes.c_void_p()
    with torch.cuda.device(DEV):
        assert hip.hipStreamCreateWithFlags(ctypes.byref(handle), 1) == 0  # (does not wait for the null stream)
    return torch.cuda.ExternalStream(handle.value, device=DEV)


@pytest.mark.parametrize("streams", [1, 2])
def test_divided_calls_of_two_host_threads(streams):
    """Calls that divide their caches (few rows, prompts, both kernels in one call), issued by two
    host threads at once, on one stream and on one each: the bits of a call by itself."""
    import threading

    D, T = 128, 16
    calls = []
    for seed, (q_lens, kv_lens, Hq, Hkv) in enumerate([([1] * 3, [4000, 700, 2900], 8, 1), ([41], [1200], 68, 17),
                                                       ([120, 1, 2], [900, 3000, 40], 20, 20)]):
        q, cache, table, kv, cu, _ = _problem(q_lens, kv_lens, Hq, Hkv, D, -1, T, torch.float16, seed=241 + seed)
        args = (q.to(DEV), torch.from_numpy(cache).to(DEV), ints(table), ints(kv), ints(cu), max(q_lens), max(kv_lens))
        calls.append((args, marlin.kv4_attention(*args)))
    assert marlin.plan_kv4_attention(3, 8, 1, D, 1, 4000)["split"] and marlin.plan_kv4_attention(1, 68, 17, D, 41, 1200)["split"]
    torch.cuda.synchronize()
    own = [_new_stream() for _ in range(streams)]
    got, errors = [[], []], []

    def work(i):
        try:
            with torch.cuda.stream(own[i % streams]):
                for k in range(24):
                    args, want = calls[(k + i) % 3]
                    got[i].append((marlin.kv4_attention(*args), want))
        except Exception as e:  # noqa: BLE001 (shown by the test's own thread)
            errors.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not errors
    for out, want in got[0] + got[1]:
        assert torch.equal(out, want)
