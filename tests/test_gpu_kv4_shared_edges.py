"""Attention behind shared prefixes where lengths do not fit each other, or there is nothing to share."""
import threading

import numpy as np
import pytest
import torch

from csed499ii_amd import marlin
from tests.gpu_util import new_stream
from tests.test_gpu_kv4 import DEV, _check, ints
from tests.test_gpu_kv4_reach import _forked, _shared, attention

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("q,R,Hq,Hkv", [(1, 6, 4, 2), (1, 40, 8, 1), (5, 6, 4, 2), (90, 6, 6, 2)])
@pytest.mark.parametrize("D,g", [(128, -1), (64, 32)])
def test_lengths_that_end_inside_the_prefix(q, R, Hq, Hkv, D, g):
    """Requests whose kv_lens end within what their contexts say that they share (one that has finished, whose
    context is out of date, has none at all): a row sees the tokens up to kv_lens, as without the prefix."""
    T, pages = 16, 20
    p, cu_groups = _forked([(pages, R)], [q + i for i in range(R)], [q] * R, Hq, Hkv, D, g, T, torch.float16, seed=q + D)
    ctx = p[3] - q
    p[3][[0, 2, 3, 4, 5]] = 0, 33, pages * T - 1, pages * T, pages * T + 1
    want = attention(p[0].double().numpy(), *p[1:5], D, p[5], T, ctx=ctx)
    assert np.isneginf(want[1][:q]).all() and np.isfinite(want[1][q:]).all()
    s, (out, lse) = _shared(p, cu_groups, g, T, one=q == 1, ctx=ctx, max_kv=pages * T + 200)
    assert s.lens.tolist() == [pages * T]
    _check(out, lse, want, torch.float16, f"{q} tokens")
    plain = marlin.kv4_attention(p[0].to(DEV), torch.from_numpy(p[1]).to(DEV), ints(p[2]), ints(p[3]), ints(p[4]), groupsize=g,
                                 max_q=q, max_kv=pages * T + 200, context_lens=ints(ctx), return_lse=True)
    _check(*plain, want, torch.float16, f"{q} tokens, without the prefix")


@pytest.mark.parametrize("R,groups", [(0, 2), (0, 0), (3, 0)])
@pytest.mark.parametrize("one", [True, False])
def test_plan_of_nothing_to_share(R, groups, one):
    """No requests, or no groups: prefixes of no tokens, whatever the memory held."""
    n = 3 * groups + 1 + R
    for fill in (7, -9):
        junk = [torch.full((n,), fill, dtype=torch.int32, device=DEV) for _ in range(8)]
        del junk
        s = marlin.kv4_shared(ints(np.arange(2 * R).reshape(R, 2)), ints([20] * R), ints([0] * (groups + 1)), 16,
                              None if one else ints(range(R + 1)))
        assert s.plan.shape == (n,) and (s.plan == 0).all() and s.lens.tolist() == [0] * groups


@pytest.mark.parametrize("cu_groups", [[0, 16], [0]])
@pytest.mark.parametrize("n", [1, 40])
def test_one_pass_takes_no_workspace(n, cu_groups):
    """A call that the sizes send through one pass allocates nothing (out is given)."""
    D, T, R, Hq, H = 128, 16, 16, 64, 8
    p, _ = _forked([(2, R)], [n + 3] * R, [n] * R, Hq, H, D, -1, T, torch.float16, seed=n)
    q, cache, table, kv, cu = p[0].to(DEV), torch.from_numpy(p[1]).to(DEV), ints(p[2]), ints(p[3]), ints(p[4])
    ctx, out = kv - n, torch.empty((R * n, Hq, D), dtype=torch.float16, device=DEV)
    kw = dict(max_q=n, max_kv=int(p[3].max()), context_lens=ctx)
    s = marlin.kv4_shared(table, ctx, ints(cu_groups), T, cu)
    plain = marlin.kv4_attention(q, cache, table, kv, cu, **kw)
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    marlin.kv4_attention(q, cache, table, kv, cu, shared=s, out=out, **kw)
    assert torch.cuda.max_memory_allocated() == before
    assert torch.equal(out, plain)


def test_layers_that_overlap_are_refused():
    """Caches of two layers that have memory in common: pages of one would be written over by those of the other."""
    pool = marlin.kv4_cache(9, 2, 128, device=DEV)
    for caches in ((pool[:4], pool[3:7]), (pool[4:8], pool[:4], pool[5:]), (pool, pool)):
        with pytest.raises(RuntimeError, match="overlap|twice"):
            marlin.kv4_layers(caches, 128)
    assert len(marlin.kv4_layers((pool[4:8], pool[:4]), 128)) == 2


def test_a_bound_on_the_prefix_decides_the_passes():
    """Short prefixes under a max_kv far above them: with the bound one pass, which needs no workspace and gives the
    bits of a call without the prefix; without it the sizes speak for two."""
    D, T, R, H = 128, 16, 32, 32
    p, cu_groups = _forked([(2, R)], [1 + i for i in range(R)], [1] * R, H, H, D, -1, T, torch.float16, seed=3)
    q, cache, table, kv = p[0].to(DEV), torch.from_numpy(p[1]).to(DEV), ints(p[2]), ints(p[3])
    kw = dict(max_kv=16384, context_lens=kv - 1)
    plain = marlin.kv4_attention(q, cache, table, kv, **kw)
    want = attention(p[0].double().numpy(), *p[1:5], D, 1, T)
    for bound, always, one in ((32, False, True), (0, False, True), (32, True, False), (None, False, False), (20000, False, False)):
        s, out = marlin.kv4_shared(table, kv - 1, ints(cu_groups), T, always=always, max_prefix=bound), torch.empty_like(q)
        torch.cuda.synchronize()
        torch.cuda.reset_peak_memory_stats()
        before = torch.cuda.memory_allocated()
        marlin.kv4_attention(q, cache, table, kv, shared=s, out=out, **kw)
        assert (torch.cuda.max_memory_allocated() == before) == one, (bound, always)
        assert torch.equal(out, plain) or not one
        _check(out, None, want, torch.float16, f"bound {bound}")
    with pytest.raises(RuntimeError, match="max_prefix"):
        marlin.kv4_shared(table, kv - 1, ints(cu_groups), T, max_prefix=-1)


@pytest.mark.parametrize("cut", [1, 16, 25, 32, 40])
def test_a_request_cut_into_shared_pages_goes_on_after_a_fork(cut):
    """Two samples of one prompt of 40 tokens; the first is cut back and goes on otherwise: forked in between, no
    token of the second is written over, and the first holds what it was cut to and its new tokens."""
    D, T, H, pages = 64, 16, 2, 12
    gen = torch.Generator().manual_seed(cut)
    rows = lambda n: torch.randn((n, 2, H, D), generator=gen).half().to(DEV).unbind(1)  # noqa: E731
    cache, table = marlin.kv4_cache(pages, H, D, T, device=DEV), torch.full((1, 4), -1, dtype=torch.int32, device=DEV)
    layers = marlin.kv4_layers(cache, D)

    def append(k, v, lens, new, table):
        free, _ = marlin.kv4_free_pages(table, lens, pages, T)
        slots, _, kv, _ = marlin.kv4_tables(lens, ints(new), free, table, k.size(0), T)
        marlin.kv4_append(k, v, cache, slots)
        return kv

    def read(table, i, n):
        pos = torch.arange(n, device=DEV)
        return marlin.kv4_gather(cache, (table[i].long()[pos // T] * T + pos % T).int(), D)

    lens = append(*rows(40), ints([0]), [40], table)
    free, _ = marlin.kv4_free_pages(table, lens, pages, T)
    table, lens, _ = marlin.kv4_fork(layers, table, lens, ints([0, 0]), free)
    first, second = (read(table, i, 40) for i in range(2))
    assert all(torch.equal(a, b) for a, b in zip(first, second))
    lens = ints([cut, 40])
    free, _ = marlin.kv4_free_pages(table, lens, pages, T)
    table, lens, _ = marlin.kv4_fork(layers, table, lens, ints([0, 1]), free)
    k, v = rows(14)
    want = marlin.kv4_cache(1, H, D, T, device=DEV)
    marlin.kv4_append(k, v, want, ints(range(14)))
    lens = append(k, v, lens, [14, 0], table)
    assert lens.tolist() == [cut + 14, 40]
    assert all(torch.equal(a, b) for a, b in zip(read(table, 1, 40), second))
    for got, old, new in zip(read(table, 0, cut + 14), first, marlin.kv4_gather(want, ints(range(14)), D)):
        assert torch.equal(got[:cut], old[:cut]) and torch.equal(got[cut:], new)


@pytest.mark.parametrize("streams", [1, 2])
def test_windows_and_prefixes_of_two_host_threads(streams):
    """Windows and shared prefixes whose tokens are divided, in either kernel, issued by two host threads at once, on
    one stream and on one each: the bits of a call by itself."""
    D, T, calls = 128, 16, []
    for seed, (q, R, Hq, H, pages) in enumerate(((1, 40, 64, 8, 60), (4, 8, 8, 2, 120), (60, 4, 20, 20, 40))):
        p, cu_groups = _forked([(pages, R)], [q + 9 + i for i in range(R)], [q] * R, Hq, H, D, -1, T, torch.float16, seed=seed)
        dev = [x.to(DEV) for x in (p[0], torch.from_numpy(p[1]))] + [ints(x) for x in p[2:5]]
        ctx, kw = dev[3] - q, dict(max_q=q, max_kv=int(p[3].max()), return_lse=True)

        def shared(dev=dev, ctx=ctx, groups=ints(cu_groups), kw=kw):
            s = marlin.kv4_shared(dev[2], ctx, groups, T, dev[4], always=True)
            return marlin.kv4_attention(*dev, context_lens=ctx, shared=s, **kw)

        def window(dev=dev, kw=kw):
            return marlin.kv4_attention(*dev, window=500, sinks=4, **kw)

        calls += [(f, f()) for f in (shared, window)]
    torch.cuda.synchronize()
    own, got, errors = [new_stream() for _ in range(streams)], [[], []], []

    def work(i):
        try:
            with torch.cuda.stream(own[i % streams]):
                for k in range(30):
                    f, want = calls[(5 * k + 2 * i) % 6]
                    got[i].append((f(), want))
        except Exception as e:  # noqa: BLE001 (shown by the test's own thread)
            errors.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not errors and len(got[0]) == len(got[1]) == 30
    for result, want in got[0] + got[1]:
        assert all(torch.equal(a, b) for a, b in zip(result, want))
