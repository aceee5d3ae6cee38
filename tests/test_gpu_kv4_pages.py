"""Pages of the 4-bit KV cache on the GPU: free lists, copies, forks and compaction against plain
implementations (tests/kv4_pages_ref.py).  Everything is whole numbers and bytes, and exact."""
import numpy as np
import pytest
import torch

from csed499ii_amd import marlin
from tests import kv4_pages_ref as pages
from tests import kv4_ref as ref
from tests.gpu_util import new_stream

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def ints(x):
    return torch.tensor(np.asarray(x), dtype=torch.int32, device=DEV)


def same(got, want, what=""):
    assert np.array_equal(got.cpu().numpy(), want), what


def _random_table(rng, R, P, num_pages, T, lens):
    """Distinct pages as far as there are, then any; stale entries past the lengths; some that are no page."""
    n = R * P
    pool = np.concatenate([rng.permutation(num_pages), rng.integers(0, num_pages, n)])[:n]
    table = pool.reshape(R, P).astype(np.int32)
    bad = rng.random((R, P)) < 0.02
    table[bad] = rng.choice([-1, -5, num_pages, num_pages + 7, 2 ** 31 - 1], bad.sum())
    return table


@pytest.mark.parametrize("R,P,num_pages,T,top", [
    (1, 1, 1, 16, 20), (3, 4, 20, 16, 70), (0, 3, 5, 32, 1), (5, 0, 33, 16, 9), (16, 16, 200, 64, 1000), (70, 40, 3000, 16, 700),
    (1030, 30, 32768, 16, 500),                                # the last sizes of the small kernel ...
    (1030, 32, 32768, 16, 500), (20, 10, 32769, 16, 160),      # ... and the first of the large ones
    (3, 70000, 60000, 16, 1 << 20), (5000, 3, 100001, 256, 900), (40, 50, 1 << 21, 16, 900),
])
def test_free_pages(R, P, num_pages, T, top):
    rng = np.random.default_rng(R + P + num_pages)
    lens = rng.integers(-3, top, R)
    lens[: R // 4] = 0
    table = _random_table(rng, R, P, num_pages, T, lens)
    free, count = marlin.kv4_free_pages(ints(table), ints(lens), num_pages, T)
    want, n = pages.free_pages(table, lens, num_pages, T)
    same(count, n)
    same(free, want)


def test_free_pages_all_and_none():
    table = np.arange(40, dtype=np.int32).reshape(4, 10)
    for lens, n in (([160] * 4, 0), ([0] * 4, 40), ([160, 0, 0, 160], 20), ([10 ** 9] * 4, 0)):
        free, count = marlin.kv4_free_pages(ints(table), ints(lens), 40, 16)
        assert count.item() == n and (free[n:] == -1).all()
        same(free, pages.free_pages(table, lens, 40, 16)[0])


def _layers(rng, count, num_pages, H, T, D, g):
    G = ref.groups(D, g)
    arrays = [rng.integers(0, 256, (num_pages, H, T * (D + 4 * G)), dtype=np.uint8) for _ in range(count)]
    return arrays, marlin.kv4_layers([torch.from_numpy(a).to(DEV) for a in arrays], D, g)


GEOMETRIES = [(128, -1, 16), (128, 64, 32), (128, 32, 64), (64, -1, 16), (64, 32, 128), (128, -1, 256)]


@pytest.mark.parametrize("D,g,T", GEOMETRIES)
@pytest.mark.parametrize("layers,H", [(1, 1), (3, 5), (130, 1)])
def test_copy_pages(D, g, T, layers, H):
    rng = np.random.default_rng(D + T + layers)
    arrays, on = _layers(rng, layers, 24, H, T, D, g)
    order = rng.permutation(24)
    src, dst = order[:9].astype(np.int32), order[9:18].astype(np.int32)
    src[2], dst[4], src[5] = -1, 24, 2 ** 31 - 1
    src[7] = src[8]  # one source of two
    marlin.kv4_copy_pages(on, ints(src), ints(dst))
    for c in arrays:
        for a, b in zip(src, dst):
            if 0 <= a < 24 and 0 <= b < 24:
                c[b] = c[a]
    for c, got in zip(arrays, on.caches):
        same(got, c)
    marlin.kv4_copy_pages(on, ints([]), ints([]))


@pytest.mark.parametrize("D,g,T", GEOMETRIES)
@pytest.mark.parametrize("layers,H,R,P,num_pages", [(1, 2, 3, 4, 20), (2, 3, 12, 6, 90), (130, 1, 2, 2, 9)])
def test_compact(D, g, T, layers, H, R, P, num_pages):
    rng = np.random.default_rng(D + T + R)
    arrays, on = _layers(rng, layers, num_pages, H, T, D, g)
    lens = rng.integers(0, P * T + 9, R)
    lens[0] = 0
    table = _random_table(rng, R, P, num_pages, T, lens)
    if R > 5:
        table[5, :2], lens[5] = table[4, :2], 2 * T  # shared pages
    old = ints(table)
    new, counts = marlin.kv4_compact(on, old, ints(lens))
    want, n = pages.compact(table, lens, arrays, num_pages, T)
    same(new, want), same(counts, n[:1]), same(old, table)
    for c, got in zip(arrays, on.caches):
        same(got, c)


@pytest.mark.parametrize("num_pages,R,P", [(40000, 20, 30), (70001, 700, 60)])
def test_compact_large_pool(num_pages, R, P):
    rng = np.random.default_rng(R)
    arrays, on = _layers(rng, 1, num_pages, 1, 16, 64, -1)
    lens = rng.integers(0, 16 * P + 1, R)
    table = _random_table(rng, R, P, num_pages, 16, lens)
    new, counts = marlin.kv4_compact(on, ints(table), ints(lens))
    want, n = pages.compact(table, lens, arrays, num_pages, 16)
    same(new, want), same(counts, n[:1]), same(on.caches[0], arrays[0])


def test_compact_full_and_empty_pools():
    rng = np.random.default_rng(0)
    arrays, on = _layers(rng, 2, 12, 1, 16, 64, -1)
    table = rng.permutation(12).astype(np.int32).reshape(3, 4)
    new, counts = marlin.kv4_compact(on, ints(table), ints([64, 64, 64]))
    same(new, table), same(counts, [12])
    new, counts = marlin.kv4_compact(on, ints(table), ints([0, 0, -4]))
    assert (new == -1).all() and counts.tolist() == [0]
    for c, got in zip(arrays, on.caches):
        same(got, c)


def _old_requests(rng, R, P, T, num_pages, lens):
    table = np.full((R, P), -1, np.int32)
    order, at = rng.permutation(num_pages), 0
    for i, n in enumerate(lens):
        k = min(-(-max(int(n), 0) // T), P)
        table[i, :k] = order[at:at + k]
        at += k
    return table, order[at:].astype(np.int32)


FORKS = [
    ([20], [0] * 5), ([16], [0, 0, 0]), ([0], [0, 0]), ([5, 37, 16, 63], [0, 1, 2, 3]), ([5, 37, 16, 63], [3, 3, 0, 1, 1, 1, 2, 0]),
    ([5, 37], [-1, 1, 7, 1, 2 ** 31 - 1, 0]), ([33, 0, 1], []), ([61] * 3, [2, 1, 0] * 20), ([1000, 7, -3], [0, 1, 2, 1]),
]


@pytest.mark.parametrize("D,g,T", GEOMETRIES)
@pytest.mark.parametrize("lens,parents", FORKS)
def test_fork(D, g, T, lens, parents):
    rng = np.random.default_rng(sum(lens) + T)
    lens = [n * T // 16 if n > 0 else n for n in lens]
    P, num_pages, layers, H = 5, 100, 3, 2
    arrays, on = _layers(rng, layers, num_pages, H, T, D, g)
    table, free = _old_requests(rng, len(lens), P, T, num_pages, lens)
    got = marlin.kv4_fork(on, ints(table), ints(lens), ints(parents), ints(free))
    want = pages.fork(table, lens, parents, free, arrays, num_pages, T, D, ref.groups(D, g))
    for name, a, b in zip(("table", "lens", "used"), got, want):
        same(a, b.reshape(a.shape), name)
    for c, a in zip(arrays, on.caches):
        same(a, c)


def test_fork_of_shortened_requests():
    """A request that was cut back into pages which others hold as full ones, or as their last: nobody's tokens
    may be written over."""
    T, D, num_pages = 16, 64, 40
    rng = np.random.default_rng(2)
    for lens, parents in (([20, 40, 25, 40], [0, 1, 2, 3]), ([20, 40, 25, 40], [2, 0, 0]), ([20, 22, 25, 31], [3, 2, 1, 0, 2]),
                          ([32, 20, 20, 0], [1, 0, 2])):
        arrays, on = _layers(rng, 2, num_pages, 2, T, D, -1)
        table = np.tile(np.array([3, 9, 17], np.int32), (4, 1))
        table[:, 2] = [17, 18, 19, 20]
        free = np.arange(25, 40, dtype=np.int32)
        got = marlin.kv4_fork(on, ints(table), ints(lens), ints(parents), ints(free))
        want = pages.fork(table, lens, parents, free, arrays, num_pages, T, D, 1)
        for a, b in zip(got, want):
            same(a, b.reshape(a.shape))
        for c, a in zip(arrays, on.caches):
            same(a, c)


@pytest.mark.parametrize("num_free", [0, 3, 7])
def test_fork_when_free_pages_run_out(num_free):
    T, D, num_pages = 16, 128, 30
    rng = np.random.default_rng(num_free)
    arrays, on = _layers(rng, 2, num_pages, 1, T, D, -1)
    table, free = _old_requests(rng, 1, 3, T, num_pages, [41])
    free = free[:num_free].copy()
    if num_free == 7:
        free[2], free[4] = -1, num_pages  # no pages
    got = marlin.kv4_fork(on, ints(table), ints([41]), ints([0] * 10), ints(free))
    want = pages.fork(table, [41], [0] * 10, free, arrays, num_pages, T, D, 1)
    for a, b in zip(got, want):
        same(a, b.reshape(a.shape))
    assert got[2].item() == 9
    for c, a in zip(arrays, on.caches):
        same(a, c)


def test_fork_of_many_requests():
    """Several rounds of requests, layers of several launches."""
    T, D, num_pages, R, N = 16, 64, 6000, 700, 2500
    rng = np.random.default_rng(9)
    lens = rng.integers(0, 50, R)
    parents = rng.integers(-1, R, N)
    arrays, on = _layers(rng, 130, 60, 1, T, D, -1)  # (layers past a launch: a small pool)
    table, free = _old_requests(rng, 4, 4, T, 60, [20, 33, 5, 64])
    small = [3, 0, 0, 1, 2, 2]
    got = marlin.kv4_fork(on, ints(table), ints([20, 33, 5, 64]), ints(small), ints(free))
    want = pages.fork(table, [20, 33, 5, 64], small, free, arrays, 60, T, D, 1)
    for a, b in zip(got, want):
        same(a, b.reshape(a.shape))
    for c, a in zip(arrays, on.caches):
        same(a, c)
    arrays, on = _layers(rng, 1, num_pages, 1, T, D, -1)
    table, free = _old_requests(rng, R, 4, T, num_pages, lens)
    got = marlin.kv4_fork(on, ints(table), ints(lens), ints(parents), ints(free))
    want = pages.fork(table, lens, parents, free, arrays, num_pages, T, D, 1)
    for a, b in zip(got, want):
        same(a, b.reshape(a.shape))
    same(on.caches[0], arrays[0])


def test_far_pages():
    """Pages whose byte offset passes 32 bits."""
    T, D, H, num_pages = 256, 128, 8, 17000
    cache = torch.zeros((num_pages, H, T * (D + 4)), dtype=torch.uint8, device=DEV)
    assert cache.numel() > 2 ** 32
    on = marlin.kv4_layers(cache, D)
    cache[16990] = torch.randint(0, 256, cache[0].shape, device=DEV, dtype=torch.uint8)
    want = cache[16990].clone()
    marlin.kv4_copy_pages(on, ints([16990]), ints([16500]))
    assert torch.equal(cache[16500], want) and not cache[16499].any() and not cache[16501].any()
    table, lens, used = marlin.kv4_fork(on, ints([[16990]]), ints([255]), ints([0, 0]), ints([16995]))
    assert table.tolist() == [[16990], [16995]] and torch.equal(cache[16995], want)
    new, counts = marlin.kv4_compact(on, table, lens)
    assert new.tolist() == [[0], [1]] and counts.tolist() == [2]
    assert torch.equal(cache[0], want) and torch.equal(cache[1], want)


def test_graph():
    """A captured step of free list, fork, free list, tables and compaction, replayed with other lengths."""
    T, D = 16, 64
    rng = np.random.default_rng(4)
    _, on = _layers(rng, 2, 60, 1, T, D, -1)
    table, _ = _old_requests(rng, 3, 8, T, 60, [100, 100, 100])
    table, lens, parents = ints(table), ints([100, 100, 100]), ints([0, 1, 1, 2])
    new_lens = ints([1] * 4)

    def step():
        free, _ = marlin.kv4_free_pages(table, lens, 60, T)
        t, n, used = marlin.kv4_fork(on, table, lens, parents, free)
        free, count = marlin.kv4_free_pages(t, n, 60, T)
        slots, cu, kv, _ = marlin.kv4_tables(n, new_lens, free, t, 4, T)
        c, counts = marlin.kv4_compact(on, t, kv)
        return t, n, used, count, slots, kv, c, counts

    side = new_stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        step()
        with torch.cuda.graph(graph, stream=side):
            out = step()
    torch.cuda.synchronize()
    first = [c.clone() for c in on.caches]
    for lengths, kin in (([37, 5, 16], [0, 1, 1, 2]), ([1, 90, 0], [1, 1, 1, 0]), ([100, 100, 100], [2, 2, -1, 0])):
        lens.copy_(ints(lengths)), parents.copy_(ints(kin))
        for c, f in zip(on.caches, first):
            c.copy_(f)
        graph.replay()
        torch.cuda.synchronize()
        got, bytes_ = [x.clone() for x in out], [c.clone() for c in on.caches]
        for c, f in zip(on.caches, first):
            c.copy_(f)
        assert all(torch.equal(a, b) for a, b in zip(step(), got))
        assert all(torch.equal(a, b) for a, b in zip(on.caches, bytes_))
