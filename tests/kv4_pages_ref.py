"""Pages of the 4-bit KV cache, request by request and entry by entry (numpy), for the tests."""
import numpy as np


def held_pages(table, lens, num_pages, T):
    held = set()
    for i, n in enumerate(lens):
        for j in range(min(-(-max(int(n), 0) // T), table.shape[1])):
            if 0 <= table[i, j] < num_pages:
                held.add(int(table[i, j]))
    return held


def free_pages(table, lens, num_pages, T):
    held = held_pages(table, lens, num_pages, T)
    free = [p for p in range(num_pages) if p not in held]
    return np.array(free + [-1] * len(held), np.int32), np.array([len(free)], np.int32)


def rows_of(n, T, D, G):
    """Bytes of a block that hold the first n tokens, rounded up to fours."""
    m = -(-n // 4) * 4
    K, V, S = T * D // 2, T * D, T * D + 2 * T * G
    return np.r_[0:m * D // 2, K:K + m * D // 2, V:V + 2 * m * G, S:S + 2 * m * G]


def compact(table, lens, caches, num_pages, T):
    held = sorted(held_pages(table, lens, num_pages, T))
    n = len(held)
    moved, holes = [p for p in held if p >= n], [p for p in range(n) if p not in set(held)]
    to = {**{p: p for p in held}, **dict(zip(moved, holes))}
    for c in caches:
        c[holes] = c[moved]
    out = np.full_like(table, -1)
    for i, m in enumerate(lens):
        for j in range(min(-(-max(int(m), 0) // T), table.shape[1])):
            out[i, j] = to.get(int(table[i, j]), -1)
    return out, np.array([n, len(moved)], np.int32)


def fork(table, lens, parents, free, caches, num_pages, T, D, G):
    R, P = table.shape
    N, new, new_lens, used = len(parents), np.full((len(parents), P), -1, np.int32), [], 0
    for i, p in enumerate(parents):
        n = min(max(int(lens[p]), 0), P * T) if 0 <= p < R else 0
        new_lens.append(n)
        for j in range(-(-n // T)):
            new[i, j] = table[p, j] if 0 <= table[p, j] < num_pages else -1
    given = new.copy()
    for i, n in enumerate(new_lens):
        j = n // T
        page = given[i, j] if n % T else -1
        if page < 0:
            continue
        full = any(given[k, j] == page and new_lens[k] >= (j + 1) * T for k in range(N))
        part = any(given[k, j] == page for k in range(i))
        if full or part:
            to = int(free[used]) if used < len(free) else -1
            used += 1
            new[i, j] = to if 0 <= to < num_pages else -1
            if new[i, j] >= 0:
                at = rows_of(n % T, T, D, G)
                for c in caches:
                    c[to][:, at] = c[page][:, at]
    return new, np.array(new_lens, np.int32), np.array([used], np.int32)
