"""The 4-bit KV cache's operators in 64 bits on the CPU (numpy), for the tests: written from
the layout and the formulas, by the place of every code, request by request."""
import math

import numpy as np
import torch


def groups(D, groupsize):
    return 1 if groupsize == -1 else D // groupsize


def quantize(x, G):
    """``x [..., D]`` float64 -> codes and scales (float64 of fp16 values)."""
    xg = x.reshape(x.shape[:-1] + (G, -1))
    with np.errstate(invalid="ignore", divide="ignore", over="ignore"):
        s = np.minimum(np.abs(xg).max(-1) * (2 / 15), 65504.0)  # a NaN stays one
        s = s.astype(np.float16).astype(np.float64)
        d = s[..., None]
        r = np.where(d > 0, np.clip(xg, -8 * d, 8 * d) / np.where(d > 0, d, 1), 0.0)
        c = np.clip(np.rint(r) + 8, 0, 15)
    c = np.where(d > 0, c, 8)
    return c.reshape(x.shape).astype(np.int64), s


def places(T, D, G):
    """Of token o, dim d: nibble index of the K code and of the V code, fp16 index of the K
    scale and of the V scale, all within a block ``[T, D]``."""
    o, d = np.arange(T)[:, None], np.arange(D)[None]
    k = o * D + (d % 32 // 8) * (D // 4) + d // 32 * 8 + d % 8
    v = T * D + (o // 4) * 4 * D + d // 8 * 32 + o % 4 * 8 + d % 8
    ks = T * D // 2 + (o // 4) * 4 * G + d // (D // G) * 4 + o % 4
    return k, v, ks, ks + T * G


def write_block(block, T, D, G, o, k, v):
    """Quantizes one token's rows ``k, v [D]`` into a block (uint8 array, changed)."""
    halves = block.view(np.float16)
    for x, at, s_at in ((k, 0, 2), (v, 1, 3)):
        c, s = quantize(x, G)
        pl = places(T, D, G)
        for d in range(D):
            n = pl[at][o, d]
            sh = 4 * (n % 2)
            block[n // 2] = (int(block[n // 2]) & ~(15 << sh) & 255) | int(c[d]) << sh
        halves[pl[s_at][o]] = np.repeat(s, D // G)


def read_block(block, T, D, G):
    """K and V ``[T, D]`` in float64 that a block stands for."""
    halves = block.view(np.float16).astype(np.float64)
    k, v, ks, vs = places(T, D, G)
    code = lambda n: (block[n // 2].astype(np.int64) >> (4 * (n % 2))) & 15  # noqa: E731
    with np.errstate(invalid="ignore"):
        return (code(k) - 8) * halves[ks], (code(v) - 8) * halves[vs]


def tables(ctx, new, free, table, num_tokens, T):
    """The bookkeeping of a step, token by token."""
    table = table.copy()
    R, P = table.shape
    slots, cu, kv, used, taken = np.full(num_tokens, -1, np.int32), [0], [], 0, 0
    t = 0
    for i in range(R):
        c, n = max(int(ctx[i]), 0), max(int(new[i]), 0)
        total, before = min(c + n, P * T), min(c, P * T)
        have = -(-before // T)
        for pos in range(c, c + n):
            if pos < P * T and t < num_tokens:
                j = pos // T
                if j < have:
                    page = table[i, j]
                else:
                    rank = used + j - have
                    page = free[rank] if rank < len(free) else -1
                    table[i, j] = page
                slots[t] = page * T + pos % T if page >= 0 else -1
            t += 1
        used += -(-total // T) - have
        cu.append(cu[-1] + n)
        kv.append(total)
    return slots, np.array(cu, np.int32), np.array(kv, np.int32), np.array([used], np.int32), table


def attention(q, cache, table, kv_lens, cu, D, G, T, scale=None):
    """``(out, lse, weight)`` in float64: ``weight[t, h, d] = sum_j softmax_j |v_jd|``, the
    measure that the rounding of the second product's operand goes by."""
    scale = 1 / math.sqrt(D) if scale is None else scale
    N, Hq, _ = q.shape
    num_pages, H, _ = cache.shape
    out, weight = np.zeros((N, Hq, D)), np.zeros((N, Hq, D))
    lse = np.full((N, Hq), -np.inf)
    for i in range(len(kv_lens)):
        kv, n = int(kv_lens[i]), int(cu[i + 1] - cu[i])
        for h in range(H):
            k, v, there = np.zeros((kv, D)), np.zeros((kv, D)), np.zeros(kv, bool)
            for j in range(-(-kv // T)):
                page, m = table[i, j], min(T, kv - j * T)
                if 0 <= page < num_pages:
                    kb, vb = read_block(cache[page, h], T, D, G)
                    k[j * T:j * T + m], v[j * T:j * T + m], there[j * T:j * T + m] = kb[:m], vb[:m], True
            for t in range(n):
                seen = there & (np.arange(kv) <= kv - n + t)
                if not seen.any():
                    continue
                for hq in range(h * Hq // H, (h + 1) * Hq // H):
                    x = k[seen] @ q[cu[i] + t, hq] * scale
                    m = x.max()
                    w = np.exp(x - m)
                    out[cu[i] + t, hq] = w @ v[seen] / w.sum()
                    weight[cu[i] + t, hq] = w @ np.abs(v[seen]) / w.sum()
                    lse[cu[i] + t, hq] = m + math.log(w.sum())
    return out, lse, weight


def random_cache(num_pages, H, T, D, G, gen, k_gain=1.0, v_gain=1.0):
    """A cache of random rows (uint8 numpy), quantized here."""
    k = torch.randn((num_pages, H, T, D), generator=gen, dtype=torch.float64).numpy() * k_gain
    v = torch.randn((num_pages, H, T, D), generator=gen, dtype=torch.float64).numpy() * v_gain
    pk, pv, pks, pvs = places(T, D, G)
    blocks = np.zeros((num_pages, H, T * (D + 4 * G)), np.uint8)
    nib = np.zeros((num_pages, H, 2 * T * D), np.uint8)
    halves = np.zeros((num_pages, H, T * (D + 4 * G) // 2), np.float16)
    for x, at, s_at in ((k, pk, pks), (v, pv, pvs)):
        c, s = quantize(x, G)
        nib[:, :, at.reshape(-1)] = c.reshape(num_pages, H, -1)
        halves[:, :, s_at.reshape(-1)] = np.repeat(s, D // G, -1).reshape(num_pages, H, -1)
    blocks[...] = halves.view(np.uint8)
    blocks[:, :, :T * D] = nib[:, :, 0::2] | nib[:, :, 1::2] << 4
    return blocks
