"""The operators around the 4-bit KV cache as a decoder uses them together: tables, positions, rotary writes,
forks, shared prefixes and windows."""
import sys
import pathlib

import pytest
import torch

from csed499ii_amd import marlin

sys.path.insert(0, str(pathlib.Path(__file__).resolve().parents[1] / "examples"))
import kv4_decode  # noqa: E402

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("args", [["--samples", "3"], ["--samples", "5", "--requests", "2", "--prompt", "333", "--page", "64"],
                                  ["--window", "50"], ["--samples", "2", "--window", "70", "--head-dim", "64", "--groupsize", "32"],
                                  ["--samples", "40", "--requests", "1", "--kv-heads", "2", "--prompt", "200", "--steps", "3"]])
def test_example(args):
    """Each layer's attention against a plain one on the rows read back: p v in fp16, 2^-11 of sum w |v|, which
    is at most four times the largest output here, and the output's own 2^-11."""
    assert kv4_decode.main(args + ["--check", "--steps", "6"] if "--steps" not in args else args + ["--check"]) <= 5 * 2.0 ** -11


@pytest.mark.parametrize("D,g,page,prompt", [(128, -1, 16, 77), (64, 32, 32, 64), (128, 32, 64, 200)])
def test_forked_samples_are_the_requests_they_would_be(D, g, page, prompt):
    """Samples of one prompt that share its pages, against requests that each hold the prompt by themselves: the same
    caches, bit for bit in the first layer, and the same attention but for the order of its sums (2^-11 of sum w |v|
    on each side; both rounded)."""
    S, Hq, H, steps = 5, 8, 2, 3 * page // 2
    gen = torch.Generator().manual_seed(prompt)
    rows = lambda n: torch.randn((n, Hq + 2 * H, D), generator=gen).half().to(DEV)  # noqa: E731
    first, freqs = rows(prompt), marlin.rotary_frequencies(D, device=DEV)
    width = -(-(prompt + steps) // page)
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731

    def write(y, cache, table, lens, new, pages):
        free, _ = marlin.kv4_free_pages(table, lens, pages, page)
        slots, cu, kv, used, positions = marlin.kv4_tables(lens, ints(new), free, table, y.size(0), page, return_positions=True)
        q, k, v = y.split_with_sizes((Hq, H, H), 1)
        return marlin.kv4_append_rotary(q, k, v, cache, slots, marlin.rotary_angles(positions, freqs), g), cu, kv

    pages = 2 * S * width
    caches = [marlin.kv4_cache(pages, H, D, page, g, DEV) for _ in range(2)]
    # by themselves
    alone = torch.full((S, width), -1, dtype=torch.int32, device=DEV)
    _, _, alone_lens = write(first.repeat(S, 1, 1), caches[0], alone, ints([0] * S), [prompt] * S, pages)
    # one, forked
    one = torch.full((1, width), -1, dtype=torch.int32, device=DEV)
    _, _, lens = write(first, caches[1], one, ints([0]), [prompt], pages)
    layers = marlin.kv4_layers(caches[1], D, g)
    free, count = marlin.kv4_free_pages(one, lens, pages, page)
    assert count.item() == pages - -(-prompt // page)
    table, lens, used = marlin.kv4_fork(layers, one, lens, ints([0] * S), free)
    assert used.item() == (S - 1 if prompt % page else 0)
    groups = ints([0, S])
    for i in range(steps):
        y = rows(S)
        q0, _, n0 = write(y, caches[0], alone, alone_lens, [1] * S, pages)
        q1, _, n1 = write(y, caches[1], table, lens, [1] * S, pages)
        assert torch.equal(q0, q1) and torch.equal(n0, n1)
        shared = marlin.kv4_shared(table, lens, groups, page, always=i % 2 == 0)
        assert shared.lens.item() == prompt // page * page
        a = marlin.kv4_attention(q0, caches[0], alone, n0, max_kv=prompt + steps, groupsize=g)
        b = marlin.kv4_attention(q1, caches[1], table, n1, max_kv=prompt + steps, groupsize=g, context_lens=lens, shared=shared)
        c = marlin.kv4_attention(q1, caches[1], table, n1, max_kv=prompt + steps, groupsize=g, window=prompt + steps)
        top = a.float().abs().max().item()
        assert (a.float() - b.float()).abs().max().item() <= 2.0 ** -8 * top
        assert (a.float() - c.float()).abs().max().item() <= 2.0 ** -8 * top
        alone_lens, lens = n0, n1
        if i == steps // 2:  # the pool moved together, in the middle of it all
            held = prompt // page + sum(-(-(prompt + i + 1) // page) - prompt // page for _ in range(S))
            table, n = marlin.kv4_compact(layers, table, lens)
            assert n.item() == held and int(table.max()) == held - 1
    # every token's rows, of every sample
    pos = torch.arange(prompt + steps, device=DEV)
    for s in range(S):
        read = [marlin.kv4_gather(cache, (t[s].long()[pos // page] * page + pos % page).int(), D, g)
                for cache, t in zip(caches, (alone, table))]
        assert all(torch.equal(x, y) for x, y in zip(*read))
