#!/usr/bin/env python3
"""A small decoder on 4 bits: 2:4 linear layers around a 4-bit paged KV cache.

Prompts of different lengths go through in one step, then every request decodes a token a
step.  The tables of a step are made once and serve all layers; each layer projects to q, k
and v with one ``Layer_2_4``, writes k and v into its cache, attends, and projects back.
Synthetic weights and inputs.

    python examples/kv4_decode.py [--layers 2] [--requests 6] [--prompt 300] [--steps 16] [--check]

``--check`` compares the last step's attention, layer by layer, with a plain one in fp32 on
the rows read back from the cache.
"""
import argparse
import pathlib
import sys
import time

import torch
import torch.nn as nn

sys.path.insert(0, str(pathlib.Path(__file__).resolve().parents[1]))
from csed499ii_amd import marlin, synth  # noqa: E402


def rms(x):
    xf = x.float()
    return (xf * torch.rsqrt(xf.pow(2).mean(-1, keepdim=True) + 1e-6)).half()


def linear(k, n, seed, device):
    """A packed 2:4 layer with synthetic weights."""
    layer = marlin.Layer_2_4(k, n, groupsize=128).to(device)
    w = synth.make_weight(k, n, seed, device=device)
    layer.B.copy_(w["B"].view_as(layer.B))
    layer.meta.copy_(w["meta"].view_as(layer.meta))
    layer.s.copy_(w["s"].view_as(layer.s))
    return layer


class Attention(nn.Module):
    """The attention block of one layer, with its own cache over the pages that all layers number alike."""

    def __init__(self, heads, kv_heads, head_dim, pages, page, groupsize, seed, device):
        super().__init__()
        self.heads, self.kv_heads, self.head_dim, self.groupsize = heads, kv_heads, head_dim, groupsize
        hidden = heads * head_dim
        self.qkv = linear(hidden, (heads + 2 * kv_heads) * head_dim, seed, device)
        self.o = linear(hidden, hidden, seed + 1, device)
        self.cache = marlin.kv4_cache(pages, kv_heads, head_dim, page, groupsize, device=device)
        self.last = None  # q and out of the last step, for the check

    def forward(self, x, slots, table, kv_lens, cu, max_q, max_kv, context_lens):
        y = self.qkv(rms(x)).view(x.size(0), self.heads + 2 * self.kv_heads, self.head_dim)
        q, k, v = y.split_with_sizes((self.heads, self.kv_heads, self.kv_heads), 1)  # views: no copy
        marlin.kv4_append(k, v, self.cache, slots, self.groupsize)
        out = marlin.kv4_attention(q, self.cache, table, kv_lens, cu, max_q, max_kv, self.groupsize,
                                   context_lens=context_lens)
        self.last = q, out
        return x + self.o(out.view(x.size(0), -1))


class Decoder:
    """Layers, block tables and the list of free pages; lengths are kept on the host too, for
    the bounds that the launches are planned with."""

    def __init__(self, layers, requests, heads, kv_heads, head_dim, max_tokens, page=16, groupsize=-1, device="cuda"):
        self.page, self.device = page, device
        width = -(-max_tokens // page)
        pages = requests * width
        self.free = torch.randperm(pages, device=device).int()
        self.table = torch.full((requests, width), -1, dtype=torch.int32, device=device)
        self.lens = [0] * requests
        self.kv_lens = torch.zeros(requests, dtype=torch.int32, device=device)
        self.layers = [Attention(heads, kv_heads, head_dim, pages, page, groupsize, 10 * i, device) for i in range(layers)]

    def step(self, x, new):
        """Runs ``new[i]`` tokens of each request (rows of ``x``, request by request) through
        the layers; returns the hidden rows and the first row of each request."""
        new_lens = torch.tensor(new, dtype=torch.int32).to(self.device)
        slots, cu, kv_lens, _ = marlin.kv4_tables(self.kv_lens, new_lens, self.free, self.table, x.size(0), self.page)
        pages = lambda n: -(-n // self.page)  # noqa: E731
        taken = sum(pages(c + n) - pages(c) for c, n in zip(self.lens, new))
        self.free = self.free[taken:]
        self.lens = [c + n for c, n in zip(self.lens, new)]
        context_lens, self.kv_lens = self.kv_lens, kv_lens
        one = None if all(n == 1 for n in new) else cu
        for layer in self.layers:
            x = layer(x, slots, self.table, kv_lens, one, max(new), max(self.lens), context_lens)
        return x, cu

    def check(self, new):
        """Largest error of the last step's attention against fp32, relative to the largest output."""
        worst = 0.0
        for layer in self.layers:
            (q, out), row = layer.last, 0
            for i, n in enumerate(new):
                kv, table = self.lens[i], self.table[i].long()
                pos = torch.arange(kv, device=self.device)
                slots = (table[pos // self.page] * self.page + pos % self.page).int()
                k, v = (t.float().repeat_interleave(layer.heads // layer.kv_heads, 1)
                        for t in marlin.kv4_gather(layer.cache, slots, layer.head_dim, layer.groupsize))
                rows = slice(row, row + n)
                x = (q[rows].float().unsqueeze(1) * k).sum(-1) / layer.head_dim ** 0.5  # [new, kv, heads]
                seen = pos[None] <= kv - n + torch.arange(n, device=self.device)[:, None]
                p = x.masked_fill(~seen[..., None], float("-inf")).softmax(1)
                want = (p.unsqueeze(-1) * v).sum(1)
                worst = max(worst, ((out[rows].float() - want).abs().max() / want.abs().max()).item())
                row += n
        return worst


def main(argv=None):
    ap = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    for name, default in (("layers", 2), ("requests", 6), ("heads", 16), ("kv-heads", 4), ("head-dim", 128),
                          ("prompt", 300), ("steps", 16), ("page", 16), ("groupsize", -1)):
        ap.add_argument("--" + name, type=int, default=default)
    ap.add_argument("--check", action="store_true")
    a = ap.parse_args(argv)
    torch.manual_seed(0)
    model = Decoder(a.layers, a.requests, a.heads, a.kv_heads, a.head_dim, a.prompt + a.steps, a.page, a.groupsize)
    new = [a.prompt - (i * a.prompt) // (2 * a.requests) for i in range(a.requests)]
    x = torch.randn((sum(new), a.heads * a.head_dim), device="cuda").half()
    x, cu = model.step(x, new)
    x = x[cu[1:].long() - 1]  # the last token of each prompt
    worst = model.check(new) if a.check else 0.0
    torch.cuda.synchronize()
    start, new = time.perf_counter(), [1] * a.requests
    for _ in range(a.steps):
        x, _ = model.step(x, new)
    torch.cuda.synchronize()
    took = time.perf_counter() - start
    if a.check and a.steps:
        worst = max(worst, model.check(new))
    print(f"{a.requests} requests, {sum(model.lens)} tokens in the caches of {a.layers} layers; "
          f"{a.requests * a.steps / took:.0f} tokens/s over {a.steps} steps"
          + (f"; attention off by {worst:.1e} of the largest output" if a.check else ""))
    return worst


if __name__ == "__main__":
    main()
