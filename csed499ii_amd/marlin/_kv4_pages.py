"""Pages of the 4-bit KV cache: which are free, copies in the caches of all layers, requests made
from others (samples of one prompt, beams), and the held pages moved together.  No reference
counterpart.

The block table with the lengths is the only state.  A page is *held* if an entry of a written token
(``block_table[i][j]`` with ``j * page_size < kv_lens[i]``) names it, however many requests do; a
request is finished by a length of zero and shortened by a smaller one.  (One that may share pages goes
through :func:`kv4_fork` before it gets tokens again: others may hold the page in which it was cut, and
its next tokens would be written over theirs.)  A decoding step with samples that share their prompt's
pages::

    layers = kv4_layers(caches, head_dim, groupsize)             # once
    free, count = kv4_free_pages(table, lens, num_pages, T)
    table, lens, used = kv4_fork(layers, table, lens, parents, free)
    free, count = kv4_free_pages(table, lens, num_pages, T)
    slots, cu, kv_lens, used = kv4_tables(lens, new_lens, free, table, tokens, T)

Tables are int32 and never read on the host; new ones are returned, the old ones stay.  Everything runs
on the current stream of the tensors' device and nothing waits for the GPU.
"""
from __future__ import annotations

import ctypes

import torch

from .. import _lib
from ._kv4 import _check_page, _device_of, _ints, _page_size, _raise, _raw_stream

__all__ = ["kv4_layers", "kv4_free_pages", "kv4_copy_pages", "kv4_fork", "kv4_compact"]


class kv4_layers:
    """The caches of a model's layers, whose pages are numbered alike: tensors of one shape made by
    :func:`kv4_cache`, on one device.  Checked once, for :func:`kv4_fork`, :func:`kv4_compact` and
    :func:`kv4_copy_pages`, which go through all of them in one launch (128 to a launch)."""

    def __init__(self, caches, head_dim: int, groupsize: int = -1):
        self.caches = (caches,) if isinstance(caches, torch.Tensor) else tuple(caches)
        if not self.caches:
            raise RuntimeError("kv4_layers needs a cache at least")
        self.device = _device_of("cache", self.caches[0])
        shape = self.caches[0].shape
        for c in self.caches:
            self.page_size = _page_size(c, self.device, None, head_dim, groupsize)
            if c.shape != shape:
                raise RuntimeError(f"the caches of layers have one shape, got {tuple(shape)} and {tuple(c.shape)}")
        at = [c.data_ptr() for c in self.caches]
        if len(set(at)) != len(at):
            raise RuntimeError("kv4_layers got one cache twice")
        order = sorted(at)
        if any(b - a < self.caches[0].numel() for a, b in zip(order, order[1:])):
            raise RuntimeError("the caches of layers must not overlap one another")
        self.num_pages, self.kv_heads = shape[0], shape[1]
        self.head_dim, self.groupsize, self.count = head_dim, groupsize, len(at)
        self._at = (ctypes.c_void_p * len(at))(*at)

    def __len__(self):
        return len(self.caches)


def _table(block_table, kv_lens):
    try:  # (what fits passes in one look; anything else is checked step by step, for the message)
        R, P = block_table.shape
        dev, kind = block_table.get_device(), torch.int32
        if dev >= 0 and kv_lens.shape == (R,) and block_table.dtype is kind and kv_lens.dtype is kind \
                and kv_lens.get_device() == dev and block_table.is_contiguous() and kv_lens.is_contiguous():
            return dev, block_table.data_ptr(), kv_lens.data_ptr(), R, P
    except (AttributeError, TypeError, ValueError):
        pass
    dev = _device_of("block_table", block_table)
    table, lens = _ints("block_table", block_table, dev, 2), _ints("kv_lens", kv_lens, dev)
    R, P = block_table.shape
    if kv_lens.size(0) != R:
        raise RuntimeError(f"kv_lens has {kv_lens.size(0)} requests, block_table {R}")
    return dev, table, lens, R, P


def _of_layers(layers, dev):
    if not isinstance(layers, kv4_layers):
        raise TypeError("layers must be a kv4_layers")
    if layers.device != dev:
        raise RuntimeError(f"the caches are on cuda:{layers.device}, the tables on cuda:{dev}")


def kv4_free_pages(block_table: torch.Tensor, kv_lens: torch.Tensor, num_pages: int, page_size: int):
    """The pages of a cache of ``num_pages`` that no request holds: ``(free [num_pages], count [1])``,
    int32, the free ones in ascending order and -1 behind them; ``free`` goes to :func:`kv4_tables` and
    :func:`kv4_fork` as it is (where their ``pages_used`` passes ``count``, the tables get -1 as if the list had
    ended there).  Entries that are no page are passed over."""
    dev, table, lens, R, P = _table(block_table, kv_lens)
    _check_page(page_size)
    if num_pages < 1 or num_pages * page_size > 2**31 - 1:
        raise RuntimeError("the KV cache holds a page at least and 2^31 - 1 tokens at most")
    # (the marks behind the results, from a multiple of 16 bytes on)
    marks = (num_pages + 1 + 3) // 4 * 4
    out = block_table.new_empty(marks + (num_pages + 15) // 16 * 4)
    at = out.data_ptr()
    err = _lib.load().marlin_hip_kv4_free_pages(table, lens, at, at + 4 * num_pages, at + 4 * marks, R, P, page_size,
                                                num_pages, dev, _raw_stream(dev))
    if err:
        _raise(err)
    return out.split_with_sizes((num_pages, 1, out.numel() - num_pages - 1))[:2]


def kv4_copy_pages(layers: kv4_layers, source: torch.Tensor, target: torch.Tensor) -> None:
    """Copies page ``source[i]`` to page ``target[i]`` (int32) in every layer.  Pairs with an entry that is
    no page are skipped.  No page may be a target twice, nor a source of one pair and the target of
    another."""
    if not isinstance(layers, kv4_layers):
        raise TypeError("layers must be a kv4_layers")
    src, dst = _ints("source", source, layers.device), _ints("target", target, layers.device)
    if source.size(0) != target.size(0):
        raise RuntimeError(f"source has {source.size(0)} pages, target {target.size(0)}")
    err = _lib.load().marlin_hip_kv4_copy_pages(layers._at, layers.count, src, dst, source.size(0), layers.kv_heads,
                                                layers.head_dim, layers.page_size, layers.num_pages, layers.groupsize,
                                                layers.device, _raw_stream(layers.device))
    if err:
        _raise(err)


def kv4_fork(layers: kv4_layers, block_table: torch.Tensor, kv_lens: torch.Tensor, parents: torch.Tensor,
             free_pages: torch.Tensor):
    """Requests made from others: new request ``i`` has the tokens of request ``parents[i]`` (int32
    ``[new requests]``; any order, any number of times; a number that is no request makes an empty one).

    Full pages are shared.  A last page that is not full is kept by the first new request that holds
    it, unless another holds it as a full page; every other gets a page of ``free_pages`` (int32
    ``[F]``, which nobody holds), in the order of the new requests, with a copy of the written tokens
    in the caches of all layers (its other slots are left as they were, but for the rest of the last
    group of four).  So each of them may be appended to.  Returns new int32 tensors

    * ``block_table [new requests, P]``: entries past a request's tokens and entries that were no page are -1;
    * ``kv_lens [new requests]``: the parents' lengths, cut at the table's width;
    * ``pages_used [1]``: pages wanted from ``free_pages``.  More than there are in it (``F``, or the ``count`` of
      :func:`kv4_free_pages`, whose list has -1 behind them) means that some requests have -1 for their last
      page, whose tokens :func:`kv4_attention` leaves out.

    Requests may share a page at the same place of their tables only, as forks do."""
    dev, table, lens, R, P = _table(block_table, kv_lens)
    _of_layers(layers, dev)
    par, free = _ints("parents", parents, dev), _ints("free_pages", free_pages, dev)
    (N,), (F,) = parents.shape, free_pages.shape
    new_table, out = block_table.new_empty((N, P)), block_table.new_empty(2 * N + 1)
    at = out.data_ptr()
    err = _lib.load().marlin_hip_kv4_fork(layers._at, layers.count, table, lens, par, free, new_table.data_ptr(), at,
                                          at + 4 * N, at + 4 * (N + 1), R, N, F, P, layers.kv_heads, layers.head_dim,
                                          layers.page_size, layers.num_pages, layers.groupsize, dev, _raw_stream(dev))
    if err:
        _raise(err)
    new_lens, used, _ = out.split_with_sizes((N, 1, N))
    return new_table, new_lens, used


def kv4_compact(layers: kv4_layers, block_table: torch.Tensor, kv_lens: torch.Tensor):
    """Moves the ``n`` held pages to the numbers ``0 ... n - 1`` in the caches of all layers: those past
    them, in ascending order, to the free ones among them.  Returns ``(block_table, held [1])``,
    int32: the table with the new numbers (-1 past a request's tokens and for entries that were no page)
    and ``n``.  The pages from ``n`` on keep what they held; a cache of the first
    ``n`` is ``cache[:n]``."""
    dev, table, lens, R, P = _table(block_table, kv_lens)
    _of_layers(layers, dev)
    pages = (layers.num_pages + 15) // 16 * 16
    new_table = block_table.new_empty((R, P))
    work = block_table.new_empty(3 * pages + pages // 4 + 2 + 4)
    counts, lists = work[:2], (work.data_ptr() + 8 + 15) // 16 * 16
    err = _lib.load().marlin_hip_kv4_compact(layers._at, layers.count, table, lens, new_table.data_ptr(),
                                             counts.data_ptr(), lists, R, P, layers.kv_heads, layers.head_dim,
                                             layers.page_size, layers.num_pages, layers.groupsize, dev, _raw_stream(dev))
    if err:
        _raise(err)
    return new_table, counts[:1]
