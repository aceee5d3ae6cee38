"""KV cache held in 4 bits, beside the 4-bit weights: tables, writes, read-back and the
attention that reads it.  No reference counterpart (the reference stops at the linear
layers).

A cache is a uint8 tensor ``[pages, kv_heads, T * D + 4 * T * D / groupsize]`` for pages of
``T`` tokens (16, 32, 64, 128 or 256) and heads of ``D`` dims (64 or 128), made by
:func:`kv4_cache`.  Rows are quantized as the packed weights are: a code ``c`` of 4 bits
stands for ``(c - 8) * s``, with one fp16 scale ``s = max|x| * 2 / 15`` per ``groupsize`` dims
(32, 64 or 128; -1: one per row).  A *slot* is a token's place, ``page * T + offset``.  The
page size follows from the tensor's width, ``head_dim`` and ``groupsize``.  The layout inside
a block is that of ``csrc/kv4_device.h``.

One decoding step of a layer, for requests in a batch::

    slots, cu, kv_lens, used = kv4_tables(context_lens, new_lens, free_pages, block_table, tokens, T)
    kv4_append(k, v, cache, slots)
    out = kv4_attention(q, cache, block_table, kv_lens, cu, max_q=..., max_kv=..., context_lens=context_lens)

The tables are made once a step and serve all layers.  Everything runs on the current
stream of the tensors' device and nothing waits for the GPU.
"""
from __future__ import annotations

import ctypes
import functools
import math
import typing

import torch

from .. import _lib

__all__ = ["kv4_cache", "kv4_tables", "kv4_append", "kv4_gather", "kv4_shared", "kv4_prefix", "kv4_attention",
           "plan_kv4_attention"]

_DTYPES = {torch.float16: 0, torch.bfloat16: 1}
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
    lambda index: torch.cuda.current_stream(index).cuda_stream)


def _raise(err: int):
    raise RuntimeError(_lib.last_error() or f"marlin_hip error {err}")


@functools.lru_cache(maxsize=None)
def _page_of(width: int, head_dim: int, groupsize: int) -> int:
    """Page size of a cache whose blocks are ``width`` bytes."""
    page, rest = divmod(width, _row_bytes(head_dim, groupsize))
    if rest or page not in (16, 32, 64, 128, 256):
        raise RuntimeError(f"cache blocks of {width} bytes hold no whole page of head_dim={head_dim}, "
                           f"groupsize={groupsize}")
    return page


def _row_bytes(head_dim: int, groupsize: int) -> int:
    """Bytes of one token's K and V of one head."""
    g = head_dim if groupsize == -1 else groupsize
    if head_dim not in (64, 128) or g not in (32, 64, 128) or head_dim % g:
        raise RuntimeError(f"the KV cache has kernels for head_dim 64 and 128 and groupsize 32, 64, 128 or -1 that "
                           f"divides it (head_dim={head_dim}, groupsize={groupsize})")
    return head_dim + 4 * (head_dim // g)


def _check_page(page_size: int):
    if page_size not in (16, 32, 64, 128, 256):
        raise RuntimeError(f"page_size must be 16, 32, 64, 128 or 256, got {page_size}")


def _device_of(name: str, t: torch.Tensor) -> int:
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    if not t.is_cuda:
        raise RuntimeError(f"{name} must be a GPU tensor (there is no CPU implementation)")
    return t.get_device()


def _ints(name: str, t: torch.Tensor, dev: int, dim: int = 1) -> int:
    """Address of a contiguous int32 tensor on device ``dev``."""
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    if t.dtype != torch.int32 or t.dim() != dim or t.get_device() != dev or not t.is_contiguous():
        raise RuntimeError(f"{name} must be a contiguous {dim}-dimensional int32 tensor on cuda:{dev}, got {t.dtype} "
                           f"{tuple(t.shape)} on {t.device}")
    return t.data_ptr()


def _page_size(cache: torch.Tensor, dev: int, kv_heads: int | None, head_dim: int, groupsize: int) -> int:
    _row_bytes(head_dim, groupsize)
    if not isinstance(cache, torch.Tensor):
        raise TypeError("cache must be a torch.Tensor")
    if cache.dtype != torch.uint8 or cache.dim() != 3 or cache.get_device() != dev or not cache.is_contiguous():
        raise RuntimeError(f"cache must be a contiguous 3-dimensional uint8 tensor on cuda:{dev}")
    if cache.data_ptr() % 16:
        raise RuntimeError("cache must be 16-byte aligned")
    if kv_heads is not None and cache.size(1) != kv_heads:
        raise RuntimeError(f"cache has {cache.size(1)} heads, k and v have {kv_heads}")
    return _page_of(cache.size(2), head_dim, groupsize)


def _rows(name: str, t: torch.Tensor, dev: int):
    """Strides of a ``[tokens, heads, D]`` tensor whose rows can be read 16 bytes at a time."""
    if t.dim() != 3 or t.get_device() != dev or t.dtype not in _DTYPES:
        raise RuntimeError(f"{name} must be a [tokens, heads, head_dim] fp16 or bf16 tensor on cuda:{dev}")
    st, sh, sd = t.stride()
    if t.size(1) == 1:
        sh = t.size(2)
    if t.size(0) == 1:
        st = 0
    if sd != 1 or st % 8 or sh % 8 or (t.numel() and t.data_ptr() % 16):
        raise RuntimeError(f"{name} needs contiguous rows, strides that are multiples of 8 elements and 16-byte alignment")
    return st, sh


def kv4_cache(num_pages: int, kv_heads: int, head_dim: int, page_size: int = 16, groupsize: int = -1,
              device="cuda") -> torch.Tensor:
    """An empty cache: uint8 ``[num_pages, kv_heads, bytes]``, zeroed."""
    _check_page(page_size)
    if num_pages < 1 or kv_heads < 1 or num_pages * page_size > 2**31 - 1:
        raise RuntimeError("the KV cache needs at least one page and one head and at most 2^31 - 1 tokens")
    return torch.zeros((num_pages, kv_heads, page_size * _row_bytes(head_dim, groupsize)), dtype=torch.uint8,
                       device=device)


def kv4_tables(context_lens: torch.Tensor, new_lens: torch.Tensor, free_pages: torch.Tensor,
               block_table: torch.Tensor, num_tokens: int, page_size: int, return_positions: bool = False):
    """Block tables and slot maps of a step, from the requests' lengths, in one launch.

    Request ``i`` holds ``context_lens[i]`` tokens and gets ``new_lens[i]`` more (int32
    ``[R]``).  The new tokens are numbered request by request; each one that is the first of
    its page takes the next entry of ``free_pages`` (int32 ``[F]``), which is written to
    ``block_table`` (int32 ``[R, P]``, updated in place; entries that the step does not fill
    stay).  Returns int32 tensors

    * ``slots [num_tokens]``: the slot of each new token, for :func:`kv4_append`; -1 past the
      last one, where ``free_pages`` has run out and where the table is full;
    * ``cu_new [R + 1]``: the first new token of each request, and their number;
    * ``kv_lens [R]``: ``context + new``, cut at the table's ``P * page_size`` (where that may
      happen :func:`kv4_attention` needs ``context_lens``, too, for the positions);
    * ``pages_used [1]``: pages wanted from ``free_pages``.  More than there are in it (``F``, or
      the ``count`` of :func:`kv4_free_pages`) means that some requests have entries of -1 in the
      table, whose tokens :func:`kv4_attention` leaves out;
    * with ``return_positions`` ``positions [num_tokens]``: the new tokens' positions in their
      requests, for :func:`rotary_angles`; 0 past the last one.

    ``num_tokens`` is the length of the slot map, an upper bound known on the host (a
    captured step may pass its padded size); tokens past it get no slot and no page, but count
    in ``cu_new``, ``kv_lens`` and ``pages_used``.
    Lengths below zero count as zero.  The sum of ``new_lens`` must stay below 2^31.
    """
    try:  # (as in kv4_append)
        R, = shape = context_lens.shape
        F, = free_pages.shape
        rows, P = block_table.shape
        dev, ctx, new = context_lens.get_device(), context_lens.data_ptr(), new_lens.data_ptr()
        free, table, kind = free_pages.data_ptr(), block_table.data_ptr(), torch.int32
        fits = (dev >= 0 and rows == R and page_size in (16, 32, 64, 128, 256) and new_lens.shape == shape
                and context_lens.dtype is new_lens.dtype is free_pages.dtype is block_table.dtype is kind
                and new_lens.get_device() == free_pages.get_device() == block_table.get_device() == dev
                and context_lens.is_contiguous() and new_lens.is_contiguous() and free_pages.is_contiguous()
                and block_table.is_contiguous())
    except (AttributeError, TypeError, ValueError):
        fits = False
    if not fits:
        dev = _device_of("context_lens", context_lens)
        _check_page(page_size)
        ctx, new = _ints("context_lens", context_lens, dev), _ints("new_lens", new_lens, dev)
        free, table = _ints("free_pages", free_pages, dev), _ints("block_table", block_table, dev, 2)
        R, F, P = context_lens.size(0), free_pages.size(0), block_table.size(1)
        if new_lens.size(0) != R or block_table.size(0) != R:
            raise RuntimeError(f"context_lens has {R} requests, new_lens {new_lens.size(0)}, block_table "
                               f"{block_table.size(0)}")
    if num_tokens < 0:
        raise RuntimeError("num_tokens must not be negative")
    sizes = (num_tokens, R + 1, R, 1, num_tokens) if return_positions else (num_tokens, R + 1, R, 1)
    out = context_lens.new_empty(sum(sizes))
    at = out.data_ptr()
    err = _lib.load().marlin_hip_kv4_tables_pos(ctx, new, free, table, at, at + 4 * num_tokens,
                                                at + 4 * (num_tokens + R + 1), at + 4 * (num_tokens + 2 * R + 1),
                                                at + 4 * (num_tokens + 2 * R + 2) if return_positions else 0, R, F, P,
                                                page_size, num_tokens, dev, _raw_stream(dev))
    if err:
        _raise(err)
    return out.split_with_sizes(sizes)


def kv4_append(k: torch.Tensor, v: torch.Tensor, cache: torch.Tensor, slots: torch.Tensor,
               groupsize: int = -1) -> None:
    """Quantize rows ``k, v [tokens, kv_heads, D]`` (fp16 or bf16) into the cache's ``slots``
    (int32 ``[tokens]``).

    Rows may be views with any token and head strides that are multiples of 8 elements, e.g.
    slices of a fused qkv projection.  A slot that is negative or past the last page is
    skipped; two tokens must not share one.  Scales saturate at 65504; a NaN makes its
    group NaN."""
    # What fits as it is passes in one look (the calls of a decoding step wait for the host);
    # anything else is checked step by step, for the message or for strides that do not count.
    try:
        N, H, D = shape = k.shape
        (kt, kh, kd), (vt, vh, vd) = k.stride(), v.stride()
        pages, heads, width = cache.shape
        dev, dtype = k.get_device(), _DTYPES.get(k.dtype)
        kp, vp, cp, sp = k.data_ptr(), v.data_ptr(), cache.data_ptr(), slots.data_ptr()
        fits = (dtype is not None and dev >= 0 and v.dtype is k.dtype and v.shape == shape and v.get_device() == dev
                and kd == vd == 1 and not (kt | kh | vt | vh) & 7 and not (kp | vp | cp) & 15 and heads == H
                and cache.dtype is torch.uint8 and cache.get_device() == dev and cache.is_contiguous()
                and slots.dtype is torch.int32 and slots.get_device() == dev and slots.is_contiguous()
                and slots.shape == (N,))
    except (AttributeError, TypeError, ValueError):
        fits = False
    if not fits:
        dev = _device_of("k", k)
        _device_of("v", v)
        kt, kh = _rows("k", k, dev)
        vt, vh = _rows("v", v, dev)
        N, H, D = k.shape
        if v.shape != k.shape or v.dtype != k.dtype:
            raise RuntimeError(f"k is {k.dtype} {tuple(k.shape)}, v is {v.dtype} {tuple(v.shape)}")
        _page_size(cache, dev, H, D, groupsize)
        sp = _ints("slots", slots, dev)
        if slots.size(0) != N:
            raise RuntimeError(f"slots has {slots.size(0)} entries, k has {N} tokens")
        pages, _, width = cache.shape
        kp, vp, cp, dtype = k.data_ptr(), v.data_ptr(), cache.data_ptr(), _DTYPES[k.dtype]
    err = _lib.load().marlin_hip_kv4_append(kp, vp, cp, sp, N, H, D, kt, kh, vt, vh, _page_of(width, D, groupsize), pages,
                                            groupsize, dtype, dev, _raw_stream(dev))
    if err:
        _raise(err)


def kv4_gather(cache: torch.Tensor, slots: torch.Tensor, head_dim: int, groupsize: int = -1,
               dtype: torch.dtype = torch.float16):
    """The values ``(k, v)``, each ``[tokens, kv_heads, head_dim]``, that the cache holds in
    ``slots``: what :func:`kv4_attention` computes with.  Zeros for slots that are negative or
    past the last page."""
    try:  # (as in kv4_append)
        pages, H, width = cache.shape
        N, = slots.shape
        dev, kind, cp, sp = cache.get_device(), _DTYPES.get(dtype), cache.data_ptr(), slots.data_ptr()
        fits = (kind is not None and dev >= 0 and cache.dtype is torch.uint8 and cache.is_contiguous() and not cp & 15
                and slots.dtype is torch.int32 and slots.get_device() == dev and slots.is_contiguous())
    except (AttributeError, TypeError, ValueError):
        fits = False
    if not fits:
        dev = _device_of("cache", cache)
        if dtype not in _DTYPES:
            raise RuntimeError(f"dtype must be fp16 or bf16, got {dtype}")
        _page_size(cache, dev, None, head_dim, groupsize)
        sp = _ints("slots", slots, dev)
        (pages, H, width), N, kind, cp = cache.shape, slots.size(0), _DTYPES[dtype], cache.data_ptr()
    page = _page_of(width, head_dim, groupsize)
    k = torch.empty((N, H, head_dim), dtype=dtype, device=cache.device)
    v = torch.empty_like(k)
    err = _lib.load().marlin_hip_kv4_gather(cp, sp, k.data_ptr(), v.data_ptr(), N, H, head_dim, page, pages, groupsize,
                                            kind, dev, _raw_stream(dev))
    if err:
        _raise(err)
    return k, v


class kv4_prefix(typing.NamedTuple):
    """What :func:`kv4_shared` found, for :func:`kv4_attention`: int32 ``[3 groups + 1 + requests]`` on the
    GPU (tokens of each group's prefix, a request that holds it, first token of each group, tokens of the
    prefix of each request) and the sizes it was made for."""
    plan: torch.Tensor
    requests: int
    groups: int
    pages: int
    page_size: int
    one: bool  # made without cu_q: a token each
    always: bool = False  # two passes, whatever the sizes
    most: int | None = None  # a bound on the prefixes' tokens (None: the attention's max_kv)

    @property
    def lens(self) -> torch.Tensor:
        """Tokens of each group's prefix, int32 ``[groups]``; 0 where nothing is shared."""
        return self.plan[:self.groups]


def kv4_shared(block_table: torch.Tensor, context_lens: torch.Tensor, cu_groups: torch.Tensor, page_size: int,
               cu_q: torch.Tensor | None = None, always: bool = False, max_prefix: int | None = None) -> kv4_prefix:
    """The prefixes that groups of requests share (after :func:`kv4_fork`, say), found in the block table
    once a step for the :func:`kv4_attention` of all layers.

    Group ``g`` is the requests ``cu_groups[g]`` to ``cu_groups[g + 1] - 1`` (int32 ``[groups + 1]``, not
    falling).  Its prefix is the leading pages that lie within ``context_lens`` and are the same in all
    rows of the group; requests without new tokens (``cu_q``, as in the attention call) and those that share no
    page with the group's first one are left out, and attend to all of their tokens by themselves.  So
    whatever the groups are, the attention is right; they decide what is read once.

    The attention then takes two passes, where the sizes say that they pay: by the blocks of rows and, for the tokens
    that are shared, ``max_prefix`` (a bound known on the host; default: the call's ``max_kv``), whose reads fall away
    (32 samples of 4096 shared tokens on 32 heads 47 us where 98; but 8 samples of 8192 on 64 and 8 heads, whose blocks
    of 16 rows fall from eight to four a head, 37 to 41 where 30, so one pass).  The lengths themselves are on the GPU:
    with a bound far above them two passes are taken where one would do, and cost 8 to 23 us more.
    ``always`` makes it two whatever the sizes."""
    try:  # (as in kv4_append)
        R, P = block_table.shape
        dev, table, ctx, at = block_table.get_device(), block_table.data_ptr(), context_lens.data_ptr(), cu_groups.data_ptr()
        kind = torch.int32
        fits = (dev >= 0 and context_lens.shape == (R,) and cu_groups.dim() == 1 and cu_groups.size(0) > 0
                and block_table.dtype is context_lens.dtype is cu_groups.dtype is kind
                and context_lens.get_device() == cu_groups.get_device() == dev and block_table.is_contiguous()
                and context_lens.is_contiguous() and cu_groups.is_contiguous()
                and page_size in (16, 32, 64, 128, 256))
    except (AttributeError, TypeError, ValueError):
        fits = False
    if not fits:
        dev = _device_of("block_table", block_table)
        table, ctx = _ints("block_table", block_table, dev, 2), _ints("context_lens", context_lens, dev)
        at, (R, P) = _ints("cu_groups", cu_groups, dev), block_table.shape
        _check_page(page_size)
        if context_lens.size(0) != R or cu_groups.size(0) < 1:
            raise RuntimeError(f"context_lens has {context_lens.size(0)} requests, block_table {R}; cu_groups needs an entry")
    cu = 0
    if cu_q is not None:
        cu = _ints("cu_q", cu_q, dev)
        if cu_q.size(0) != R + 1:
            raise RuntimeError(f"cu_q has {cu_q.size(0)} entries, expected {R + 1}")
    if max_prefix is not None and max_prefix < 0:
        raise RuntimeError(f"max_prefix must not be negative, got {max_prefix}")
    groups = cu_groups.size(0) - 1
    plan = (block_table.new_empty if R and groups else block_table.new_zeros)(3 * groups + 1 + R)  # (nothing: not launched)
    err = _lib.load().marlin_hip_kv4_shared(table, ctx, cu, at, plan.data_ptr(), R, groups, P, page_size, dev,
                                            _raw_stream(dev))
    if err:
        _raise(err)
    return kv4_prefix(plan, R, groups, P, page_size, cu_q is None, always, max_prefix)


@functools.lru_cache(maxsize=4096)
def _shared_bytes(tokens, requests, groups, q_heads, kv_heads, head_dim, groupsize, max_q, max_kv, cu_q, always, dev) -> int:
    """Workspace of an attention call with a prefix (0: the sizes send it through one pass).  A step asks for all layers."""
    out = (ctypes.c_longlong * 3)()
    err = _lib.load().marlin_hip_kv4_shared_plan(tokens, requests, groups, q_heads, kv_heads, head_dim, groupsize, max_q,
                                                 max_kv, cu_q, always, dev, out)
    if err:
        _raise(err)
    return out[0]


def kv4_attention(q: torch.Tensor, cache: torch.Tensor, block_table: torch.Tensor, kv_lens: torch.Tensor,
                  cu_q: torch.Tensor | None = None, max_q: int | None = None, max_kv: int | None = None,
                  groupsize: int = -1, scale: float | None = None, return_lse: bool = False,
                  out: torch.Tensor | None = None, context_lens: torch.Tensor | None = None,
                  shared: kv4_prefix | None = None, window: int | None = None, sinks: int = 0):
    """Causal attention of new tokens over the requests' cached rows, theirs included.

    ``q [tokens, q_heads, D]`` (fp16 or bf16; a view as in :func:`kv4_append`) holds the new
    tokens request by request: those of request ``i`` are ``q[cu_q[i]:cu_q[i + 1]]`` (int32
    ``[R + 1]``; None: one token a request).  Their positions start at ``context_lens[i]``
    (int32 ``[R]``; None: they are the last of the ``kv_lens[i]`` tokens).  The request has
    ``kv_lens[i]`` (int32 ``[R]``) tokens in all, whose rows lie in the pages ``block_table[i]``
    (int32 ``[R, P]``); the token at position ``p`` sees the positions up to ``p``.  After
    :func:`kv4_tables` pass its ``context_lens`` here, too: the ``kv_lens`` that it returns are
    cut where the table is full, and no longer tell the new tokens' positions.  ``q_heads`` is a multiple of the
    cache's heads, and query head ``h`` reads kv head ``h // (q_heads / kv_heads)``.

    ``max_q`` is the most new tokens of a request (a longer one's later tokens are not
    computed; default: 1 without ``cu_q``, else all tokens) and ``max_kv`` a bound on
    ``kv_lens`` that the split of long caches, and with ``shared`` one pass or two, is planned for
    (any value is correct; default: the table's ``P`` pages).  ``scale`` (positive; default ``1 / sqrt(D)``) multiplies the
    scores.  Returns ``out [tokens, q_heads, D]`` in ``q``'s type, and with ``return_lse`` the
    rows' log-sum-exp, fp32 ``[tokens, q_heads]``.

    With ``window`` the token at position ``p`` sees the positions ``j <= p`` of which ``j > p - window``, its
    own and the ``window - 1`` before, and the first ``sinks`` of its request; only their pages are
    read.  With ``shared`` (:func:`kv4_shared` of the same step; ``context_lens`` needed, too) the tokens that
    requests of a group share are attended to once for all of them, in a pass of its own before the
    one over each request's other tokens, where that pays: the same sums in another order (a request whose ``kv_lens``
    end inside the prefix attends by itself).  Not both.  ``shared`` is made from the
    ``block_table``, ``context_lens`` and ``cu_q`` of this call: with others the result is wrong.

    A row that sees no token gets zeros and ``-inf``.  Rows that belong to no request (before
    ``cu_q[0]``, from ``cu_q[R]`` on: a captured step's padding) and those past a request's
    ``max_q`` are not written: they keep what ``out`` held, or hold anything.  ``out`` must not
    overlap ``q``.  No gradient flows through the call, as through the other kernels.  Positions whose table entry is no page
    of the cache (e.g. -1) are left out; slots past ``kv_lens`` may hold anything.
    A call that splits uses the stream's split-K scratch, as :func:`mul_2_4` does: under
    stream capture make an eager call of the shape first, else it runs unsplit."""
    try:  # (as in kv4_append)
        N, Hq, D = q.shape
        qt, qh, qd = q.stride()
        pages, H, width = cache.shape
        R, P = block_table.shape
        dev, dtype = q.get_device(), _DTYPES.get(q.dtype)
        qp, cp, table, lens = q.data_ptr(), cache.data_ptr(), block_table.data_ptr(), kv_lens.data_ptr()
        fits = (dtype is not None and dev >= 0 and qd == 1 and not (qt | qh) & 7 and not (qp | cp) & 15
                and cache.dtype is torch.uint8 and cache.get_device() == dev and cache.is_contiguous()
                and block_table.dtype is torch.int32 and block_table.get_device() == dev and block_table.is_contiguous()
                and kv_lens.dtype is torch.int32 and kv_lens.get_device() == dev and kv_lens.is_contiguous()
                and kv_lens.shape == (R,))
    except (AttributeError, TypeError, ValueError):
        fits = False
    if not fits:
        dev = _device_of("q", q)
        qt, qh = _rows("q", q, dev)
        N, Hq, D = q.shape
        _page_size(cache, dev, None, D, groupsize)
        table, lens = _ints("block_table", block_table, dev, 2), _ints("kv_lens", kv_lens, dev)
        R, P = block_table.shape
        if kv_lens.size(0) != R:
            raise RuntimeError(f"kv_lens has {kv_lens.size(0)} requests, block_table {R}")
        pages, H, width = cache.shape
        qp, cp, dtype = q.data_ptr(), cache.data_ptr(), _DTYPES[q.dtype]
    page = _page_of(width, D, groupsize)
    if H == 0 or Hq % H:
        raise RuntimeError(f"{Hq} query heads are no multiple of the cache's {H}")
    if cu_q is None:
        cu = 0
        if N != R:
            raise RuntimeError(f"q has {N} tokens for {R} requests: pass cu_q")
        if max_q is None:
            max_q = 1
    else:
        cu = _ints("cu_q", cu_q, dev)
        if cu_q.size(0) != R + 1:
            raise RuntimeError(f"cu_q has {cu_q.size(0)} entries, expected {R + 1}")
        if max_q is None:
            max_q = N
    if context_lens is None:
        ctx = 0
    else:
        ctx = _ints("context_lens", context_lens, dev)
        if context_lens.size(0) != R:
            raise RuntimeError(f"context_lens has {context_lens.size(0)} requests, block_table {R}")
    if max_kv is None:
        max_kv = P * page
    if out is None:
        out = torch.empty_like(q) if q.is_contiguous() else q.new_empty((N, Hq, D))  # (torch.empty costs the host more)
    elif out.shape != q.shape or out.dtype != q.dtype or out.get_device() != dev or not out.is_contiguous() \
            or out.data_ptr() % 16:
        raise RuntimeError(f"out must be a contiguous, 16-byte aligned {q.dtype} {tuple(q.shape)} tensor on cuda:{dev}")
    elif N and out.data_ptr() < qp + 2 * ((N - 1) * qt + (Hq - 1) * qh + D) and qp < out.data_ptr() + 2 * N * Hq * D:
        raise RuntimeError("out must not overlap q, whose rows are read while out's are written")
    lse = torch.empty((N, Hq), dtype=torch.float32, device=q.device) if return_lse else None
    op, lp = out.data_ptr(), 0 if lse is None else lse.data_ptr()
    if scale is None:
        scale = 1.0 / math.sqrt(D)
    size = 0  # of the workspace for two passes
    if shared is not None:
        if window is not None or sinks:
            raise RuntimeError("kv4_attention takes shared or window and sinks, not both")
        if not isinstance(shared, kv4_prefix):
            raise TypeError("shared must be what kv4_shared returns")
        if (shared.requests, shared.pages, shared.page_size) != (R, P, page) or shared.plan.get_device() != dev \
                or context_lens is None or shared.one != (cu_q is None):
            raise RuntimeError(f"shared is of {shared.requests} requests with {shared.pages} pages of {shared.page_size} "
                               f"tokens, {'without' if shared.one else 'with'} cu_q, and needs context_lens; the call has "
                               f"{R}, {P} and {page}")
        size = _shared_bytes(N, R, shared.groups, Hq, H, D, groupsize, min(max_q, N),
                             max_kv if shared.most is None else min(max_kv, shared.most), cu != 0, shared.always, dev)
    if size:
        work = torch.empty(size // 4, dtype=torch.float32, device=q.device)
        err = _lib.load().marlin_hip_kv4_attention_shared(
            qp, cp, table, lens, cu, ctx, shared.plan.data_ptr(), op, lp, work.data_ptr(), N, R, shared.groups, Hq, H, D, qt,
            qh, page, pages, P, groupsize, min(max_q, N), max_kv, scale, dtype, size, 1, dev, _raw_stream(dev))
    elif window is not None:
        if window < 1 or sinks < 0:
            raise RuntimeError(f"a window holds a token at least, and sinks are not negative (window={window}, sinks={sinks})")
        err = _lib.load().marlin_hip_kv4_attention_window(
            qp, cp, table, lens, cu, ctx, op, lp, N, R, Hq, H, D, qt, qh, page, pages, P, groupsize, min(max_q, N), max_kv,
            scale, min(window, 1 << 30), min(sinks, 1 << 30), dtype, dev, _raw_stream(dev))
    else:
        if sinks:
            raise RuntimeError("sinks without a window: every row sees them already")
        err = _lib.load().marlin_hip_kv4_attention_ctx(
            qp, cp, table, lens, cu, ctx, op, lp, N, R, Hq, H, D, qt, qh, page, pages, P, groupsize, min(max_q, N), max_kv,
            scale, dtype, dev, _raw_stream(dev))
    if err:
        _raise(err)
    return (out, lse) if return_lse else out


def plan_kv4_attention(requests: int, q_heads: int, kv_heads: int, head_dim: int, max_q: int = 1, max_kv: int = 1,
                       groupsize: int = -1, sms: int = -1) -> dict:
    """The launch plan of a :func:`kv4_attention` call for ``requests`` requests of ``max_q`` new
    tokens each, computed on the host without a GPU (``sms``: compute units, -1: 256):
    ``workgroups`` of the kernel that runs (of few rows or of prompts, which the rows, new tokens
    times the query heads of a kv head, decide), and ``split``: whether a request's cache may be
    divided among workgroups, through the stream's split-K scratch, in such a call or one with
    shorter requests among them.  How it is divided follows from the real lengths, on the GPU."""
    out = (ctypes.c_int * 3)()
    err = _lib.load().marlin_hip_kv4_plan(requests, q_heads, kv_heads, head_dim, groupsize, max_q, max_kv, sms, out)
    if err:
        _raise(err)
    return {"workgroups": out[1], "split": bool(out[2])}
