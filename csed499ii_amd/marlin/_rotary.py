"""Rotary positions of rows, and on the way into the 4-bit KV cache.  No reference counterpart
(the reference stops at the linear layers).

Of a row's first ``r`` dims the pairs ``(x_i, x_{i + r/2})``, or interleaved ``(x_{2i}, x_{2i+1})``,
are turned by the angle ``p f_i`` of the token's position ``p``::

    a' = a cos(p f) - b sin(p f),   b' = b cos(p f) + a sin(p f)

The frequencies are made once a model, the angles once a step, for all layers::

    freqs = rotary_frequencies(128)
    slots, cu, kv_lens, used, positions = kv4_tables(..., return_positions=True)
    angles = rotary_angles(positions, freqs)
    q = kv4_append_rotary(q, k, v, cache, slots, angles)        # per layer: instead of kv4_append
    out = kv4_attention(q, cache, ...)

Everything runs on the current stream of the tensors' device and nothing waits for the GPU.
"""
from __future__ import annotations

import math

import torch

from .. import _lib
from ._kv4 import _DTYPES, _device_of, _ints, _page_of, _page_size, _raise, _raw_stream, _rows

__all__ = ["rotary_frequencies", "rotary_angles", "rotary", "kv4_append_rotary"]


def rotary_frequencies(rotary_dim: int, base: float = 10000.0, scale: float = 1.0, original: float | None = None,
                       slow: float = 1.0, fast: float = 32.0, device="cuda") -> torch.Tensor:
    """The angles that pairs turn by a position, ``f_i = base^(-2 i / rotary_dim)``: int64
    ``[rotary_dim / 2]`` in units of 2^-64 of a turn, modulo a turn, for :func:`rotary_angles`.

    For contexts longer than the one trained with, ``scale`` s divides them all
    (interpolated positions) or, with the trained length ``original`` L, by parts: a pair
    that makes ``fast`` or more turns over L positions keeps its frequency, one that makes
    ``slow`` or fewer is divided, and those between are mixed, ``f (m + (1 - m) / s)`` with
    ``m = (L f / 2 pi - slow) / (fast - slow)``."""
    if rotary_dim < 2 or rotary_dim % 2:
        raise RuntimeError(f"rotary_dim must be even and 2 at least, got {rotary_dim}")
    if not (0 < base < math.inf and 0 < scale < math.inf):
        raise RuntimeError("rotary_frequencies needs a positive, finite base and scale")
    if original is not None and not (0 < original < math.inf and -math.inf < slow < fast < math.inf):
        raise RuntimeError("rotary_frequencies by parts needs a positive original length and slow < fast")
    out = []
    try:
        for i in range(rotary_dim // 2):
            f = base ** (-2 * i / rotary_dim)
            m = 0.0 if original is None else min(max((original * f / (2 * math.pi) - slow) / (fast - slow), 0.0), 1.0)
            turns = int(f * (m + (1.0 - m) / scale) / (2 * math.pi) * 2.0 ** 64) % 2 ** 64
            out.append(turns - 2 ** 64 if turns >= 2 ** 63 else turns)
    except OverflowError:
        raise RuntimeError(f"base {base} and scale {scale} make frequencies that are not finite") from None
    return torch.tensor(out, dtype=torch.int64).to(device)


def rotary_angles(positions: torch.Tensor, freqs: torch.Tensor, factor: float = 1.0) -> torch.Tensor:
    """Cosine and sine, times ``factor``, of the angles of ``positions`` (int32 ``[tokens]``, of any
    size and sign): float64 ``[tokens, pairs, 2]``.  Positions of the other sign turn rows back."""
    try:  # (as in kv4_append)
        (tokens,), (pairs,) = positions.shape, freqs.shape
        dev, at = positions.get_device(), positions.data_ptr()
        fits = (dev >= 0 and positions.dtype is torch.int32 and positions.is_contiguous() and freqs.dtype is torch.int64
                and freqs.get_device() == dev and freqs.is_contiguous())
    except (AttributeError, TypeError, ValueError):
        fits = False
    if not fits:
        dev = _device_of("positions", positions)
        at = _ints("positions", positions, dev)
        if not isinstance(freqs, torch.Tensor):
            raise TypeError("freqs must be a torch.Tensor")
        if freqs.dtype != torch.int64 or freqs.dim() != 1 or freqs.get_device() != dev or not freqs.is_contiguous():
            raise RuntimeError(f"freqs must be a contiguous 1-dimensional int64 tensor on cuda:{dev}, as "
                               f"rotary_frequencies makes it")
        tokens, pairs = positions.size(0), freqs.size(0)
    out = freqs.new_empty((tokens, pairs, 2), dtype=torch.float64)
    err = _lib.load().marlin_hip_rotary_angles(at, freqs.data_ptr(), out.data_ptr(), tokens, pairs, factor, dev,
                                               _raw_stream(dev))
    if err:
        _raise(err)
    return out


def _angles(t: torch.Tensor, tokens: int, head_dim: int, dev: int) -> int:
    """Dims that ``[tokens, pairs, 2]`` angles turn."""
    if not isinstance(t, torch.Tensor):
        raise TypeError("angles must be a torch.Tensor")
    if t.dtype != torch.float64 or t.dim() != 3 or t.size(2) != 2 or t.get_device() != dev or not t.is_contiguous() \
            or t.data_ptr() % 16:
        raise RuntimeError(f"angles must be a contiguous float64 [tokens, pairs, 2] tensor on cuda:{dev}, as "
                           f"rotary_angles makes it")
    if t.size(0) != tokens:
        raise RuntimeError(f"angles are of {t.size(0)} tokens, the rows of {tokens}")
    if not 1 <= t.size(1) <= head_dim // 2:
        raise RuntimeError(f"angles of {t.size(1)} pairs for heads of {head_dim} dims")
    return 2 * t.size(1)


def _strides(t: torch.Tensor):
    """Token and head strides, where there is more than one."""
    st, sh, _ = t.stride()
    return (st if t.size(0) > 1 else 0), (sh if t.size(1) > 1 else t.size(2))


def _apart(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether no element of ``a`` is one of ``b`` (two ``[tokens, heads, D]`` tensors of the same type)."""
    if a.numel() == 0 or b.numel() == 0:
        return True
    (at, ah), (bt, bh) = _strides(a), _strides(b)
    if min(at, ah, bt, bh) < 0:
        return False
    a0, b0 = a.data_ptr(), b.data_ptr()
    # bytes of one token's heads, and of all
    wa, wb = 2 * ((a.size(1) - 1) * ah + a.size(2)), 2 * ((b.size(1) - 1) * bh + b.size(2))
    if a0 + 2 * (a.size(0) - 1) * at + wa <= b0 or b0 + 2 * (b.size(0) - 1) * bt + wb <= a0:
        return True
    # side by side in the rows of one tensor (slices of a fused projection)
    step = 2 * max(at, bt)
    if a.size(0) > 1 and b.size(0) > 1 and at != bt or step == 0:
        return False
    off = (b0 - a0) % step
    return wa <= off and off + wb <= step


def _out_for(x: torch.Tensor, out, dev: int, *others):
    """``out``, checked: x itself or a tensor of its shape apart from it and from the others."""
    if not isinstance(out, torch.Tensor):
        raise TypeError("out must be a torch.Tensor")
    if out.shape != x.shape or out.dtype != x.dtype or out.get_device() != dev:
        raise RuntimeError(f"out must be a {x.dtype} {tuple(x.shape)} tensor on cuda:{dev}")
    yt, yh = _rows("out", out, dev)
    if (out.size(0) > 1 and yt < out.size(2)) or (out.size(1) > 1 and yh < out.size(2)) or (
            out.size(0) > 1 and out.size(1) > 1 and yt < yh * out.size(1) and yh < yt * out.size(0)):
        raise RuntimeError("the rows of out must not overlap one another")
    same = out.data_ptr() == x.data_ptr() and _strides(out) == _strides(x)
    if not same and not _apart(out, x):
        raise RuntimeError("out must be the rotated tensor itself or not overlap it, whose rows are read while out's "
                           "are written")
    for t in others:
        if not _apart(out, t):
            raise RuntimeError("out must not overlap k or v, whose rows are read while out's are written")
    return out


def rotary(x: torch.Tensor, angles: torch.Tensor, interleaved: bool = False, out: torch.Tensor | None = None) -> torch.Tensor:
    """Rows ``x [tokens, heads, D]`` (fp16 or bf16; a view as in :func:`kv4_append`; D a multiple of 8
    up to 1024), the first ``2 pairs`` dims of each turned by its token's ``angles`` and the others as they
    are.  Pairs are ``(i, i + pairs)`` or, ``interleaved``, ``(2 i, 2 i + 1)``.  The products are in 64
    bits, rounded once to ``x``'s type (by way of fp32, as torch does).  Returns ``out``, which may be
    ``x`` itself; its rows may have strides as ``x``'s may.  No gradient flows through the call; turning
    by the angles of the negative positions is its transpose."""
    try:  # (as in kv4_append)
        N, H, D = x.shape
        xt, xh, xd = x.stride()
        dev, dtype, xp, ap = x.get_device(), _DTYPES.get(x.dtype), x.data_ptr(), angles.data_ptr()
        r = 2 * angles.shape[1]
        fits = (dtype is not None and dev >= 0 and out is None and xd == 1 and not (xt | xh | D) & 7 and not (xp | ap) & 15
                and angles.dtype is torch.float64 and angles.get_device() == dev and angles.is_contiguous()
                and angles.shape == (N, r // 2, 2) and 2 <= r <= D <= 1024)
    except (AttributeError, TypeError, ValueError, IndexError):
        fits = False
    if not fits:
        dev = _device_of("x", x)
        xt, xh = _rows("x", x, dev)
        N, H, D = x.shape
        if D % 8 or not 8 <= D <= 1024:
            raise RuntimeError(f"rotary takes heads of a multiple of 8 dims, 1024 at most, got {D}")
        r = _angles(angles, N, D, dev)
        xp, ap, dtype = x.data_ptr(), angles.data_ptr(), _DTYPES[x.dtype]
    if out is None:
        out = torch.empty_like(x) if x.is_contiguous() else x.new_empty((N, H, D))
        yt, yh = H * D, D
    else:
        out = _out_for(x, out, dev)
        yt, yh = _strides(out)
    err = _lib.load().marlin_hip_rotary(xp, ap, out.data_ptr(), N, H, D, r, xt, xh, yt, yh, int(interleaved), dtype, dev,
                                        _raw_stream(dev))
    if err:
        _raise(err)
    return out


def kv4_append_rotary(q: torch.Tensor | None, k: torch.Tensor, v: torch.Tensor, cache: torch.Tensor, slots: torch.Tensor,
                      angles: torch.Tensor, groupsize: int = -1, interleaved: bool = False,
                      out: torch.Tensor | None = None) -> torch.Tensor | None:
    """:func:`rotary` of ``q`` and :func:`kv4_append` of the turned ``k`` and of ``v``, in one launch
    and to the same bits (the turned rows of ``k`` are rounded to their type before they are
    quantized).

    ``q [tokens, q_heads, D]``, ``k, v [tokens, kv_heads, D]``: fp16 or bf16, views as in
    :func:`kv4_append`; ``q`` None: none to turn.  Rows of ``q`` are turned whatever their slot.
    Returns ``q`` turned, in ``out``, which may be ``q`` itself (slices of a fused projection stay
    where they are)."""
    try:  # (as in kv4_append)
        N, H, D = shape = k.shape
        (kt, kh, kd), (vt, vh, vd), (qt, qh, qd) = k.stride(), v.stride(), q.stride()
        pages, heads, width = cache.shape
        Nq, Hq, Dq = q.shape
        dev, dtype = k.get_device(), _DTYPES.get(k.dtype)
        kp, vp, cp, sp, qp, ap = (k.data_ptr(), v.data_ptr(), cache.data_ptr(), slots.data_ptr(), q.data_ptr(),
                                  angles.data_ptr())
        r = 2 * angles.shape[1]
        fits = (dtype is not None and dev >= 0 and out is None and v.dtype is k.dtype and q.dtype is k.dtype
                and v.shape == shape and Nq == N and Dq == D and v.get_device() == q.get_device() == dev
                and kd == vd == qd == 1 and not (kt | kh | vt | vh | qt | qh) & 7 and not (kp | vp | cp | qp | ap) & 15
                and heads == H and cache.dtype is torch.uint8 and cache.get_device() == dev and cache.is_contiguous()
                and slots.dtype is torch.int32 and slots.get_device() == dev and slots.is_contiguous()
                and slots.shape == (N,) and angles.dtype is torch.float64 and angles.get_device() == dev
                and angles.is_contiguous() and angles.shape == (N, r // 2, 2) and 2 <= r <= D)
    except (AttributeError, TypeError, ValueError, IndexError):
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
        r = _angles(angles, N, D, dev)
        qt = qh = Hq = qp = 0
        if q is None:
            if out is not None:
                raise RuntimeError("out without q")
        else:
            _device_of("q", q)
            qt, qh = _rows("q", q, dev)
            if q.dtype != k.dtype or q.size(0) != N or q.size(2) != D:
                raise RuntimeError(f"q is {q.dtype} {tuple(q.shape)}, k is {k.dtype} {tuple(k.shape)}")
            Hq, qp = q.size(1), q.data_ptr()
        pages, _, width = cache.shape
        kp, vp, cp, ap, dtype = k.data_ptr(), v.data_ptr(), cache.data_ptr(), angles.data_ptr(), _DTYPES[k.dtype]
    yp = yt = yh = 0
    if q is not None:
        if out is None:
            out = q.new_empty((N, Hq, D))
            yt, yh = Hq * D, D
        else:
            out = _out_for(q, out, dev, k, v)
            yt, yh = _strides(out)
        yp = out.data_ptr()
    err = _lib.load().marlin_hip_kv4_append_rotary(qp, kp, vp, ap, yp, cp, sp, N, Hq, H, D, r, qt, qh, kt, kh, vt, vh, yt,
                                                   yh, _page_of(width, D, groupsize), pages, groupsize, int(interleaved),
                                                   dtype, dev, _raw_stream(dev))
    if err:
        _raise(err)
    return out
