"""Rotary positions of queries and keys, batch-invariant.

    inv_freq = bi.rotary_frequencies(128)
    q, k = bi.rotary(q, k, t.positions, inv_freq)       # t: bi.page_tables' result

Angles are reduced in 64 bits inside the kernel (csrc/bi_rotary.hip), so there
is no table of sines and cosines to keep, and far positions are as exact as near
ones. A token's result depends on the token and its position alone. There is no
backward pass.
"""

import ctypes
import math

import torch

from . import _lib
from ._paged import _at, _call, _int32, _no_grad, _on_one_gpu

_I64x4 = ctypes.c_int64 * 4


def rotary_frequencies(dim, base=10000.0, *, method=None, factor=1.0, original=None, low=1.0,
                       high=32.0, device="cuda"):
    """The ``dim // 2`` angles per position that :func:`rotary` takes, float64:
    pair i turns by ``base ** (-2 i / dim)`` radians.

    ``method`` scales them for contexts ``factor`` times as long as the
    ``original`` tokens a model was trained on:

    - ``"linear"``: all divided by ``factor``;
    - ``"base"``: the base becomes ``base * factor ** (dim / (dim - 2))``, which
      leaves the fastest pair as it is and divides the slowest by ``factor``;
    - ``"parts"``: a pair that turns more than ``high`` times in ``original``
      tokens keeps its angle, one that turns less than ``low`` times has it
      divided by ``factor``, and those between blend both linearly.
    """
    if dim < 2 or dim % 2:
        raise ValueError("dim must be even and at least 2, got %r" % (dim,))
    if not base > 0 or not factor > 0:
        raise ValueError("base and factor must be positive, got %r and %r" % (base, factor))
    if method not in (None, "linear", "base", "parts"):
        raise ValueError("method must be None, 'linear', 'base' or 'parts', got %r" % (method,))
    if method == "base":
        if dim == 2:
            raise ValueError("method 'base' needs dim of 4 or more")
        base = base * factor ** (dim / (dim - 2))
    f = base ** (-torch.arange(0, dim, 2, dtype=torch.float64) / dim)
    if method == "linear":
        f = f / factor
    elif method == "parts":
        if not original or not high > low:
            raise ValueError("method 'parts' needs original and high > low, got %r, %r and %r"
                             % (original, high, low))
        keep = ((original * f / (2 * math.pi) - low) / (high - low)).clamp(0, 1)
        f = f * (keep + (1 - keep) / factor)
    return f.to(device)


def rotary(q, k, positions, inv_freq, *, interleaved=False, offset=0, scale=1.0):
    """Turns the pairs of every head of ``q`` (T, H, D) and ``k`` (T, Hkv, D; or
    None) by their token's position: (x, y) becomes scale * (x cos a - y sin a,
    x sin a + y cos a), a = positions[t] * inv_freq[i]. Returns (q, k), new and
    contiguous.

    ``positions`` (T,) is int32, as :func:`page_tables` returns them, and may be
    negative. ``inv_freq`` (n,) is float64 on the GPU
    (:func:`rotary_frequencies`). Pair i is dims ``offset + i`` and ``offset + n
    + i`` of a head, with ``interleaved`` dims ``offset + 2 i`` and ``offset + 2
    i + 1``; the other dims are copied. ``scale`` multiplies the turned dims.
    ``q`` and ``k`` may be strided views, such as slices of a projection's
    output.
    """
    qs, dt = q.shape, q.dtype
    ks = qs if k is None else k.shape
    if len(qs) != 3 or len(ks) != 3 or ks[0] != qs[0] or ks[2] != qs[2]:
        raise ValueError("q and k must be (tokens, heads, head dim), got %s and %s"
                         % (tuple(qs), None if k is None else tuple(ks)))
    if dt not in _lib.DTYPE_CODES or (k is not None and k.dtype is not dt):
        raise ValueError("q and k must share a dtype of float32, float16 or bfloat16, got %s and %s"
                         % (dt, None if k is None else k.dtype))
    _int32("positions", positions, qs[0])
    if inv_freq.dtype is not torch.float64 or inv_freq.ndim != 1:
        raise ValueError("inv_freq must be float64 of one dimension, got %s of shape %s"
                         % (inv_freq.dtype, tuple(inv_freq.shape)))
    n = inv_freq.shape[0]
    if offset < 0 or offset + 2 * n > qs[2]:
        raise ValueError("%d pairs from dim %r on do not fit heads of %d" % (n, offset, qs[2]))
    _no_grad("rotary", q, k)
    args = (q, k, positions, inv_freq, bool(interleaved), int(offset), float(scale))
    if torch.compiler.is_compiling():
        from . import _ops  # noqa: F401  (registers the ops)

        if k is None:
            return torch.ops.mlx_bi.rotary(q, q[:, :0], *args[2:])[0], None
        return tuple(torch.ops.mlx_bi.rotary(*args))
    return _rotary_eager(*args)


def _rotary_eager(q, k, positions, inv_freq, interleaved, offset, scale):
    dev = q.device
    _on_one_gpu("rotary", dev, (k, positions, inv_freq))
    T, H, D = q.shape
    Hkv = 0 if k is None else k.shape[1]
    q_out = torch.empty((T, H, D), dtype=q.dtype, device=dev)
    k_out = None if k is None else torch.empty((T, Hkv, D), dtype=q.dtype, device=dev)
    if not T or not D or not H + Hkv:
        return q_out, k_out
    qt, qh, one = q.stride()
    if one != 1:
        q = q.contiguous()
        qt, qh, _ = q.stride()
    kt = kh = 0
    if k is not None:
        kt, kh, one = k.stride()
        if one != 1:
            k = k.contiguous()
            kt, kh, _ = k.stride()
    positions, inv_freq = positions.contiguous(), inv_freq.contiguous()
    _call(dev, "bi_rotary", _lib.lib().bi_rotary, q.data_ptr(), _at(k), q_out.data_ptr(), _at(k_out),
          positions.data_ptr(), inv_freq.data_ptr(), T, H, Hkv, D, inv_freq.shape[0], offset,
          _I64x4(qt, qh, kt, kh), scale, interleaved, _lib.DTYPE_CODES[q.dtype])
    return q_out, k_out
