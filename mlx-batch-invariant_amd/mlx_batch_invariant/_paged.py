"""A paged key/value cache and attention over it, batch-invariant.

A cache is two tensors of pages, ``k_cache`` (num_pages, Hkv, page_size, D) and
``v_cache`` (num_pages, Hkv, page_size, V); any strides but a contiguous last
dimension, so a token-major pool is passed as ``pool.transpose(1, 2)``. Request
r keeps its row i in page ``block_tables[r, i // page_size]``, row
``i % page_size``. A serving step is

    t = bi.page_tables(block_tables, context_lens, new_lens, free_pages, page_size, tokens)
    bi.paged_cache_update(k, v, k_cache, v_cache, t.slots)
    o = bi.paged_attention(q, k_cache, v_cache, t.block_tables, t.query_start, t.seq_lens)

for the step's tokens laid out one request behind the other, one new token per
request (decode), a chunk of a prompt, or any mixture. Nothing is read back to
the host, so a step can be captured in a HIP graph and replayed with other
lengths. :func:`window_attention` is the same attention over contiguous keys.

Keys are taken by their position in the request, in segments of a fixed length
whose results are folded in a fixed order: a token's output has the same bits
whatever else is in the batch, however many tokens are new, whichever pages
hold its keys, and for paged and contiguous keys alike. Rows that a token does
not see never reach it, infinities and NaN in them included. The kernels
(csrc/bi_paged*.hip) have no backward pass.
"""

import collections
import ctypes
import functools
import math

import torch

from . import _lib
from ._attention import _kernel_view

PAGED_HEAD_DIMS = ((64, 64), (96, 96), (128, 128), (192, 128), (192, 192), (256, 256))

PageTables = collections.namedtuple(
    "PageTables", ("block_tables", "slots", "positions", "query_start", "seq_lens", "pages_used"))


_I32 = torch.int32
_I64x9 = ctypes.c_int64 * 9
_I64x10 = ctypes.c_int64 * 10


def _on_one_gpu(what, dev, tensors):
    if dev.type == "cuda":
        for t in tensors:
            if t is not None and t.device != dev:
                break
        else:
            return
    raise ValueError("%s runs on the GPU; all operands must be on one cuda device, got %s"
                     % (what, sorted({str(t.device) for t in tensors if t is not None} | {str(dev)})))


def _int32(name, t, *shape):
    """Checks for int32 and a shape; None in it: any length."""
    if t.dtype is _I32 and (t.shape == shape or shape == (None,) and t.ndim == 1):
        return
    if t.dtype != _I32:
        raise ValueError("%s must be int32, got %s" % (name, t.dtype))
    if t.ndim != len(shape) or any(s is not None and s != n for s, n in zip(shape, t.shape)):
        raise ValueError("%s must have shape (%s), got %s"
                         % (name, ", ".join("any" if s is None else str(s) for s in shape),
                            tuple(t.shape)))


def _table(t):
    """Distance of the (R, W) table's rows, which are contiguous."""
    if t.dtype is not _I32 or t.ndim != 2:
        _int32("block_tables", t, None, None)
    W = t.shape[1]
    row, one = t.stride()
    if W > 1 and one != 1:
        raise ValueError("block_tables must have contiguous rows")
    return row if t.shape[0] > 1 else W


def _call(device, what, fn, *args):
    stream, switch = _lib.launch_stream(device)
    if switch:
        with torch.cuda.device(device):
            rc = fn(*args, stream)
    else:
        rc = fn(*args, stream)
    if rc:
        _lib.check(rc, what)


def _at(t):
    return None if t is None else t.data_ptr()


def page_tables(block_tables, context_lens, new_lens, free_pages, page_size, num_tokens):
    """Block tables and slot maps of a step, from the requests' lengths.

    ``context_lens`` and ``new_lens`` (R,) are the rows each request has in the
    cache and those it brings now; ``free_pages`` (F,) lists unused pages. All
    are int32 on the GPU. The pages that the new rows begin are taken from the
    front of ``free_pages``, request by request, and written into
    ``block_tables`` (R, W) in place (-1 where the free pages do not reach; no
    other entry changes). Returns a :class:`PageTables`:

    - ``block_tables``: the table itself;
    - ``slots`` (num_tokens,): page * page_size + row of every new token, -1
      for a token without a page and for the places behind the last token;
    - ``positions`` (num_tokens,): its row in the request, -1 behind the last;
    - ``query_start`` (R + 1,), ``seq_lens`` (R,): what attention takes;
    - ``pages_used`` (): pages taken; more than F if they ran out.

    ``num_tokens`` is the length of the step's token tensors: the sum of
    ``new_lens``, or more for a padded step.
    """
    _int32("context_lens", context_lens, None)
    R = context_lens.shape[0]
    _int32("new_lens", new_lens, R)
    _int32("free_pages", free_pages, None)
    row = _table(block_tables)
    if block_tables.shape[0] != R:
        raise ValueError("block_tables must have %d rows, got %d" % (R, block_tables.shape[0]))
    if page_size < 1 or num_tokens < 0:
        raise ValueError("page_size must be positive and num_tokens not negative, got %r and %r"
                         % (page_size, num_tokens))
    if torch.compiler.is_compiling():
        from . import _ops  # noqa: F401  (registers the ops)

        return PageTables(block_tables, *torch.ops.mlx_bi.page_tables(
            block_tables, context_lens, new_lens, free_pages, int(page_size), num_tokens))
    return PageTables(block_tables, *_page_tables_eager(block_tables, context_lens, new_lens,
                                                        free_pages, page_size, num_tokens, row))


def _page_tables_eager(block_tables, context_lens, new_lens, free_pages, page_size, num_tokens,
                       row=None):
    dev = context_lens.device
    _on_one_gpu("page_tables", dev, (block_tables, new_lens, free_pages))
    (R, W), T = block_tables.shape, int(num_tokens)
    # One allocation for all outputs.
    buf = torch.empty(2 * T + 2 * R + 2, dtype=_I32, device=dev)
    slots, positions, start, seq, used = buf.split_with_sizes((T, T, R + 1, R, 1))
    context_lens, new_lens = context_lens.contiguous(), new_lens.contiguous()
    free_pages = free_pages.contiguous()
    at = buf.data_ptr()
    _call(dev, "bi_page_tables", _lib.lib().bi_page_tables, block_tables.data_ptr(),
          context_lens.data_ptr(), new_lens.data_ptr(), free_pages.data_ptr(), at, at + 4 * T,
          at + 8 * T, at + 8 * T + 4 * R + 4, at + 8 * T + 8 * R + 4, R, W,
          _table(block_tables) if row is None else row,
          free_pages.shape[0], T, int(page_size))
    return slots, positions, start, seq, used.view(())


def _cache_shapes(k_cache, v_cache):
    """The caches' strides (page, head, row, 1), after their checks."""
    ks, vs = k_cache.shape, v_cache.shape
    if len(ks) != 4 or len(vs) != 4 or ks[:3] != vs[:3]:
        raise ValueError("caches must be (num_pages, Hkv, page_size, head dim), got %s and %s"
                         % (tuple(ks), tuple(vs)))
    kst, vst = k_cache.stride(), v_cache.stride()
    if kst[3] != 1 or vst[3] != 1:
        raise ValueError("the caches' last dimension must be contiguous")
    if k_cache.dtype != v_cache.dtype or k_cache.dtype not in _lib.DTYPE_CODES:
        raise ValueError("caches must share a dtype of float32, float16 or bfloat16, got %s and %s"
                         % (k_cache.dtype, v_cache.dtype))
    if ks[0] * ks[2] >= 2 ** 31:
        raise ValueError("a cache holds fewer than 2**31 rows per head, got %d pages of %d"
                         % (ks[0], ks[2]))
    return kst, vst


def paged_cache_update(k, v, k_cache, v_cache, slots):
    """Writes new tokens' keys (T, Hkv, D) and values (T, Hkv, V) into the
    caches, in place: token t goes to row ``slots[t] % page_size`` of page
    ``slots[t] // page_size`` (int32, from :func:`page_tables`). A token whose
    slot is negative or not a row of the cache is not written. The slots that
    are written must be distinct. ``k`` and ``v`` may be strided views, such as
    slices of a projection's output."""
    _cache_shapes(k_cache, v_cache)
    if k.ndim != 3 or v.ndim != 3 or k.shape[:2] != v.shape[:2]:
        raise ValueError("k and v must be (tokens, Hkv, head dim), got %s and %s"
                         % (tuple(k.shape), tuple(v.shape)))
    if (k.shape[1], k.shape[2], v.shape[2]) != (k_cache.shape[1], k_cache.shape[3],
                                                v_cache.shape[3]):
        raise ValueError("k %s and v %s do not fit caches %s and %s"
                         % (tuple(k.shape), tuple(v.shape), tuple(k_cache.shape),
                            tuple(v_cache.shape)))
    if not k.dtype == v.dtype == k_cache.dtype:
        raise ValueError("k and v must share the caches' dtype %s, got %s and %s"
                         % (k_cache.dtype, k.dtype, v.dtype))
    _int32("slots", slots, k.shape[0])
    if torch.compiler.is_compiling():
        from . import _ops  # noqa: F401  (registers the ops)

        torch.ops.mlx_bi.paged_cache_update(k, v, k_cache, v_cache, slots)
    else:
        _update_eager(k, v, k_cache, v_cache, slots)


def _update_eager(k, v, k_cache, v_cache, slots):
    dev = k.device
    _on_one_gpu("paged_cache_update", dev, (v, k_cache, v_cache, slots))
    T, Hkv, D = k.shape
    P, _, page, V = v_cache.shape
    if not (T and P and Hkv and page and D and V):
        return
    kt, kh, one = k.stride()
    if one != 1:
        k = k.contiguous()
        kt, kh, _ = k.stride()
    vt, vh, one = v.stride()
    if one != 1:
        v = v.contiguous()
        vt, vh, _ = v.stride()
    slots = slots.contiguous()
    kp, kg, kr, _ = k_cache.stride()
    vp, vg, vr, _ = v_cache.stride()
    st = _I64x10(kt, kh, vt, vh, kp, kg, kr, vp, vg, vr)
    _call(dev, "bi_paged_update", _lib.lib().bi_paged_update, k.data_ptr(), v.data_ptr(),
          k_cache.data_ptr(), v_cache.data_ptr(), slots.data_ptr(), T, Hkv, D, V, P, page, st,
          _lib.DTYPE_CODES[k.dtype])


def _attention_options(q, D, V, H, Hkv, scale, window, sink_tokens, sinks):
    if q.dtype not in _lib.DTYPE_CODES:
        raise ValueError("unsupported dtype %s" % q.dtype)
    if Hkv == 0 or H % Hkv:
        raise ValueError("head count %d is not a multiple of kv head count %d" % (H, Hkv))
    if (D, V) not in PAGED_HEAD_DIMS:
        raise NotImplementedError("head dimensions D=%d V=%d are not built (built (D, V): %s)"
                                  % (D, V, PAGED_HEAD_DIMS))
    if window is not None and window < 1:
        raise ValueError("window must be None or at least 1, got %r" % (window,))
    if sink_tokens < 0:
        raise ValueError("sink_tokens must not be negative, got %r" % (sink_tokens,))
    if sinks is not None:
        if tuple(sinks.shape) != (H,):
            raise ValueError("sinks must have shape (%d,), got %s" % (H, tuple(sinks.shape)))
        sinks = sinks.to(q.dtype).contiguous()
    return 1.0 / math.sqrt(D) if scale is None else float(scale), int(window or 0), sinks


def paged_attention(q, k_cache, v_cache, block_tables, query_start, seq_lens, *, max_query=None,
                    max_seq=None, scale=None, window=None, sink_tokens=0, sinks=None):
    """Causal attention of a step's tokens over a paged cache that holds their
    keys and values already.

    ``q`` (T, H, D) holds the requests' new tokens one request behind the
    other: tokens ``query_start[r]`` to ``query_start[r + 1] - 1`` are the last
    ones of request r's ``seq_lens[r]`` rows (int32, as :func:`page_tables`
    returns them). Returns (T, H, V); tokens that no request owns, and tokens
    that see nothing, are 0. H is a multiple of Hkv.

    ``window=w`` lets a token at position p see rows j > p - w only, and
    besides them the first ``sink_tokens`` rows. ``sinks`` (H,) is a logit per
    head that enters its denominator, rounded to q's type. Rows whose table
    entry is not a page of the cache are not seen. A call of many tokens per
    request takes far longer where a value that only some of them see is
    infinite or NaN.

    ``max_query`` and ``max_seq`` bound the requests' new tokens and lengths
    (by default T and the table's capacity). The launch is sized by them, so
    tight bounds are faster; a request beyond one gets NaN.
    """
    _cache_shapes(k_cache, v_cache)
    if q.ndim != 3:
        raise ValueError("q must be (tokens, H, head dim), got %s" % (tuple(q.shape),))
    if q.dtype != k_cache.dtype:
        raise ValueError("q must share the caches' dtype %s, got %s" % (k_cache.dtype, q.dtype))
    T, H, D = q.shape
    P, Hkv, page, Dk = k_cache.shape
    if D != Dk:
        raise ValueError("q has head dimension %d, the cache %d" % (D, Dk))
    _table(block_tables)
    R = block_tables.shape[0]
    _int32("query_start", query_start, R + 1)
    _int32("seq_lens", seq_lens, R)
    scale, window, sinks = _attention_options(q, D, v_cache.shape[3], H, Hkv, scale, window,
                                              sink_tokens, sinks)
    max_query = T if max_query is None else max_query
    capacity = block_tables.shape[1] * page
    max_seq = capacity if max_seq is None else max_seq
    if max_query < 0 or max_seq < 0:
        raise ValueError("max_query and max_seq must not be negative, got %r and %r"
                         % (max_query, max_seq))
    args = (q, k_cache, v_cache, block_tables, query_start, seq_lens, max_query, max_seq, scale,
            window, int(sink_tokens), sinks)
    if torch.compiler.is_compiling():
        from . import _ops  # noqa: F401  (registers the ops)

        return torch.ops.mlx_bi.paged_attention(*args)
    return _paged_eager(*args)


@functools.lru_cache(maxsize=1024)
def _paged_bytes(device, *sizes):
    return _lib.lib().bi_paged_attention_workspace(*sizes)


@functools.lru_cache(maxsize=1024)
def _window_bytes(device, *sizes):
    return _lib.lib().bi_window_attention_workspace(*sizes)


def _workspace(need, device):
    """The partial results' memory, or None where it cannot be had (the same
    bits, slower). It is used by this stream's launches only, so the caching
    allocator may give it to the next call on the stream once dropped."""
    if not need:
        return None
    try:
        return torch.empty(need, dtype=torch.uint8, device=device)
    except torch.OutOfMemoryError:
        return None


def _paged_eager(q, k_cache, v_cache, block_tables, query_start, seq_lens, max_query, max_seq,
                 scale, window, sink_tokens, sinks):
    dev = q.device
    _on_one_gpu("paged_attention", dev, (k_cache, v_cache, block_tables, query_start, seq_lens,
                                         sinks))
    kp, kh, kn, _ = k_cache.stride()
    vp, vh, vn, _ = v_cache.stride()
    ka, va = k_cache.data_ptr(), v_cache.data_ptr()
    if (kp | kh | kn | vp | vh | vn) * q.element_size() % 16 or (ka | va) % 16:
        raise ValueError("the caches must be 16-byte aligned, with strides of multiples of 16 bytes")
    T, H, D = q.shape
    P, Hkv, page, V = v_cache.shape
    R, W = block_tables.shape
    out = torch.empty((T, H, V), dtype=q.dtype, device=dev)
    if not T:
        return out
    q = _kernel_view(q)
    query_start, seq_lens = query_start.contiguous(), seq_lens.contiguous()
    qt, qh, _ = q.stride()
    st = _I64x9(qt, qh, kp, kh, kn, vp, vh, vn, _table(block_tables))
    dt = _lib.DTYPE_CODES[q.dtype]
    need = _paged_bytes(dev, T, R, H, Hkv, D, V, window, sink_tokens, max_query, max_seq, dt)
    ws = _workspace(need, dev)
    _call(dev, "bi_paged_attention", _lib.lib().bi_paged_attention, q.data_ptr(), ka, va,
          block_tables.data_ptr(), query_start.data_ptr(), seq_lens.data_ptr(), _at(sinks),
          out.data_ptr(), T, R, H, Hkv, D, V, P, page, W, st, scale, window, sink_tokens,
          max_query, max_seq, dt, _at(ws), 0 if ws is None else need)
    return out


def window_attention(q, k, v, window, *, sink_tokens=0, scale=None, sinks=None):
    """Causal attention with a sliding window over contiguous keys. ``q`` is
    (B, H, L, D), ``k``/``v`` are (B, Hkv, N, ...); query row s sits at position
    p = N - L + s and sees keys j <= p with j > p - ``window``, and besides
    them the first ``sink_tokens`` keys (``window=None``: all j <= p). ``sinks``
    (H,) is a logit per head that enters its denominator. A row that sees
    nothing is 0. Returns (B, H, L, V); the bits are :func:`paged_attention`'s
    for the same rows."""
    if q.ndim != 4 or k.ndim != 4 or v.ndim != 4:
        raise ValueError("q, k and v must be 4-dimensional (B, H, L, D)")
    if not (q.dtype == k.dtype == v.dtype):
        raise ValueError("q, k and v must share a dtype")
    B, H, L, D = q.shape
    Hkv, N, V = k.shape[1], k.shape[2], v.shape[3]
    if tuple(k.shape) != (B, Hkv, N, D) or tuple(v.shape) != (B, Hkv, N, V):
        raise ValueError("inconsistent q/k/v shapes: %s %s %s"
                         % (tuple(q.shape), tuple(k.shape), tuple(v.shape)))
    scale, window, sinks = _attention_options(q, D, V, H, Hkv, scale, window, sink_tokens, sinks)
    args = (q, k, v, scale, window, int(sink_tokens), sinks)
    if torch.compiler.is_compiling():
        from . import _ops  # noqa: F401  (registers the ops)

        return torch.ops.mlx_bi.window_attention(*args)
    return _window_eager(*args)


def _window_eager(q, k, v, scale, window, sink_tokens, sinks):
    dev = q.device
    _on_one_gpu("window_attention", dev, (k, v, sinks))
    B, H, qL, D = q.shape
    _, Hkv, N, V = v.shape
    out = torch.empty((B, H, qL, V), dtype=q.dtype, device=dev)
    if not (B and qL):
        return out
    q, k, v = _kernel_view(q), _kernel_view(k), _kernel_view(v)
    st = _I64x9(*q.stride()[:3], *k.stride()[:3], *v.stride()[:3])
    dt = _lib.DTYPE_CODES[q.dtype]
    need = _window_bytes(dev, B, H, Hkv, qL, N, D, V, window, sink_tokens, dt)
    ws = _workspace(need, dev)
    _call(dev, "bi_window_attention", _lib.lib().bi_window_attention, q.data_ptr(), k.data_ptr(),
          v.data_ptr(), _at(sinks), out.data_ptr(), B, H, Hkv, qL, N, D, V, st, scale, window,
          sink_tokens, dt, _at(ws), 0 if ws is None else need)
    return out
