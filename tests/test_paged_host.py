"""The paged cache's operators without a GPU: refusals of the C ABI (before any
HIP call) and of the Python layer, and the shapes torch.compile sees."""

import pytest
import torch

import mlx_batch_invariant as bi
from mlx_batch_invariant import _lib

P = 16  # a pointer that is never followed: validation fails first


def _err():
    return _lib.lib().bi_last_error().decode()


def test_page_tables_abi_refusals():
    L = _lib.lib()

    def call(table=P, ctx=P, used=P, R=2, W=4, F=3, T=5, page=16):
        return L.bi_page_tables(table, ctx, P, P, P, P, P, P, used, R, W, W, F, T, page, None)

    assert call(R=-1) == _lib.EINVAL and "negative" in _err()
    assert call(page=0) == _lib.EINVAL and "page size" in _err()
    assert call(T=1 << 31) == _lib.EINVAL
    assert call(ctx=None) == _lib.EINVAL and "null" in _err()
    assert call(table=None) == _lib.EINVAL
    assert call(used=None) == _lib.EINVAL


def test_paged_update_abi_refusals():
    L = _lib.lib()

    def call(k=P, kc=P, T=4, Hkv=2, D=64, V=64, pages=3, page=16, dtype=_lib.BF16, st=None,
             strides=True):
        st = _lib.i64_array(st or (128, 64, 128, 64, 2048, 1024, 64, 2048, 1024, 64))
        return L.bi_paged_update(k, P, kc, P, P, T, Hkv, D, V, pages, page,
                                 st if strides else None, dtype, None)

    assert call(dtype=7) == _lib.EINVAL and "dtype" in _err()
    assert call(Hkv=0) == _lib.EINVAL and "sizes" in _err()
    assert call(page=0) == _lib.EINVAL
    assert call(pages=1 << 28, page=16) == _lib.EINVAL and "too large" in _err()
    assert call(k=None) == _lib.EINVAL and "null" in _err()
    assert call(strides=False) == _lib.EINVAL
    assert call(k=17) == _lib.EINVAL and "aligned" in _err()
    assert call(T=0) == _lib.OK and call(pages=0) == _lib.OK


def test_attention_abi_refusals():
    L = _lib.lib()

    def paged(q=P, T=4, R=2, H=8, Hkv=2, D=128, V=128, pages=9, page=16, W=4, scale=0.1, window=0,
              first=0, dtype=_lib.BF16, k=P, kn=128):
        st = _lib.i64_array((1024, 128, 4096, 2048, kn, 4096, 2048, 128, W))
        return L.bi_paged_attention(q, k, P, P, P, P, None, P, T, R, H, Hkv, D, V, pages, page, W,
                                    st, scale, window, first, 1, 64, dtype, None, 0, None)

    assert paged(dtype=5) == _lib.EINVAL and "dtype" in _err()
    assert paged(H=6, Hkv=4) == _lib.EINVAL and "multiple" in _err()
    assert paged(D=48, V=48) == _lib.EUNSUPPORTED and "head dims" in _err()
    assert paged(window=-1) == _lib.EINVAL and paged(first=-1) == _lib.EINVAL
    assert paged(scale=float("nan")) == _lib.EINVAL and "NaN" in _err()
    assert paged(page=0) == _lib.EINVAL and paged(R=-1) == _lib.EINVAL
    assert paged(q=None) == _lib.EINVAL and "null" in _err()
    assert paged(k=24) == _lib.EINVAL and "aligned" in _err()
    assert paged(kn=129) == _lib.EINVAL
    assert paged(T=0) == _lib.OK

    def window(q=P, B=1, H=8, Hkv=2, qL=4, N=16, D=128, V=128, w=8, first=0, dtype=_lib.F16):
        st = _lib.i64_array((4096, 512, 128, 4096, 2048, 128, 4096, 2048, 128))
        return L.bi_window_attention(q, P, P, None, P, B, H, Hkv, qL, N, D, V, st, 0.1, w, first,
                                     dtype, None, 0, None)

    assert window(Hkv=3) == _lib.EINVAL
    assert window(D=128, V=96) == _lib.EUNSUPPORTED
    assert window(N=-1) == _lib.EINVAL and window(w=-2) == _lib.EINVAL
    assert window(q=None) == _lib.EINVAL
    assert window(B=0) == _lib.OK and window(qL=0) == _lib.OK


def _i32(*shape):
    return torch.zeros(*shape, dtype=torch.int32)


def test_page_tables_refusals():
    ok = dict(block_tables=_i32(3, 4), context_lens=_i32(3), new_lens=_i32(3), free_pages=_i32(5),
              page_size=16, num_tokens=3)

    def refuse(match, **kw):
        with pytest.raises(ValueError, match=match):
            bi.page_tables(**{**ok, **kw})

    refuse("cuda device")  # right in every other way
    refuse("int32", context_lens=torch.zeros(3, dtype=torch.int64))
    refuse("shape", new_lens=_i32(2))
    refuse("rows", block_tables=_i32(2, 4))
    refuse("contiguous rows", block_tables=_i32(4, 3).T)
    refuse("page_size", page_size=0)
    refuse("num_tokens", num_tokens=-1)


def test_cache_update_refusals():
    kc = torch.zeros(5, 2, 16, 64)
    ok = dict(k=torch.zeros(3, 2, 64), v=torch.zeros(3, 2, 64), k_cache=kc, v_cache=kc.clone(),
              slots=_i32(3))

    def refuse(match, **kw):
        with pytest.raises(ValueError, match=match):
            bi.paged_cache_update(**{**ok, **kw})

    refuse("cuda device")
    refuse("do not fit", k=torch.zeros(3, 2, 32))
    refuse("do not fit", k=torch.zeros(3, 4, 64), v=torch.zeros(3, 4, 64))
    refuse("tokens, Hkv", v=torch.zeros(2, 2, 64))
    refuse("dtype", k=torch.zeros(3, 2, 64).half())
    refuse("shape", slots=_i32(4))
    refuse("int32", slots=torch.zeros(3))
    refuse("num_pages", v_cache=torch.zeros(5, 2, 8, 64))
    refuse("contiguous", k_cache=torch.zeros(5, 2, 64, 16).transpose(2, 3))
    refuse("dtype", k_cache=kc.double(), v_cache=kc.double())


def test_paged_attention_refusals():
    kc = torch.zeros(5, 2, 16, 64)
    ok = dict(q=torch.zeros(3, 8, 64), k_cache=kc, v_cache=kc, block_tables=_i32(2, 4),
              query_start=_i32(3), seq_lens=_i32(2))

    def refuse(match, error=ValueError, **kw):
        with pytest.raises(error, match=match):
            bi.paged_attention(**{**ok, **kw})

    refuse("cuda device")
    refuse("multiple", q=torch.zeros(3, 7, 64))
    refuse("head dimension", q=torch.zeros(3, 8, 32))
    refuse("dtype", q=torch.zeros(3, 8, 64).half())
    refuse("tokens, H", q=torch.zeros(1, 3, 8, 64))
    refuse("shape", query_start=_i32(2))
    refuse("shape", seq_lens=_i32(3))
    refuse("window", window=0)
    refuse("sink_tokens", sink_tokens=-1)
    refuse("sinks", sinks=torch.zeros(7))
    refuse("max_query", max_query=-1)
    k48 = torch.zeros(5, 2, 16, 48)
    refuse("not built", NotImplementedError, q=torch.zeros(3, 8, 48), k_cache=k48, v_cache=k48)


def test_window_attention_refusals():
    ok = dict(q=torch.zeros(2, 8, 3, 64), k=torch.zeros(2, 2, 9, 64), v=torch.zeros(2, 2, 9, 64),
              window=4)

    def refuse(match, error=ValueError, **kw):
        with pytest.raises(error, match=match):
            bi.window_attention(**{**ok, **kw})

    refuse("cuda device")
    refuse("4-dimensional", q=torch.zeros(8, 3, 64))
    refuse("inconsistent", k=torch.zeros(2, 2, 8, 64))
    refuse("dtype", q=torch.zeros(2, 8, 3, 64).half())
    refuse("multiple", k=torch.zeros(2, 3, 9, 64), v=torch.zeros(2, 3, 9, 64))
    refuse("window", window=-3)
    refuse("not built", NotImplementedError, v=torch.zeros(2, 2, 9, 32))


def test_compiled_shapes():
    from torch._subclasses.fake_tensor import FakeTensorMode

    from mlx_batch_invariant import _ops  # noqa: F401

    op = torch.ops.mlx_bi
    with FakeTensorMode():
        got = op.page_tables(_i32(3, 4), _i32(3), _i32(3), _i32(5), 16, 7)
        assert [tuple(t.shape) for t in got] == [(7,), (7,), (4,), (3,), ()]
        kc, vc = torch.empty(5, 2, 16, 192), torch.empty(5, 2, 16, 128)
        y = op.paged_attention(torch.empty(3, 8, 192), kc, vc, _i32(2, 4), _i32(3), _i32(2), 3, 64,
                               0.1, 0, 0, None)
        assert y.shape == (3, 8, 128)
        y = op.window_attention(torch.empty(2, 8, 3, 192), torch.empty(2, 2, 9, 192),
                                torch.empty(2, 2, 9, 128), 0.1, 4, 0, None)
        assert y.shape == (2, 8, 3, 128)


def test_decoder_cache_refusals():
    """The decoder's cache checks a step on the host before any launch."""
    from mlx_batch_invariant import decoder

    c = decoder.DecoderConfig(hidden=64, inter=96, heads=2, kv_heads=1, head_dim=64, layers=1, vocab=50)
    cache = decoder.PagedCache(c, 2, 100, page_size=16, num_pages=5, device="cpu")
    assert cache.tables.shape == (2, 7) and cache.k.shape == (1, 5, 1, 16, 64)
    with pytest.raises(ValueError, match="token counts"):
        cache.begin([1])
    with pytest.raises(ValueError, match="token counts"):
        cache.begin([1, -1])
    with pytest.raises(ValueError, match="max_len"):
        cache.begin([101, 0])
    with pytest.raises(RuntimeError, match="pages"):
        cache.begin([90, 1])
    assert cache.used == 0 and cache.lens == [0, 0]
    for prompts, steps, chunk in (([], 1, None), ([torch.zeros(0).long()], 1, None),
                                  ([torch.zeros(2).long()], 0, None), ([torch.zeros(2).long()], 1, 0)):
        with pytest.raises(ValueError):
            decoder.generate(None, prompts, steps, chunk)
