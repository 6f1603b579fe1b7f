"""Calls whose launch would have 2^32 threads or more are refused before any HIP call:
such a launch starts what is left modulo 2^32, without an error."""

import pytest

from mlx_batch_invariant import _lib

P = 16  # a pointer that is never followed: validation fails first


def _refused(rc, *words):
    err = _lib.lib().bi_last_error().decode()
    assert rc == _lib.EINVAL and any(w in err for w in words), (rc, err)


@pytest.mark.parametrize("dtype", [_lib.F32, _lib.F16, _lib.BF16])
def test_products(dtype):
    L = _lib.lib()
    most = 2 ** 31 - 1
    for M, N in ((most, 16), (16, most), (1, most)):
        _refused(L.bi_gemm(P, P, None, P, M, N, 8, dtype, 1, 1.0, 1.0, None), "too many tiles")
    if dtype != _lib.F32:
        for M, N in ((most, 16), (16, most), (1, most)):
            _refused(L.bi_qgemm(P, P, P, P, P, M, N, 64, 64, 4, dtype, None), "too many tiles")


@pytest.mark.parametrize("dtype", [_lib.F32, _lib.F16, _lib.BF16])
@pytest.mark.parametrize("H, Hkv", [(64, 64), (64, 8)])
def test_attention(dtype, H, Hkv):
    """Few tokens each of very many requests, of 2^30 heads in all."""
    L, D = _lib.lib(), 128
    n = 2 ** 30 // H
    _refused(L.bi_sdpa(P, P, P, None, None, None, P, n, H, Hkv, 1, 16, D, D, None, 0.1, 0, 0, dtype, None),
             "grid too large")
    st = _lib.i64_array((H * D, D, 16 * Hkv * D, 16 * D, D, 16 * Hkv * D, 16 * D, D, 4))
    _refused(L.bi_paged_attention(P, P, P, P, P, P, None, P, n, n, H, Hkv, D, D, 9, 16, 4, st, 0.1, 0, 0, 1, 64,
                                  dtype, None, 0, None), "grid too large")
    st = _lib.i64_array((H * D, D, D, 16 * Hkv * D, 16 * D, D, 16 * Hkv * D, 16 * D, D))
    _refused(L.bi_window_attention(P, P, P, None, P, n, H, Hkv, 1, 16, D, D, st, 0.1, 8, 0, dtype, None, 0, None),
             "grid too large")
    if dtype == _lib.F32:
        return
    st = _lib.i64_array((H * D, D, 16 * Hkv * D, 16 * D, D, 16 * Hkv * D, 16 * D, D, 4))
    _refused(L.bi_paged_attention_q8(P, P, P, P, P, P, P, P, None, P, n, n, H, Hkv, D, D, 9, 16, 4, st,
                                     _lib.i64_array((32, 16, 1) * 2), 0.1, 0, 0, 1, 64, dtype, None, 0, None),
             "grid too large")
