"""Rotary positions, the 8-bit cache and log probabilities without a GPU:
refusals of the C ABI (before any HIP call) and of the Python layer, and the
frequencies."""

import math

import pytest
import torch

import mlx_batch_invariant as bi
from mlx_batch_invariant import _lib

P = 16  # a pointer that is never followed: validation fails first
I32 = torch.int32


def _err():
    return _lib.lib().bi_last_error().decode()


# --------------------------------------------------------------------- C ABI


def test_rotary_abi_refusals():
    def call(q=P, out=P, pos=P, f=P, T=4, H=2, Hkv=1, D=64, n=32, offset=0, strides=True,
             dtype=_lib.BF16):
        st = _lib.i64_array((128, 64, 64, 64)) if strides else None
        return _lib.lib().bi_rotary(q, P, out, P, pos, f, T, H, Hkv, D, n, offset, st, 1.0, 0, dtype,
                                    None)

    assert call(dtype=9) == _lib.EINVAL and "dtype" in _err()
    assert call(T=-1) == _lib.EINVAL and "sizes" in _err()
    assert call(D=0) == _lib.EINVAL
    assert call(n=33) == _lib.EINVAL and "fit" in _err()
    assert call(offset=1) == _lib.EINVAL and "fit" in _err()
    assert call(n=1 << 62) == _lib.EINVAL and "fit" in _err()
    assert call(offset=1 << 62) == _lib.EINVAL and "fit" in _err()
    assert call(offset=(1 << 63) - 1) == _lib.EINVAL and "fit" in _err()
    assert call(q=None) == _lib.EINVAL and "null" in _err()
    assert call(f=None) == _lib.EINVAL and call(pos=None) == _lib.EINVAL
    assert call(strides=False) == _lib.EINVAL
    assert call(q=17) == _lib.EINVAL and "aligned" in _err()
    assert call(T=1 << 30, H=1 << 20) == _lib.EINVAL and "too large" in _err()
    assert call(T=0) == _lib.OK and call(H=0, Hkv=0) == _lib.OK


def test_update_and_read_abi_refusals():
    st = _lib.i64_array((128, 64, 128, 64, 2048, 1024, 64, 2048, 1024, 64))
    sst = _lib.i64_array((32, 16, 1) * 2)

    def update(k=P, ks=P, T=4, Hkv=2, D=64, V=64, pages=3, page=16, dtype=_lib.BF16, st=st, sst=sst):
        return _lib.lib().bi_paged_update_q8(k, P, P, P, ks, P, P, T, Hkv, D, V, pages, page, st, sst,
                                             0, dtype, None)

    def read(k=P, kc=P, ks=P, vs=P, T=4, Hkv=2, D=64, V=64, pages=3, page=16, dtype=_lib.BF16, st=st,
             sst=sst):
        return _lib.lib().bi_paged_read(kc, P, ks, vs, P, k, P, T, Hkv, D, V, pages, page, st, sst,
                                        dtype, None)

    for call in (update, read):
        assert call(dtype=7) == _lib.EINVAL and "dtype" in _err()
        assert call(Hkv=0) == _lib.EINVAL and "sizes" in _err()
        assert call(page=0) == _lib.EINVAL
        assert call(pages=1 << 28) == _lib.EINVAL and "too large" in _err()
        assert call(T=1 << 30, Hkv=4) == _lib.EINVAL and "too large" in _err()
        assert call(k=None) == _lib.EINVAL and "null" in _err()
        assert call(st=None) == _lib.EINVAL and call(sst=None) == _lib.EINVAL
        assert call(k=17) == _lib.EINVAL and "aligned" in _err()
        assert call(ks=18) == _lib.EINVAL and "aligned" in _err()
        assert call(T=0) == _lib.OK
    assert update(ks=None) == _lib.EINVAL and update(pages=0) == _lib.OK
    assert read(kc=None) == _lib.EINVAL
    assert read(vs=None) == _lib.EINVAL and read(ks=None) == _lib.EINVAL


def test_attention_abi_refusals():
    D = 64
    st = (4 * D, D, 2 * 16 * D, 16 * D, D, 2 * 16 * D, 16 * D, D, 3)
    sst = (32, 16, 1) * 2

    def call(q=P, kc=P, ks=P, table=P, T=4, R=2, H=4, Hkv=2, D=D, V=D, pages=5, page=16, W=3, st=st, sst=sst,
             dtype=_lib.BF16, window=0):
        return _lib.lib().bi_paged_attention_q8(
            q, kc, P, ks, P, table, P, P, None, P, T, R, H, Hkv, D, V, pages, page, W,
            _lib.i64_array(st) if st else None, _lib.i64_array(sst) if sst else None, 0.125, window, 0, 4, 48,
            dtype, None, 0, None)

    other = lambda t, i, x: t[:i] + (x,) + t[i + 1:]
    assert call(dtype=_lib.F32) == _lib.EUNSUPPORTED and "fp32" in _err()
    assert call(dtype=7) == _lib.EINVAL and "dtype" in _err()
    assert call(H=5) == _lib.EINVAL and "multiple" in _err()
    assert call(D=80) == _lib.EUNSUPPORTED and "built" in _err()
    assert call(window=-1) == _lib.EINVAL
    assert call(page=0) == _lib.EINVAL and call(R=-1) == _lib.EINVAL and "sizes" in _err()
    for kw in (dict(q=None), dict(kc=None), dict(ks=None), dict(table=None), dict(st=None), dict(sst=None)):
        assert call(**kw) == _lib.EINVAL and "null" in _err()
    assert call(q=24) == _lib.EINVAL and "16-byte" in _err()
    assert call(kc=24) == _lib.EINVAL and "16-byte" in _err()
    assert call(st=other(st, 4, 72)) == _lib.EINVAL and "16-byte" in _err()  # 72 codes of 8 bits
    assert call(ks=18) == _lib.EINVAL and "scales" in _err()
    for i in (2, 4, 5, 7):  # pages and rows of the caches
        assert call(st=other(st, i, 1 << 32)) == _lib.EUNSUPPORTED and "4 GiB" in _err()
        assert call(st=other(st, i, -64)) == _lib.EUNSUPPORTED
    for i in (0, 2, 3, 5):  # and of the scales
        assert call(sst=other(sst, i, 1 << 30)) == _lib.EUNSUPPORTED and "4 GiB" in _err()
        assert call(sst=other(sst, i, -1)) == _lib.EUNSUPPORTED
    assert call(T=0) == _lib.OK


def test_attention_workspace():
    def ws(T=1, R=1, H=32, Hkv=8, D=128, V=128, window=0, first=0, most=1, longest=8192, dtype=_lib.BF16):
        return _lib.lib().bi_paged_attention_q8_workspace(T, R, H, Hkv, D, V, window, first, most, longest,
                                                          dtype)

    # Two sums and a row of V for each column and segment of 512 rows.
    assert ws() == 32 * 16 * 130 * 4
    assert ws(dtype=_lib.F16) == ws() and ws(longest=8193) == 32 * 17 * 130 * 4
    # Rows laid out for those who walk them whole; not where they would take too much.
    step = -(-(64 * 4 * 128 + 512 + 16) // 512) * 512
    assert ws(T=4096, most=4096) == 8 * 128 * step
    for R in (1 << 10, 1 << 20, 1 << 29):
        for Hkv in (1, 32):
            assert 0 <= ws(T=1 << 25, R=R, H=32, Hkv=Hkv, most=1 << 25, longest=1 << 29) <= 1 << 32
    assert ws(T=0) == ws(R=0) == ws(H=0) == ws(longest=0) == ws(most=0) == 0
    assert ws(dtype=_lib.F32) == ws(D=80) == ws(H=33) == ws(window=-1) == ws(T=1 << 40) == 0


def test_logprobs_abi_refusals():
    def call(x=P, out=P, ids=P, rows=4, V=100, stride=100, top=5, token_bytes=8, dtype=_lib.F16):
        return _lib.lib().bi_token_logprobs(x, P, out, P, ids, P, rows, V, stride, top, token_bytes,
                                            dtype, None)

    assert call(dtype=3) == _lib.EINVAL and "dtype" in _err()
    assert call(V=0) == _lib.EINVAL and call(rows=-1) == _lib.EINVAL and call(stride=-1) == _lib.EINVAL
    assert call(V=1 << 31) == _lib.EINVAL and "sizes" in _err()
    assert call(top=65) == _lib.EINVAL and "top" in _err()
    assert call(V=4) == _lib.EINVAL and "top" in _err()
    assert call(top=-1) == _lib.EINVAL
    assert call(token_bytes=2) == _lib.EINVAL and "tokens" in _err()
    assert call(x=None) == _lib.EINVAL and call(ids=None) == _lib.EINVAL and call(out=None) == _lib.EINVAL
    assert call(x=17) == _lib.EINVAL and "aligned" in _err()
    assert call(rows=0) == _lib.OK


# -------------------------------------------------------------------- Python


def test_rotary_refusals():
    q, k = torch.zeros(3, 4, 64), torch.zeros(3, 2, 64)
    pos, f = torch.zeros(3, dtype=I32), torch.zeros(32, dtype=torch.float64)
    for bad, words in [((q[0], k, pos, f), "tokens, heads"), ((q, k[:2], pos, f), "tokens, heads"),
                       ((q, k[..., :32], pos, f), "tokens, heads"), ((q, k.half(), pos, f), "dtype"),
                       ((q.double(), None, pos, f), "dtype"), ((q, k, pos.long(), f), "int32"),
                       ((q, k, pos[:2], f), "shape"), ((q, k, pos, f.float()), "float64"),
                       ((q, k, pos, f[None]), "float64"), ((q, k, pos, torch.cat([f, f])), "fit")]:
        with pytest.raises(ValueError, match=words):
            bi.rotary(*bad)
    with pytest.raises(ValueError, match="fit"):
        bi.rotary(q, k, pos, f, offset=2)
    with pytest.raises(ValueError, match="fit"):
        bi.rotary(q, k, pos, f[:8], offset=-1)
    with pytest.raises(ValueError, match="GPU"):
        bi.rotary(q, k, pos, f)
    with pytest.raises(NotImplementedError, match="backward"):
        bi.rotary(q.requires_grad_(), k, pos, f)


def test_frequencies():
    f = bi.rotary_frequencies(8, device="cpu")
    assert f.dtype == torch.float64
    assert f.tolist() == pytest.approx([1, 0.1, 0.01, 0.001], rel=1e-14)
    assert bi.rotary_frequencies(8, method="linear", factor=4.0, device="cpu").tolist() == (f / 4).tolist()
    g = bi.rotary_frequencies(8, method="base", factor=4.0, device="cpu")
    assert g[0] == 1 and g[3] == pytest.approx(f[3] / 4, rel=1e-14)
    f = bi.rotary_frequencies(128, base=5e5, device="cpu")
    g = bi.rotary_frequencies(128, base=5e5, method="parts", factor=8.0, original=8192, low=1.0,
                              high=4.0, device="cpu")
    turns = 8192 * f / (2 * math.pi)
    assert (g[turns > 4] == f[turns > 4]).all()
    assert torch.allclose(g[turns < 1], f[turns < 1] / 8, rtol=1e-14)
    mid = (turns > 1) & (turns < 4)
    assert mid.any() and ((g < f) & (g > f / 8))[mid].all()
    for kw in (dict(dim=7), dict(dim=0), dict(dim=8, base=0.0), dict(dim=8, factor=0.0),
               dict(dim=8, method="other"), dict(dim=2, method="base", factor=2.0),
               dict(dim=8, method="parts", factor=2.0),
               dict(dim=8, method="parts", factor=2.0, original=10, low=4.0, high=4.0)):
        with pytest.raises(ValueError):
            bi.rotary_frequencies(**kw, device="cpu")


def q8_cache(pages=4, Hkv=2, page=16, D=64):
    return (torch.zeros(pages, Hkv, page, D, dtype=torch.int8), torch.zeros(pages, Hkv, page, D, dtype=torch.int8),
            torch.zeros(pages, Hkv, page), torch.zeros(pages, Hkv, page))


def test_scales_and_caches_go_together():
    kc, vc, ks, vs = q8_cache()
    x, slots = torch.zeros(3, 2, 64), torch.zeros(3, dtype=I32)
    update = lambda kc=kc, vc=vc, k=x, v=x, **kw: bi.paged_cache_update(k, v, kc, vc, slots, **kw)
    read = lambda kc=kc, vc=vc, **kw: bi.paged_cache_read(kc, vc, slots, **kw)
    for call in (update, read):
        for kw in (dict(), dict(k_scales=ks), dict(v_scales=vs)):
            with pytest.raises(ValueError, match="int8 caches"):
                call(**kw)
        with pytest.raises(ValueError, match="int8 caches"):
            call(kc=kc.float(), vc=vc.float(), k_scales=ks, v_scales=vs)
        with pytest.raises(ValueError, match="int8 caches"):
            call(vc=vc.float(), k_scales=ks, v_scales=vs)
        with pytest.raises(ValueError, match="k_scales must"):
            call(k_scales=ks.half(), v_scales=vs)
        with pytest.raises(ValueError, match="v_scales must"):
            call(k_scales=ks, v_scales=vs[:3])
        with pytest.raises(ValueError, match="GPU"):
            call(k_scales=ks, v_scales=vs)
    with pytest.raises(ValueError, match="dtype"):
        update(k=x.to(torch.int8), v=x.to(torch.int8), k_scales=ks, v_scales=vs)
    with pytest.raises(ValueError, match="dtype"):
        update(k=x.half(), k_scales=ks, v_scales=vs)
    wide = ks[:, :, :1].expand(4, 2, 16)
    with pytest.raises(ValueError, match="v_scales is an expanded"):
        update(k_scales=ks, v_scales=wide)
    with pytest.raises(ValueError, match="GPU"):
        update(k_scales=wide, v_scales=wide, keep_scales=True)
    with pytest.raises(ValueError, match="keep_scales"):
        update(kc=kc.float(), vc=vc.float(), keep_scales=True)
    with pytest.raises(ValueError, match="read as"):
        read(k_scales=ks, v_scales=vs, dtype=torch.int8)
    with pytest.raises(ValueError, match="read as"):
        read(kc=kc.half(), vc=vc.half(), dtype=torch.float32)
    with pytest.raises(ValueError, match="int32"):
        bi.paged_cache_read(kc, vc, slots.long(), k_scales=ks, v_scales=vs)


def test_token_logprobs_refusals():
    x, t = torch.zeros(3, 50), torch.zeros(3, dtype=torch.long)
    for bad, words in [((x.double(), t), "logits"), ((x, t[:2]), "tokens"), ((x, t.short()), "tokens"),
                       ((x[0, 0], t[0]), "logits"), ((x[:, :0], t), "vocabulary")]:
        with pytest.raises(ValueError, match=words):
            bi.token_logprobs(*bad)
    for top in (-1, 51, 65):
        with pytest.raises(ValueError, match="top"):
            bi.token_logprobs(x, t, top=top)
    with pytest.raises(ValueError, match="GPU"):
        bi.token_logprobs(x, t)
    with pytest.raises(NotImplementedError, match="backward"):
        bi.token_logprobs(x.requires_grad_(), t)


def test_attention_over_codes_refusals():
    kc, vc, ks, vs = q8_cache()
    q, start, lens = torch.zeros(3, 4, 64).half(), torch.tensor([0, 3], dtype=I32), torch.tensor([3], dtype=I32)
    table = torch.zeros(1, 2, dtype=I32)

    def call(q=q, kc=kc, vc=vc, **kw):
        return bi.paged_attention(q, kc, vc, table, start, lens, **kw)

    for kw in (dict(), dict(k_scales=ks), dict(v_scales=vs)):
        with pytest.raises(ValueError, match="int8 caches"):
            call(**kw)
    for bad in (dict(kc=kc.half(), vc=vc.half()), dict(vc=vc.half())):
        with pytest.raises(ValueError, match="int8 caches"):
            call(**bad, k_scales=ks, v_scales=vs)
    with pytest.raises(ValueError, match="k_scales must"):
        call(k_scales=ks.half(), v_scales=vs)
    with pytest.raises(ValueError, match="v_scales must"):
        call(k_scales=ks, v_scales=vs[:, :1])
    with pytest.raises(NotImplementedError, match="float32"):
        call(q=q.float(), k_scales=ks, v_scales=vs)
    with pytest.raises(ValueError, match="GPU"):
        call(k_scales=ks, v_scales=vs)


def test_scoring_refusals_and_caches():
    from mlx_batch_invariant import decoder

    c = decoder.DecoderConfig(hidden=64, inter=64, heads=2, kv_heads=1, head_dim=64, layers=2, vocab=16)
    m = decoder.build(c, device="cpu", dtype=torch.float32)
    with pytest.raises(ValueError, match="one token"):
        decoder.score(m, [])
    with pytest.raises(ValueError, match="one token"):
        decoder.score(m, [torch.zeros(3, dtype=torch.long), torch.zeros(0, dtype=torch.long)])
    with pytest.raises(ValueError, match="chunk"):
        decoder.score(m, [torch.zeros(3, dtype=torch.long)], chunk=0)
    assert m.inv_freq is None and m.turn(None) is None
    cache = decoder.PagedCache(c, 2, 50, page_size=16, device="cpu", dtype=torch.int8)
    assert cache.k.dtype == torch.int8 and cache.k_scales.shape == cache.k.shape[:-1] == (2, 8, 1, 16)
    assert cache.scales(1)["v_scales"].data_ptr() == cache.v_scales[1].data_ptr()
    assert decoder.PagedCache(c, 2, 50, device="cpu").scales(0) == {}
    turned = decoder.Decoder(decoder.DecoderConfig(hidden=64, inter=64, heads=2, kv_heads=1, head_dim=64, layers=1,
                                                   vocab=16, rope_base=100.0, rope_dim=8), "cpu", torch.float32)
    assert turned.inv_freq.tolist() == bi.rotary_frequencies(8, 100.0, device="cpu").tolist()


def test_attention_workspace_of_one_chunk_among_many():
    """Rows laid out where one of 64 requests of up to 8192 rows brings a chunk: no more
    than 128 MiB beside the partial results, not a place for every row of all."""
    step = -(-(64 * 4 * 128 + 512 + 16) // 512) * 512
    ws = lambda T, R, most, longest=8192, window=0: _lib.lib().bi_paged_attention_q8_workspace(
        T, R, 32, 8, 128, 128, window, 0, most, longest, _lib.BF16)
    part = lambda R: R * 8 * 32 * 16 * 130 * 4  # 32 columns, 16 segments
    assert part(64) < ws(1063, 64, 1000) <= part(64) + (1 << 27) + 512
    # Requests that all bring a chunk have places for what they walk.
    n = ws(64 * 1000, 64, 1000)
    assert n == 64 * 8 * 128 * step
    n = ws(64 * 1000, 64, 1000, window=1000)
    assert 64 * 8 * 34 * step <= n <= 64 * 8 * 36 * step
    assert ws(4 * 1000, 4, 1000) == 4 * 8 * 128 * step  # within 128 MiB and more: as many as there are


def test_attention_least_workspace():
    """The partial results alone, and nothing where there are none."""
    def ws(T, R, most, least=True, **kw):
        f = _lib.lib().bi_paged_attention_q8_least_workspace if least else _lib.lib().bi_paged_attention_q8_workspace
        return f(T, R, 32, 8, 128, 128, 0, 0, most, 8192, kw.get("dtype", _lib.F16))

    assert ws(1063, 64, 1000) == 64 * 8 * 32 * 16 * 130 * 4 < ws(1063, 64, 1000, False)
    assert ws(64, 64, 1) == ws(64, 64, 1, False) > 0
    assert ws(4096, 1, 4096) == 0 < ws(4096, 1, 4096, False)
    assert ws(4096, 1, 4096, dtype=_lib.F32) == ws(0, 1, 1) == 0


def test_rotary_of_more_than_64_bits_is_refused():
    """Sizes within their bounds whose product passes 2^63."""
    st = _lib.i64_array((1, 1, 1, 1))
    most = 1 << 20
    for T, H, Hkv, D, n in ((2 ** 31 - 1, most, most, most, 0), (2 ** 31 - 1, most, most, most, most // 2),
                            (1 << 30, most // 2, most // 2, most // 2, 3), (2 ** 31 - 1, most, most, most // 4, 0),
                            (1 << 26, most, 0, most, 0), (2 ** 31 - 1, 1, 0, 16, 8)):
        rc = _lib.lib().bi_rotary(P, P, P, P, P, P, T, H, Hkv, D, n, 0, st, 1.0, 0, _lib.F32, None)
        assert rc == _lib.EINVAL and "too large" in _err(), (T, H, Hkv, D, n)


@pytest.mark.parametrize("D, V", [(64, 0), (0, 64)])
def test_caches_of_one_side_are_refused(D, V):
    """Keys without values, or values without keys: nothing was written, and zeros read."""
    x = lambda d: torch.zeros(3, 2, d).half()
    slots = torch.zeros(3, dtype=I32)
    caches = torch.zeros(4, 2, 16, D).half(), torch.zeros(4, 2, 16, V).half()
    codes = tuple(c.to(torch.int8) for c in caches)
    scales = dict(k_scales=torch.zeros(4, 2, 16), v_scales=torch.zeros(4, 2, 16))
    for call in (lambda: bi.paged_cache_update(x(D), x(V), *caches, slots),
                 lambda: bi.paged_cache_update(x(D), x(V), *codes, slots, **scales),
                 lambda: bi.paged_cache_read(*caches, slots), lambda: bi.paged_cache_read(*codes, slots, **scales)):
        with pytest.raises(ValueError, match="head dim"):
            call()
