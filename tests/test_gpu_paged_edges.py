"""Calls of the paged cache's operators that their documentation allows and
that lie at its edges."""

import pytest
import torch

import mlx_batch_invariant as bi

import paged_ref as ref

pytestmark = pytest.mark.gpu
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def i32(x, device):
    return torch.tensor(x, dtype=torch.int32, device=device)


def test_slots_of_entries_that_are_no_pages(cuda):
    """A page number whose slots pass 31 bits gives no slot: not that of the page
    it would wrap to, neither as a table's entry nor as a free page."""
    page = 16
    far = [2 ** 27 - 1, 2 ** 27, 2 ** 28, 2 ** 28 + 1, 2 ** 31 - 1]  # the first one's slots just fit
    table = i32([[p, -1] for p in far], cuda)
    t = bi.page_tables(table, i32([3] * 5, cuda), i32([14] * 5, cuda), i32(far, cuda), page, 70)
    assert table[:, 1].tolist() == far  # the 14th token's page
    want = []
    for p in far:
        rows = [p * page + r for r in range(3, 16)] + [p * page]
        want += [s if s < 2 ** 31 else -1 for s in rows]
    assert t.slots.tolist() == want and want[:2] == [2 ** 31 - 13, 2 ** 31 - 12]
    # The cache is left alone by all but those of a page that it has.
    kc = torch.zeros(4, 1, page, 64, dtype=BF16, device=cuda)
    vc = torch.zeros_like(kc)
    k = torch.ones(70, 1, 64, dtype=BF16, device=cuda)
    bi.paged_cache_update(k, k, kc, vc, t.slots)
    assert not bool(kc.any()) and not bool(vc.any())


def as_int(x):
    return x.contiguous().view(torch.int32 if x.dtype == F32 else torch.int16)


@pytest.mark.parametrize("D, V", [(64, 64), (96, 96), (128, 128), (192, 128), (192, 192), (256, 256)])
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("L, H, Hkv", [(6, 8, 2), (40, 8, 8), (500, 12, 2), (300, 3, 1)])
@pytest.mark.parametrize("window, first", [(None, 0), (130, 3)])
def test_a_token_is_safe_from_rows_that_only_others_see(cuda, dtype, D, V, L, H, Hkv, window, first):
    """Infinities and NaN in keys and values that some of a chunk's tokens see,
    as the window begins and as it ends: the others have the bits that they have
    without them, those that see one the bits that they have alone."""
    n, page = 900, 16
    g = torch.Generator(device=cuda).manual_seed(D + V + L)
    rn = lambda *s: torch.randn(*s, generator=g, device=cuda).to(dtype)
    k, v, q = rn(1, Hkv, n, D), rn(1, Hkv, n, V), rn(1, H, L, D)
    run = lambda k, v, lo, hi: bi.window_attention(q[:, :, lo:hi], k[:, :, :n - L + hi],
                                                   v[:, :, :n - L + hi], window, sink_tokens=first)
    clean = run(k, v, 0, L)
    kb, vb = k.clone(), v.clone()
    inf, nan = float("inf"), float("nan")
    at = n - L + L // 2  # from this token on
    vb[:, :, at, 0], vb[:, 0, at, 5], vb[:, :, at, V - 1] = inf, nan, -inf
    kb[:, :, at + 2, 3] = nan
    bad = [at, at + 2]
    if window:
        early = n - L - window + 1 + L // 3  # up to the token window - 1 behind it
        vb[:, :, early, 1] = -inf
        bad.append(early)
    got = run(kb, vb, 0, L)
    pos = torch.arange(n - L, n, device=cuda)
    sees = torch.zeros(L, dtype=torch.bool, device=cuda)
    for b in bad:
        sees |= (b <= pos) & ((b > pos - window) if window else True)
    assert bool(sees.any()) and (bool((~sees).any()) or L == 6)  # 6: each sees one of them, none both
    free = ~sees
    assert torch.equal(as_int(got[:, :, free]), as_int(clean[:, :, free]))
    edge = set(range(min(L, 3))) | {L // 3, L // 3 + 1, L // 2 - 1, L // 2, L // 2 + 1, L // 2 + 2, L - 1}
    for t in sorted(edge):
        alone = run(kb, vb, t, t + 1)
        assert torch.equal(as_int(got[:, :, t:t + 1]), as_int(alone)), t
        if sees[t]:
            assert not bool(alone.isfinite().all())
    # Over pages, beside a single token of the same request.
    pages = -(-n // page)
    order = torch.randperm(pages, generator=g, device=cuda)
    i = torch.arange(n, device=cuda)
    kc, vc = rn(pages, Hkv, page, D), rn(pages, Hkv, page, V)
    kc[order[i // page], :, i % page], vc[order[i // page], :, i % page] = kb[0].transpose(0, 1), vb[0].transpose(0, 1)
    table = order.to(torch.int32)[None].repeat(2, 1)
    qt = q[0].transpose(0, 1)
    y = bi.paged_attention(torch.cat([qt, qt[L // 3:L // 3 + 1]]), kc, vc, table, i32([0, L, L + 1], cuda),
                           i32([n, n - L + L // 3 + 1], cuda), window=window, sink_tokens=first)
    want = got[0].transpose(0, 1)
    assert torch.equal(as_int(y[:L]), as_int(want))
    assert torch.equal(as_int(y[L:]), as_int(want[L // 3:L // 3 + 1]))


@pytest.mark.parametrize("dtype, D", [(BF16, 128), (F16, 64), (BF16, 256), (F32, 96)])
@pytest.mark.parametrize("border", [512, 1024])
@pytest.mark.parametrize("window, first", [(None, 0), (40, 0), (12, 2)])
def test_a_token_is_safe_where_segments_meet(cuda, dtype, D, border, window, first):
    """Tokens on both sides of a segment's border, so that some see nothing of
    a segment that others see, with NaN in values before and behind it."""
    n, L, H, Hkv = border + 11, 24, 6, 3
    g = torch.Generator(device=cuda).manual_seed(border + D)
    rn = lambda *s: torch.randn(*s, generator=g, device=cuda).to(dtype)
    q, k, v = rn(1, H, L, D), rn(1, Hkv, n, D), rn(1, Hkv, n, D)
    nan = float("nan")
    v[:, 0, border + 4, 7] = nan  # seen by the last seven tokens only
    v[:, 1, border - 3, D - 1] = nan  # by those from the eleventh on
    v[:, 2, border - 20, 0] = nan  # by all, but under a window by the first ones only, or none
    got = bi.window_attention(q, k, v, window, sink_tokens=first)
    for t in range(L):
        end = n - L + t + 1
        alone = bi.window_attention(q[:, :, t:t + 1], k[:, :, :end], v[:, :, :end], window, sink_tokens=first)
        assert torch.equal(as_int(got[:, :, t:t + 1]), as_int(alone)), t
    for h, row in enumerate((border + 4, border - 3, border - 20)):
        pos = torch.arange(n - L, n, device=cuda)
        sees = (row <= pos) & ((row > pos - window) if window else True)
        assert torch.equal(got[0, 2 * h:2 * h + 2].isfinite().all(-1), ~sees.expand(2, L))


@pytest.mark.parametrize("window", [None, 4400])
def test_a_token_is_safe_under_a_loose_bound(cuda, window):
    """256 requests of two tokens under a bound of 65536 rows, whose workgroups
    take several segments each, with NaN in the last row of some of them."""
    R, H, Hkv, D, page, W = 256, 16, 8, 64, 16, 300
    g = torch.Generator(device=cuda).manual_seed(4)
    rn = lambda *s: torch.randn(*s, generator=g, device=cuda).to(BF16)
    k, v, q = rn(Hkv, W * page, D), rn(Hkv, W * page, D), rn(2 * R, H, D)
    ends = (4601, 2101, 701, 513, 4097, 65)  # kv head h has NaN in the last row of the h-th
    for h, end in enumerate(ends):
        v[h, end - 1, h] = float("nan")
    pages = lambda x: x.view(Hkv, W, page, D).transpose(0, 1).contiguous()
    lens = [ends[r % 6] if r % 7 else 4800 - r for r in range(R)]
    table = torch.arange(W, dtype=torch.int32, device=cuda).repeat(R, 1)
    got = bi.paged_attention(q, pages(k), pages(v), table, i32(range(0, 2 * R + 1, 2), cuda), i32(lens, cuda),
                             window=window, max_query=2, max_seq=65536)
    for r in range(0, R, 5):
        for t in range(2):
            end = lens[r] - 1 + t
            alone = bi.window_attention(q[2 * r + t][None, :, None], k[None, :, :end], v[None, :, :end], window)
            assert torch.equal(as_int(got[2 * r + t]), as_int(alone[0, :, 0])), (r, t)
            for h, row in enumerate(e - 1 for e in ends):
                sees = row < end and (window is None or row > end - 1 - window)
                assert bool(got[2 * r + t, 2 * h:2 * h + 2].isfinite().all()) == (not sees), (r, t, h)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("window", [None, 1100])
def test_a_prompt_is_safe_from_its_last_row(cuda, dtype, window):
    """A prompt of the size that eight waves to a workgroup take, whose last
    token's values are infinite: only that token's result is."""
    H, Hkv, n, D = 32, 8, 2200, 128
    g = torch.Generator(device=cuda).manual_seed(1)
    rn = lambda *s: torch.randn(*s, generator=g, device=cuda).to(dtype)
    q, k, v = rn(1, H, n, D), rn(1, Hkv, n, D), rn(1, Hkv, n, D)
    clean = bi.window_attention(q, k, v, window)
    v[:, :, n - 1] = float("inf")
    got = bi.window_attention(q, k, v, window)
    assert torch.equal(as_int(got[:, :, :-1]), as_int(clean[:, :, :-1]))
    assert bool((got[:, :, -1] == float("inf")).all())


@pytest.mark.parametrize("D, V, H, Hkv, n, L, window, first, sharp", [
    (256, 256, 16, 1, 471, 471, 428, 0, 3), (256, 256, 40, 1, 700, 64, None, 0, 3),
    (192, 128, 16, 8, 393, 32, None, 0, 1), (256, 256, 24, 3, 1010, 40, 960, 4, 1)])
def test_sharp_scores_in_32_bits(cuda, D, V, H, Hkv, n, L, window, first, sharp):
    """Scores of several hundred: what a weight may be off by is set by the sum
    of the products' magnitudes, not by the score that is left of it."""
    g = torch.Generator().manual_seed(n)
    q = torch.randn(L, H, D, generator=g) * sharp
    k, v = torch.randn(n, Hkv, D, generator=g), torch.randn(n, Hkv, V, generator=g)
    heads = lambda x: x.to(cuda).transpose(0, 1)[None]
    got = bi.window_attention(heads(q), heads(k), heads(v), window, sink_tokens=first, scale=5.0)
    want, tol = ref.rows(q, k, v, n, window or 0, first, 5.0, None)
    err = (got[0].transpose(0, 1).double().cpu() - want).abs()
    assert bool((err <= tol).all()), (err / tol).max()
