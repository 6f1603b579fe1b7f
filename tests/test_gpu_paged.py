"""The paged cache's operators on the GPU against 64-bit restatements
(paged_ref), and the bits that may not change."""

import math

import numpy as np
import pytest
import torch

import mlx_batch_invariant as bi
from mlx_batch_invariant import _lib, _paged

import paged_ref as ref
from helpers import bits

pytestmark = pytest.mark.gpu
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def same(a, b):
    return bool((bits(a) == bits(b)).all())


# ------------------------------------------------------------------- tables


def _tables_case(R, page, W, seed, hi, new_hi):
    g = np.random.default_rng(seed)
    ctx = g.integers(0, hi + 1, R)
    new = g.integers(0, new_hi + 1, R)
    table = g.integers(0, 10 ** 6, (R, W))
    return ctx, new, table


@pytest.mark.parametrize("R, page, W, hi, new_hi, pad, lack", [
    (1, 16, 4, 0, 1, 0, 0),
    (3, 16, 8, 100, 1, 0, 0),
    (64, 16, 40, 600, 3, 5, 0),
    (7, 5, 300, 900, 600, 100, 0),      # pages of five rows, chunks past one workgroup
    (200, 256, 6, 1500, 40, 0, 20),     # the free pages run out; some rows past the table
    (2500, 8, 9, 60, 3, 33, 0),         # more requests than one pass of the scan
    (30, 1, 70, 60, 9, 0, 0),           # pages of one row
])
def test_page_tables(cuda, R, page, W, hi, new_hi, pad, lack):
    ctx, new, table = _tables_case(R, page, W, R, hi, new_hi)
    if R > 2:
        new[1], ctx[2] = 0, 0
    total = int(new.sum())
    T = total + pad
    free = np.random.default_rng(1).permutation(10 ** 6)[:200000].astype(np.int32)
    used = ref.page_tables(table, ctx, new, free, page, T)[5]
    if lack:
        free = free[:max(used - lack, 0)]
    want = ref.page_tables(table, ctx, new, free, page, T)
    i32 = lambda a: torch.tensor(np.asarray(a), dtype=torch.int32, device=cuda)
    tb = i32(table)
    for _ in range(2):  # again on its own result: the same
        got = bi.page_tables(tb, i32(ctx), i32(new), i32(free), page, T)
        assert got.block_tables is tb
        for name, w in zip(got._fields, want):
            g = getattr(got, name).cpu().numpy()
            assert (g == np.asarray(w)).all(), name


def test_page_tables_odd_calls(cuda):
    i32 = lambda a: torch.tensor(a, dtype=torch.int32, device=cuda)
    # No request; no token; every place behind the last one.
    got = bi.page_tables(i32([]).view(0, 4), i32([]), i32([]), i32([]), 16, 3)
    assert got.query_start.tolist() == [0] and got.pages_used.item() == 0
    assert got.slots.tolist() == [-1] * 3 == got.positions.tolist()
    # A negative length counts as 0; fewer places than tokens: the pages are taken all the same.
    tb = torch.full((2, 8), -7, dtype=torch.int32, device=cuda)[:, :4]
    got = bi.page_tables(tb, i32([-5, 3]), i32([5, 6]), i32([9, 8, 7, 6]), 4, 2)
    assert got.seq_lens.tolist() == [5, 9] and got.query_start.tolist() == [0, 5, 11]
    assert got.slots.tolist() == [36, 37] and got.pages_used.item() == 4
    assert tb.tolist() == [[9, 8, -7, -7], [-7, 7, 6, -7]]


def test_page_tables_long_chunk(cuda):
    """More tokens than the launch's workgroups take at once."""
    T, page = (1 << 20) + 5000, 64
    i32 = lambda a: torch.tensor(a, dtype=torch.int32, device=cuda)
    W = -(-T // page) + 2
    tb = torch.full((2, W), -1, dtype=torch.int32, device=cuda)
    got = bi.page_tables(tb, i32([0, 70]), i32([T - 9, 9]),
                         torch.arange(W, dtype=torch.int32, device=cuda).flip(0), page, T)
    want = torch.arange(T - 9, dtype=torch.int32, device=cuda)
    assert torch.equal(got.positions[:T - 9], want)
    assert torch.equal(got.slots[:T - 9], (W - 1 - want // page) * page + want % page)
    assert got.positions[T - 9:].tolist() == list(range(70, 79))
    assert got.slots[T - 9:].tolist() == [-1] * 9  # its first page was never given


# ------------------------------------------------------------------- update


@pytest.mark.parametrize("dtype, Hkv, D, V, page, order, T", [
    (BF16, 8, 128, 128, 16, "phtd", 1),
    (BF16, 8, 128, 128, 16, "pthd", 33),
    (F16, 2, 192, 128, 7, "phtd", 100),
    (F32, 3, 5, 9, 4, "pthd", 17),      # rows of no multiple of 16 bytes
    (BF16, 1, 3, 3, 8, "phtd", 9),      # rows of no multiple of 4 bytes
    (BF16, 16, 256, 256, 32, "pthd", 700),
])
def test_cache_update(cuda, dtype, Hkv, D, V, page, order, T):
    g = torch.Generator().manual_seed(T)
    pages = T // page + 4
    slots = torch.randperm(pages * page, generator=g)[:T].to(torch.int32)
    if T > 8:
        slots[3], slots[5], slots[7] = -1, pages * page, 2 ** 31 - 1
    kv = torch.randn(T, Hkv, D + V, generator=g).to(dtype)
    shape = (pages, Hkv, page) if order == "phtd" else (pages, page, Hkv)
    kc = torch.randn(*shape, D, generator=g).to(dtype)
    vc = torch.randn(*shape, V, generator=g).to(dtype)
    dev = lambda t: t.to(cuda) if order == "phtd" else t.to(cuda).transpose(1, 2)
    k_got, v_got, kv_dev = dev(kc), dev(vc), kv.to(cuda)
    bi.paged_cache_update(kv_dev[..., :D], kv_dev[..., D:], k_got, v_got, slots.to(cuda))
    if order == "pthd":
        kc, vc = kc.transpose(1, 2), vc.transpose(1, 2)
    for t, s in enumerate(slots.tolist()):
        if 0 <= s < pages * page:
            kc[s // page, :, s % page] = kv[t, :, :D]
            vc[s // page, :, s % page] = kv[t, :, D:]
    assert same(k_got.contiguous(), kc.contiguous()) and same(v_got.contiguous(), vc.contiguous())


def test_cache_update_past_32_bits(cuda):
    """Rows more than 2^32 bytes into the cache."""
    pages, page, Hkv, D = 40000, 64, 8, 128
    kc = torch.empty(pages, Hkv, page, D, dtype=BF16, device=cuda)
    vc = torch.empty(pages, Hkv, page, D, dtype=BF16, device=cuda)
    assert kc.numel() > 2 ** 31
    k = torch.randn(3, Hkv, D, device=cuda).to(BF16)
    slots = torch.tensor([5, pages * page - 1, pages * page // 2 + 3], dtype=torch.int32, device=cuda)
    bi.paged_cache_update(k, -k, kc, vc, slots)
    for t, s in enumerate(slots.tolist()):
        assert same(kc[s // page, :, s % page], k[t])
        assert same(vc[s // page, :, s % page], -k[t])


# ---------------------------------------------------------------- attention


def check(got, want, tol, what=""):
    err = (got.double().cpu() - want).abs()
    assert bool((err <= tol).all()), "%s error %g at tolerance %g" % (
        what, (err - tol).max(), tol.flatten()[(err - tol).argmax()])


def attend(c, q, new, **kw):
    return bi.paged_attention(q.to(c.kc.device), c.kc, c.vc, c.table,
                              ref.starts(new, c.kc.device), c.lens, **kw)


# Requests (length, new tokens): one token, first tokens, lengths around the
# tiles and segments of the kernels, chunks past a column tile.
MIXED = [(1, 1), (31, 1), (32, 1), (33, 2), (64, 64), (65, 1), (127, 3), (128, 1), (129, 7),
         (255, 1), (256, 5), (257, 1), (300, 300), (513, 40), (0, 0), (40, 0), (777, 1), (1030, 9)]


@pytest.mark.parametrize("D, V, H, Hkv", [(64, 64, 8, 8), (96, 96, 6, 2), (128, 128, 32, 8),
                                          (192, 128, 4, 4), (192, 192, 3, 1), (256, 256, 16, 2)])
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_paged_attention_mixed(cuda, dtype, D, V, H, Hkv):
    seq, new = zip(*MIXED)
    c = ref.Cache(seq, Hkv, D, V, 16, dtype, D + H, cuda, fill=float("nan"))
    g = torch.Generator().manual_seed(1)
    q = torch.randn(sum(new), H, D, generator=g).to(dtype)
    got = attend(c, q, new)
    t = 0
    for r, (n, L) in enumerate(MIXED):
        want, tol = ref.rows(q[t:t + L], c.k[r], c.v[r], n, 0, 0, D ** -0.5, None)
        check(got[t:t + L], want, tol, "request %d" % r)
        t += L


@pytest.mark.parametrize("window, first, scale, sink", [
    (1, 0, None, False), (100, 0, None, True), (64, 4, 0.3, False), (257, 300, None, False),
    (5000, 2, -0.1, True), (40, 65, None, True), (0, 0, None, True)])
@pytest.mark.parametrize("dtype, page, order", [(BF16, 16, "pthd"), (F16, 40, "phtd"), (F32, 3, "pthd")])
def test_paged_attention_window(cuda, dtype, page, order, window, first, scale, sink):
    cases = [(1, 1), (100, 100), (400, 33), (600, 1), (900, 4), (1300, 130)]
    seq, new = zip(*cases)
    H, Hkv, D = 8, 2, 64
    c = ref.Cache(seq, Hkv, D, D, page, dtype, 5, cuda, order=order)
    g = torch.Generator().manual_seed(2)
    q = torch.randn(sum(new), H, D, generator=g).to(dtype)
    sinks = (torch.randn(H, generator=g) * 3).to(dtype) if sink else None
    got = attend(c, q, new, window=window or None, sink_tokens=first, scale=scale,
                 sinks=None if sinks is None else sinks.to(cuda))
    t = 0
    for r, (n, L) in enumerate(cases):
        want, tol = ref.rows(q[t:t + L], c.k[r], c.v[r], n, window, first,
                             D ** -0.5 if scale is None else scale, sinks)
        check(got[t:t + L], want, tol, "request %d" % r)
        t += L


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("B, H, Hkv, L, N, D, window, first", [
    (1, 8, 8, 1, 1, 64, 1, 0), (3, 16, 8, 77, 333, 64, 100, 3), (2, 32, 8, 1, 2000, 128, 512, 4),
    (2, 6, 2, 300, 300, 96, 33, 1), (1, 4, 1, 20, 9, 128, 7, 0), (1, 2, 2, 5, 0, 64, 3, 0),
    (1, 4, 4, 520, 700, 128, None, 0)])
def test_window_attention(cuda, dtype, B, H, Hkv, L, N, D, window, first):
    g = torch.Generator().manual_seed(N)
    q = torch.randn(B, L, H, D, generator=g).to(dtype)
    k = torch.randn(B, Hkv, N, D, generator=g).to(dtype)
    v = torch.randn(B, N, Hkv, D, generator=g).to(dtype)
    got = bi.window_attention(q.to(cuda).transpose(1, 2), k.to(cuda), v.to(cuda).transpose(1, 2),
                              window, sink_tokens=first)
    assert got.shape == (B, H, L, D)
    for b in range(B):
        M = min(L, N)  # rows before the first key see nothing
        want, tol = ref.rows(q[b, L - M:], k[b].transpose(0, 1), v[b], N, window or 0, first,
                             D ** -0.5, None)
        out = got[b].transpose(0, 1)
        check(out[L - M:], want, tol, "batch %d" % b)
        assert bool((out[:L - M] == 0).all())


def test_many_heads_share_one(cuda):
    """More query heads than a column tile per key head; one token and a chunk."""
    cases = [(300, 1), (70, 3)]
    seq, new = zip(*cases)
    c = ref.Cache(seq, 1, 64, 64, 16, BF16, 3, cuda)
    q = torch.randn(4, 71, 64, generator=torch.Generator().manual_seed(4)).to(BF16)
    got = attend(c, q, new)
    t = 0
    for r, (n, L) in enumerate(cases):
        want, tol = ref.rows(q[t:t + L], c.k[r], c.v[r], n, 0, 0, 0.125, None)
        check(got[t:t + L], want, tol)
        t += L


def test_large_scores(cuda):
    """Scores far from 0 in both directions, growing and falling along the keys:
    the running base has to follow them, across segments too."""
    n, D = 1500, 64
    g = torch.Generator().manual_seed(6)
    for name, ramp in (("up", torch.linspace(-300, 300, n)), ("down", torch.linspace(300, -300, n)),
                       ("far", torch.full((n,), -5000.0))):
        q = torch.zeros(3, 2, D)
        q[..., 0] = 8.0
        k = torch.randn(n, 2, D, generator=g) * 0.1
        k[..., 0] = ramp[:, None]
        v = torch.randn(n, 2, D, generator=g)
        for dtype in (F32, BF16, F16):
            kv = [(k.to(dtype), v.to(dtype))]
            c = ref.Cache([n], 2, D, D, 16, dtype, 1, cuda, kv=kv)
            got = attend(c, q.to(dtype), [3])
            want, tol = ref.rows(q.to(dtype), *kv[0], n, 0, 0, 0.125, None)
            check(got, want, tol, name)


# --------------------------------------------------------------------- bits


@pytest.mark.parametrize("window, first", [(0, 0), (150, 5)])
@pytest.mark.parametrize("dtype, D, H, Hkv", [(BF16, 128, 32, 8), (F16, 64, 8, 8), (F32, 128, 8, 2),
                                              (BF16, 256, 4, 2), (BF16, 96, 16, 1)])
def test_bits_do_not_depend_on_the_call(cuda, dtype, D, H, Hkv, window, first):
    """A request of 700 rows whose last 300 tokens are new: as one chunk, in
    chunks, token by token, between other requests, with and without a
    workspace, over other pages, and over contiguous keys."""
    n, L = 700, 300
    g = torch.Generator().manual_seed(D)
    kv = [(torch.randn(n, Hkv, D, generator=g).to(dtype), torch.randn(n, Hkv, D, generator=g).to(dtype))]
    q = torch.randn(L, H, D, generator=g).to(dtype).to(cuda)
    kw = dict(window=window or None, sink_tokens=first)
    c = ref.Cache([n], Hkv, D, D, 16, dtype, 1, cuda, kv=kv)
    base = attend(c, q, [L], **kw)
    assert same(attend(ref.Cache([n], Hkv, D, D, 37, dtype, 2, cuda, order="pthd", kv=kv), q, [L],
                       **kw), base)
    dev = lambda t: t.to(cuda).transpose(0, 1)[None]
    w = bi.window_attention(q.transpose(0, 1)[None], dev(kv[0][0]), dev(kv[0][1]), window or None,
                            sink_tokens=first)
    assert same(w[0].transpose(0, 1).contiguous(), base)
    # In pieces: the keys behind a piece are in the cache already, unseen.
    at = 0
    for piece in (1, 2, 5, 8, 31, 33, 1, 64, 100, 55):
        c.lens.fill_(n - L + at + piece)
        y = attend(c, q[at:at + piece], [piece], **kw)
        assert same(y, base[at:at + piece]), piece
        y = attend(c, q[at:at + piece], [piece], max_query=piece, max_seq=n - L + at + piece, **kw)
        assert same(y, base[at:at + piece]), piece
        at += piece
    # Between others, which bring one token, a chunk, nothing.
    others = [(50, 1), (n, L), (900, 200), (n, 1), (5, 0), (n, 7)]
    seq, new = zip(*others)
    kvs = [kv[0] if s == n else (torch.randn(s, Hkv, D, generator=g).to(dtype),
                                 torch.randn(s, Hkv, D, generator=g).to(dtype)) for s in seq]
    m = ref.Cache(seq, Hkv, D, D, 16, dtype, 3, cuda, kv=kvs)
    qm = torch.cat([q[L - k:] if s == n else torch.randn(k, H, D, generator=g).to(dtype).to(cuda)
                    for s, k in others])
    y = attend(m, qm, new, **kw)
    t = 0
    for s, k in others:
        if s == n:
            assert same(y[t:t + k], base[L - k:]), k
        t += k


@pytest.mark.parametrize("D, V", [(64, 64), (96, 96), (128, 128), (192, 128), (192, 192), (256, 256)])
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("window", [190, 1100])
def test_bits_of_every_launch(cuda, dtype, D, V, window):
    """A prompt and, under the longer window, a walk long enough for workgroups
    of eight waves, one for two workgroups per compute unit, a chunk with
    loading waves and single tokens: the same rows, the same bits, over paged
    and contiguous keys."""
    H, Hkv, n = 32, 8, 2200
    g = torch.Generator(device=cuda).manual_seed(D + V)
    rn = lambda *s: torch.randn(*s, generator=g, device=cuda).to(dtype)
    q, k, v = rn(1, H, n, D), rn(1, Hkv, n, D), rn(1, Hkv, n, V)
    base = bi.window_attention(q, k, v, window, sink_tokens=3)
    for lo, hi in ((0, 1100), (1100, 2200), (700, 1000), (2195, 2200), (2000, 2001), (0, 1)):
        y = bi.window_attention(q[:, :, lo:hi], k[:, :, :hi], v[:, :, :hi], window, sink_tokens=3)
        assert same(y, base[:, :, lo:hi]), (lo, hi)
    page = 64
    table = torch.randperm(-(-n // page), generator=g, device=cuda).to(torch.int32)[None]
    kc, vc = rn(table.shape[1], Hkv, page, D), rn(table.shape[1], Hkv, page, V)
    i = torch.arange(n, device=cuda)
    slots = (table[0, i // page] * page + i % page).to(torch.int32)
    bi.paged_cache_update(k[0].transpose(0, 1), v[0].transpose(0, 1), kc, vc, slots)
    qt = q[0].transpose(0, 1)
    for lo, hi in ((0, 2200), (900, 2000), (1500, 1800)):
        lens = torch.tensor([hi], dtype=torch.int32, device=cuda)
        y = bi.paged_attention(qt[lo:hi], kc, vc, table, ref.starts([hi - lo], cuda), lens,
                               window=window, sink_tokens=3)
        assert same(y, base[0, :, lo:hi].transpose(0, 1).contiguous()), (lo, hi)


def test_prompt_against_64_bits(cuda):
    """Rows of a prompt of the size that takes eight waves per workgroup."""
    H, Hkv, n, D = 32, 8, 2200, 128
    g = torch.Generator().manual_seed(3)
    q = torch.randn(n, H, D, generator=g).to(BF16)
    k = torch.randn(n, Hkv, D, generator=g).to(BF16)
    v = torch.randn(n, Hkv, D, generator=g).to(BF16)
    dev = lambda t: t.to(cuda).transpose(0, 1)[None]
    got = bi.window_attention(dev(q), dev(k), dev(v), None)[0].transpose(0, 1)
    for lo, hi in ((0, 70), (1000, 1040), (2150, 2200)):
        want, tol = ref.rows(q[lo:hi], k[:hi], v[:hi], hi, 0, 0, D ** -0.5, None)
        check(got[lo:hi], want, tol, "rows %d" % lo)


def _without_workspace(monkeypatch):
    monkeypatch.setattr(_paged, "_workspace", lambda need, device: None)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_bits_without_a_workspace(cuda, dtype, monkeypatch):
    cases = [(2000, 1), (1300, 4), (90, 1), (600, 50)]
    seq, new = zip(*cases)
    c = ref.Cache(seq, 2, 128, 128, 16, dtype, 9, cuda)
    q = torch.randn(sum(new), 8, 128, generator=torch.Generator().manual_seed(1)).to(dtype)
    base = [attend(c, q, new), attend(c, q, new, window=300, sink_tokens=9)]
    k = c.k[0].to(cuda).transpose(0, 1)[None]
    v = c.v[0].to(cuda).transpose(0, 1)[None]
    qw = q[:2].to(cuda).transpose(0, 1)[None]
    wbase = bi.window_attention(qw, k, v, 700)
    _without_workspace(monkeypatch)
    assert same(attend(c, q, new), base[0])
    assert same(attend(c, q, new, window=300, sink_tokens=9), base[1])
    assert same(bi.window_attention(qw, k, v, 700), wbase)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_unseen_rows_may_hold_anything(cuda, dtype):
    """NaN and infinities in every row that no token sees: the tail of a page,
    rows before the window, pages that no request owns."""
    n, window, first = 1000, 200, 3
    for L in (1, 40):
        kv, bad = [], []
        g = torch.Generator().manual_seed(L)
        k = torch.randn(n, 2, 128, generator=g).to(dtype)
        v = torch.randn(n, 2, 128, generator=g).to(dtype)
        lo = n - L - window + 1
        kb, vb = k.clone(), v.clone()
        kb[first:lo], vb[first:lo] = float("inf"), float("nan")
        q = torch.randn(L, 8, 128, generator=g).to(dtype)
        kw = dict(window=window, sink_tokens=first)
        good = attend(ref.Cache([n], 2, 128, 128, 48, dtype, 1, cuda, kv=[(k, v)]), q, [L], **kw)
        got = attend(ref.Cache([n], 2, 128, 128, 48, dtype, 1, cuda, kv=[(kb, vb)],
                               fill=float("nan")), q, [L], **kw)
        assert same(got, good) and not bool(good.isnan().any())


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_pages_that_are_not_there(cuda, dtype):
    """Entries below 0, past the cache and past the table hide their rows."""
    n, page = 600, 16
    c = ref.Cache([n, n], 2, 64, 64, page, dtype, 4, cuda)
    q = torch.randn(41, 4, 64, generator=torch.Generator().manual_seed(2)).to(dtype)
    seen = torch.ones(n, dtype=torch.bool)
    for j, bad in ((0, -1), (1, -2 ** 31), (9, c.kc.shape[0]), (20, 2 ** 31 - 1), (37, -1)):
        c.table[0, j] = c.table[1, j] = bad
        seen[j * page:(j + 1) * page] = False
    got = attend(c, q, [40, 1])
    want, tol = ref.rows(q[:40], c.k[0], c.v[0], n, 0, 0, 0.125, None, seen)
    check(got[:40], want, tol)
    want, tol = ref.rows(q[40:], c.k[1], c.v[1], n, 0, 0, 0.125, None, seen)
    check(got[40:], want, tol)
    # A table narrower than the sequence; one of no columns, where nothing is seen.
    seen[10 * page:] = False
    y = bi.paged_attention(q.to(cuda), c.kc, c.vc, c.table[:, :10], ref.starts([40, 1], cuda),
                           c.lens, max_seq=n)
    want, tol = ref.rows(q[:40], c.k[0], c.v[0], n, 0, 0, 0.125, None, seen)
    check(y[:40], want, tol)
    y = bi.paged_attention(q.to(cuda), c.kc, c.vc, c.table[:, :0], ref.starts([40, 1], cuda),
                           c.lens, max_seq=n)
    assert bool((y == 0).all())


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_tokens_without_a_request_and_bounds(cuda, dtype):
    """Padding tokens are 0, a token before every key is 0, a request beyond a
    bound is NaN, and none of them touches another."""
    c = ref.Cache([100, 3, 500], 2, 64, 64, 16, dtype, 4, cuda)
    q = torch.randn(60, 4, 64, generator=torch.Generator().manual_seed(2)).to(dtype).to(cuda)
    c.lens[1] = 2  # four tokens at rows -2 .. 1
    start = torch.tensor([3, 4, 8, 48], dtype=torch.int32, device=cuda)
    run = lambda **kw: bi.paged_attention(q, c.kc, c.vc, c.table, start, c.lens, **kw)
    y = run()
    assert bool((y[:3] == 0).all()) and bool((y[48:] == 0).all()) and bool((y[4:6] == 0).all())
    want, tol = ref.rows(q[6:8].cpu(), c.k[1][:2], c.v[1][:2], 2, 0, 0, 0.125, None)
    check(y[6:8], want, tol)
    z = run(max_query=40, max_seq=500)
    assert same(z, y)
    z = run(max_query=39)
    assert bool(z[8:48].isnan().all()) and same(z[:8], y[:8]) and same(z[48:], y[48:])
    z = run(max_query=1, max_seq=500)
    assert bool(z[4:48].isnan().all()) and same(z[:4], y[:4])
    z = run(max_seq=499)
    assert bool(z[8:48].isnan().all()) and same(z[:8], y[:8])
    z = run(max_query=0, max_seq=0)
    assert bool(z[3:48].isnan().all()) and bool((z[:3] == 0).all()) and bool((z[48:] == 0).all())
    none = torch.zeros(0, dtype=torch.int32, device=cuda)
    z = bi.paged_attention(q, c.kc, c.vc, none.view(0, 4), torch.zeros(1, dtype=torch.int32,
                                                                       device=cuda), none)
    assert bool((z == 0).all())


def test_offsets_past_32_bits(cuda):
    """Pages more than 2^32 bytes into the cache, and a long table."""
    pages, page, Hkv, D, n = 40000, 64, 8, 128, 5000
    kc = torch.empty(pages, Hkv, page, D, dtype=BF16, device=cuda)
    vc = torch.empty(pages, Hkv, page, D, dtype=BF16, device=cuda)
    g = torch.Generator().manual_seed(8)
    k = torch.randn(n, Hkv, D, generator=g).to(BF16)
    v = torch.randn(n, Hkv, D, generator=g).to(BF16)
    need = -(-n // page)
    table = (pages - 1 - torch.arange(need, dtype=torch.int32) * 500)[None].to(cuda)
    i = torch.arange(n, device=cuda)
    slots = (table[0, i // page] * page + i % page).to(torch.int32)
    bi.paged_cache_update(k.to(cuda), v.to(cuda), kc, vc, slots)
    q = torch.randn(34, 32, D, generator=g).to(BF16)
    lens = torch.tensor([n], dtype=torch.int32, device=cuda)
    for L in (1, 34):
        got = bi.paged_attention(q[:L].to(cuda), kc, vc, table, ref.starts([L], cuda), lens)
        want, tol = ref.rows(q[:L], k, v, n, 0, 0, D ** -0.5, None)
        check(got, want, tol)


# ----------------------------------------------------------- used as a whole


def _serve(cuda, dtype, run_step):
    """Two requests through prompts of 37 and 70 tokens in chunks and three
    decode steps, every step padded to the same number of tokens; run_step
    makes a step's calls. Checks each step's attention."""
    H, Hkv, D, page, T = 8, 2, 64, 16, 64
    g = torch.Generator().manual_seed(3)
    steps = [(37, 20), (0, 50)] + [(1, 1)] * 3
    pool = torch.randperm(40, generator=g).to(torch.int32)
    buf = dict(table=torch.full((2, 8), -1, dtype=torch.int32, device=cuda),
               ctx=torch.zeros(2, dtype=torch.int32, device=cuda),
               new=torch.zeros(2, dtype=torch.int32, device=cuda),
               free=torch.zeros(40, dtype=torch.int32, device=cuda),
               q=torch.zeros(T, H, D, dtype=dtype, device=cuda),
               k=torch.zeros(T, Hkv, D, dtype=dtype, device=cuda),
               v=torch.zeros(T, Hkv, D, dtype=dtype, device=cuda),
               kc=torch.full((40, Hkv, page, D), float("nan"), dtype=dtype, device=cuda),
               vc=torch.full((40, Hkv, page, D), float("nan"), dtype=dtype, device=cuda))
    keys, values, at = [[], []], [[], []], 0
    ctx = [0, 0]
    for new in steps:
        buf["ctx"].copy_(torch.tensor(ctx, dtype=torch.int32))
        buf["new"].copy_(torch.tensor(new, dtype=torch.int32))
        buf["free"].copy_(torch.cat([pool[at:], torch.full((at,), -1, dtype=torch.int32)]))
        q, k, v = (torch.randn(T, h, D, generator=g).to(dtype) for h in (H, Hkv, Hkv))
        buf["q"].copy_(q), buf["k"].copy_(k), buf["v"].copy_(v)
        out, used = run_step(buf, page, T)
        torch.cuda.synchronize()
        t = 0
        for r in range(2):
            keys[r].append(k[t:t + new[r]])
            values[r].append(v[t:t + new[r]])
            ctx[r] += new[r]
            want, tol = ref.rows(q[t:t + new[r]], torch.cat(keys[r]), torch.cat(values[r]), ctx[r],
                                 0, 0, D ** -0.5, None)
            check(out[t:t + new[r]], want, tol, "request %d at %d" % (r, ctx[r]))
            t += new[r]
        assert bool((out[t:] == 0).all())
        at += int(used)
    return out.clone()


def _step(b, page, T):
    t = bi.page_tables(b["table"], b["ctx"], b["new"], b["free"], page, T)
    bi.paged_cache_update(b["k"], b["v"], b["kc"], b["vc"], t.slots)
    o = bi.paged_attention(b["q"], b["kc"], b["vc"], t.block_tables, t.query_start, t.seq_lens)
    return o, t.pages_used


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_serving_steps(cuda, dtype):
    _serve(cuda, dtype, _step)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_serving_steps_on_another_stream(cuda, dtype):
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = _serve(cuda, dtype, _step)
    torch.cuda.current_stream().wait_stream(s)
    assert same(got, _serve(cuda, dtype, _step))


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_serving_steps_captured(cuda, dtype):
    """One graph of a step, replayed with other lengths, between eager work."""
    eager = _serve(cuda, dtype, _step)
    kept = {}

    def replay(b, page, T):
        if not kept:
            table, kc, vc = b["table"].clone(), b["kc"].clone(), b["vc"].clone()
            side = torch.cuda.Stream()
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                _step(b, page, T)
            torch.cuda.current_stream().wait_stream(side)
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                kept["out"] = _step(b, page, T)
            kept["graph"] = graph
            b["table"].copy_(table), b["kc"].copy_(kc), b["vc"].copy_(vc)
        kept["graph"].replay()
        torch.cuda.synchronize()
        torch.empty(1 << 24, device=cuda).fill_(float("nan"))  # the graph's memory is its own
        return kept["out"]

    assert same(_serve(cuda, dtype, replay), eager)


def test_serving_step_compiled(cuda):
    eager = _serve(cuda, BF16, _step)
    assert same(_serve(cuda, BF16, torch.compile(_step, backend="aot_eager", fullgraph=True)), eager)


def test_last_page_of_the_cache(cuda):
    """A cache whose last row is the last byte of its memory."""
    c = ref.Cache([64], 1, 64, 64, 16, BF16, 1, cuda, spare=0)
    q = torch.randn(2, 1, 64, generator=torch.Generator().manual_seed(2)).to(BF16)
    want, tol = ref.rows(q, c.k[0], c.v[0], 64, 0, 0, 0.125, None)
    check(attend(c, q, [2]), want, tol)


def test_unaligned_operands(cuda):
    """A query that is a slice of a fused projection is read in place or copied;
    a cache whose rows are not 16-byte aligned is refused."""
    c = ref.Cache([90], 2, 64, 64, 16, BF16, 1, cuda)
    fused = torch.randn(5, 4 * 64 + 3, generator=torch.Generator().manual_seed(2)).to(BF16).to(cuda)
    q = fused[:, 3:].unflatten(1, (4, 64))
    want, tol = ref.rows(q.cpu(), c.k[0], c.v[0], 90, 0, 0, 0.125, None)
    check(attend(c, q, [5]), want, tol)
    odd = torch.zeros(c.kc.numel() + 1, dtype=BF16, device=cuda)[1:].view(c.kc.shape)
    with pytest.raises(ValueError, match="aligned"):
        bi.paged_attention(q, odd, c.vc, c.table, ref.starts([5], cuda), c.lens)


def test_workspace_too_small_is_done_without(cuda):
    """The C entry point with a workspace of fewer bytes than it asks for."""
    L = _lib.lib()
    n, H, Hkv, D, page = 900, 8, 2, 128, 16
    c = ref.Cache([n], Hkv, D, D, page, BF16, 1, cuda)
    q = torch.randn(1, H, D, generator=torch.Generator().manual_seed(2)).to(BF16).to(cuda)
    base = attend(c, q, [1])
    out = torch.empty_like(base)
    st = _lib.i64_array(q.stride()[:2] + c.kc.stride()[:3] + c.vc.stride()[:3] + (c.table.shape[1],))
    start = ref.starts([1], cuda)
    ws = torch.empty(64, dtype=torch.uint8, device=cuda)
    for wp, wb in ((None, 0), (ws.data_ptr(), 64)):
        rc = L.bi_paged_attention(q.data_ptr(), c.kc.data_ptr(), c.vc.data_ptr(), c.table.data_ptr(),
                                  start.data_ptr(), c.lens.data_ptr(), None, out.data_ptr(), 1, 1, H,
                                  Hkv, D, D, c.kc.shape[0], page, c.table.shape[1], st,
                                  1 / math.sqrt(D), 0, 0, 1, n, _lib.BF16, wp, wb,
                                  torch.cuda.current_stream().cuda_stream)
        assert rc == 0 and same(out, base)


def test_decoder_over_a_paged_cache(cuda):
    """The synthetic decoder served over a paged cache: a request's logits have
    the same bits alone, in a batch of other lengths and with its prompt in
    chunks, and they are those of the contiguous model within the rounding of
    its activations."""
    from mlx_batch_invariant import decoder

    c = decoder.DecoderConfig(hidden=512, inter=768, heads=8, kv_heads=2, head_dim=64, layers=2,
                              vocab=1000)
    m = decoder.build(c, device=cuda, seed=1)
    g = torch.Generator().manual_seed(0)
    prompts = [torch.randint(0, c.vocab, (n,), generator=g) for n in (77, 5, 300, 1)]
    with bi.batch_invariant_mode():
        alone, both, cut = [], [], []
        ids = decoder.generate(m, prompts[2:3], 6, logits=alone)
        ids_b = decoder.generate(m, prompts, 6, logits=both)
        ids_c = decoder.generate(m, prompts, 6, chunk=64, page_size=16, logits=cut)
        with torch.no_grad():
            full = m(prompts[2][None].to(cuda))
    assert torch.equal(ids[0], ids_b[2]) and torch.equal(ids_b, ids_c)
    for a, b, x in zip(alone, both, cut):
        assert same(a[0], b[2]) and same(b, x)
    # Two layers of bf16 activations, each rounded to 2^-8 some ten times.
    err = (alone[0].double() - full.double()).abs().max() / full.double().abs().max()
    assert float(err) < 2 * 10 * 2.0 ** -8


def test_bits_where_the_base_just_moves(cuda):
    """A score just over the base's limit whose 2^x rounds to the limit itself,
    alone in its step: the chunk's kernel has to see it as the single token's
    does. (What shows it: f16 weights of 2^-18.5 under the one base, 0 under the
    other, on values of 30000.)"""
    n = 2000
    k = torch.zeros(1, 1, n, 64, dtype=F16, device=cuda)
    v = torch.zeros_like(k)
    k[..., 65:128, 0] = -30.0
    k[..., 64, 0], k[..., 64, 1] = 6.0, 0.0003
    k[..., 128:512, 0] = -18.5
    v[..., 128:512, :] = 30000.0
    q = torch.zeros(1, 1, n, 64, dtype=F16, device=cuda)
    q[..., :2] = 1.0
    chunk = bi.window_attention(q, k, v, None, scale=math.log(2.0))
    one = bi.window_attention(q[:, :, -1:], k, v, None, scale=math.log(2.0))
    assert same(chunk[:, :, -1:], one)


@pytest.mark.parametrize("G", [1, 3, 4, 40])
def test_few_tokens_beside_a_chunk(cuda, G):
    """Requests of one token and of a few beside a chunk: each has the bits that
    it has alone."""
    D, page, Hkv = 64, 16, 2
    g = torch.Generator(device=cuda).manual_seed(G)
    lens, news = [900, 1300, 5, 700, 2100], [1, 5, 5, 8, 1100 if G < 40 else 40]
    W = -(-max(lens) // page)
    table = torch.randperm(W * len(lens), generator=g, device=cuda).to(torch.int32).view(len(lens), W)
    kc = torch.randn(W * len(lens), Hkv, page, D, generator=g, device=cuda).to(BF16)
    vc = torch.randn(W * len(lens), Hkv, page, D, generator=g, device=cuda).to(BF16)
    q = torch.randn(sum(news), Hkv * G, D, generator=g, device=cuda).to(BF16)
    start = [0]
    for n in news:
        start.append(start[-1] + n)
    i32 = lambda a: torch.tensor(a, dtype=torch.int32, device=cuda)
    both = bi.paged_attention(q, kc, vc, table, i32(start), i32(lens), max_query=max(news),
                              max_seq=max(lens))
    for r, n in enumerate(news):
        a, b = start[r], start[r + 1]
        one = bi.paged_attention(q[a:b], kc, vc, table[r:r + 1], i32([0, n]), i32([lens[r]]))
        assert same(both[a:b], one), r


@pytest.mark.parametrize("window", [None, 40000])
def test_many_segments_of_many_requests(cuda, window):
    """More segments than the launch has places for: a workgroup takes several.
    The bits are those of the long request alone, which has a place for each."""
    D, page, Hkv, R, n = 64, 256, 2, 60, 60000
    g = torch.Generator(device=cuda).manual_seed(3)
    W = -(-n // page)
    table = torch.full((R, W), -1, dtype=torch.int32, device=cuda)
    table[17] = torch.randperm(W, generator=g, device=cuda).to(torch.int32)
    table[:17, 0] = table[18:, 0] = 5
    kc = torch.randn(W, Hkv, page, D, generator=g, device=cuda).to(BF16)
    vc = torch.randn(W, Hkv, page, D, generator=g, device=cuda).to(BF16)
    q = torch.randn(R, 2 * Hkv, D, generator=g, device=cuda).to(BF16)
    lens = torch.randint(0, 200, (R,), generator=g, device=cuda, dtype=torch.int32)
    lens[17] = n
    kw = dict(window=window, sink_tokens=700)
    both = bi.paged_attention(q, kc, vc, table, ref.starts([1] * R, cuda), lens, max_query=1, **kw)
    for r in (17, 3, 59):
        one = bi.paged_attention(q[r:r + 1], kc, vc, table[r:r + 1], ref.starts([1], cuda),
                                 lens[r:r + 1].clone(), **kw)
        assert same(both[r:r + 1], one), r
