"""Attention over an 8-bit paged cache on the GPU against 64 bits, and the bits
that may not change."""

import numpy as np
import pytest
import torch

import mlx_batch_invariant as bi
from mlx_batch_invariant import _paged

from helpers import bits
from paged_ref import UNIT, starts

pytestmark = pytest.mark.gpu
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
NAN, INF = float("nan"), float("inf")
DIMS = [(64, 64), (96, 96), (128, 128), (192, 128), (192, 192), (256, 256)]


def same(a, b):
    return bool((bits(a) == bits(b)).all())


def rows(q, k, v, n, window=0, first=0, scale=None, sinks=None, seen=None):
    """Attention of the last L of n rows in float64 and its tolerance: q (L, H,
    D); k = (codes (n, Hkv, D), scales (n, Hkv)), v alike; CPU tensors. `seen`
    (n,) hides rows."""
    dtype, (L, H, D), V = q.dtype, q.shape, v[0].shape[2]
    Hkv = k[0].shape[1]
    scale = D ** -0.5 if scale is None else scale
    q = q.double()
    pos, key = torch.arange(n - L, n)[:, None], torch.arange(n)[None]
    see = key <= pos
    if window:
        see = see & ((key > pos - window) | (key < first))
    if seen is not None:
        see = see & seen[None]
    out = torch.zeros(L, H, V, dtype=torch.float64)
    tol = torch.zeros(L, H, V, dtype=torch.float64)
    if n == 0:
        return out, tol
    u, e32 = UNIT[dtype], 2.0 ** -24
    for h in range(H):
        g = h * Hkv // H
        some = see.any(0)  # a row hidden from all may hold anything
        kh = torch.where(some[:, None], k[0][:, g].double() * k[1][:, g].double()[:, None], 0.0)
        vh = torch.where(some[:, None], v[0][:, g].double() * v[1][:, g].double()[:, None], 0.0)
        s = q[:, h] @ kh.T * scale
        mag = (q[:, h].abs() @ kh.abs().T * abs(scale)).masked_fill(~see, 0).amax(1)
        s = s.masked_fill(~see, -INF)
        top = s.amax(1)
        if sinks is not None:
            top = torch.maximum(top, sinks[h].double())
        top = torch.where(torch.isinf(top), torch.zeros_like(top), top)
        e = torch.exp(s - top[:, None])
        den = e.sum(1)
        if sinks is not None:
            den = den + torch.exp(sinks[h].double() - top)
        w = torch.where(den[:, None] > 0, e / den.clamp(min=1e-300)[:, None], 0.0)
        out[:, h] = w @ vh
        # A score is off by its fp32 sum (D roundings of at most `mag`, the
        # products of codes being exact), the row's factor (the scale times log2
        # e, and that times the row's: 3) and the product and subtraction of the
        # base (3), and exp2 (2); p by that. A weight's numerator is off by that,
        # its product with the row's scale and its rounding to the type (f16: of p
        # times at most 2, below 2^-14 by 2^-25, beside codes times the scale's
        # power of two, 2^-14 at least, and against a denominator of at least
        # 2^-4); the denominator sums what was not rounded. Sums over n rows cost
        # n roundings each and a fold's few, numerator and denominator; the result
        # is rounded once.
        delta = (D + 6) * e32 * mag + 2 * e32
        part = u + 2 * delta + (2 * n + 16) * e32
        tol[:, h] = 1.01 * u * out[:, h].abs() + 1.01 * part[:, None] * (w @ vh.abs()) + 1e-30
        if dtype == F16:
            big = max(float(vh.abs().amax()), 127 * 2.0 ** -14)
            tol[:, h] += n * 2.0 ** -21 * big + 2.0 ** -25  # the result's own half step
    return out, tol


def draw(n, Hkv, D, V, seed, spread=0.5):
    """A request's keys and values: ((codes, scales), (codes, scales))."""
    g = torch.Generator().manual_seed(seed)
    side = lambda d: ((torch.randn(n, Hkv, d, generator=g) * 40).round().clamp(-127, 127).to(torch.int8),
                      torch.exp(torch.randn(n, Hkv, generator=g) * spread) / 40)
    return side(D), side(V)


class Cache:
    """Requests in an 8-bit cache with shuffled pages; what belongs to no row holds
    codes of 99 and scales of `fill`."""

    def __init__(self, kv, page, device, order="phtd", seed=0, spare=3, fill=NAN, width=None):
        self.kv, self.page = kv, page
        seq = [k[0].shape[0] for k, _ in kv]
        Hkv, D, V = kv[0][0][0].shape[1], kv[0][0][0].shape[2], kv[0][1][0].shape[2]
        g = torch.Generator().manual_seed(seed)
        need = [-(-n // page) for n in seq]
        pages = sum(need) + spare
        perm = torch.randperm(pages, generator=g).to(torch.int32)
        table = torch.full((len(seq), max(need + [1]) if width is None else width), -1, dtype=torch.int32)
        kc = torch.full((pages, page, Hkv, D), 99, dtype=torch.int8)
        vc = torch.full((pages, page, Hkv, V), 99, dtype=torch.int8)
        ks, vs = torch.full((pages, page, Hkv), fill), torch.full((pages, page, Hkv), fill)
        at = 0
        for r, n in enumerate(seq):
            table[r, :need[r]] = perm[at:at + need[r]]
            at += need[r]
            i = torch.arange(n)
            p = table[r][i // page].long()
            (kc[p, i % page], ks[p, i % page]), (vc[p, i % page], vs[p, i % page]) = kv[r]
        move = (lambda t: t.transpose(1, 2).contiguous().to(device)) if order == "phtd" else \
            (lambda t: t.to(device).transpose(1, 2))
        self.k, self.v, self.ks, self.vs = move(kc), move(vc), move(ks), move(vs)
        self.table = table.to(device)
        self.lens = torch.tensor(seq, dtype=torch.int32, device=device)

    def __call__(self, q, new, **kw):
        kw = dict(dict(k_scales=self.ks, v_scales=self.vs), **kw)
        dev = self.k.device
        return bi.paged_attention(q.to(dev), self.k, self.v, self.table, starts(new, dev), self.lens, **kw)


def check(got, want, tol, what=""):
    err = (got.double().cpu() - want).abs()
    assert bool((err <= tol).all()), "%s error %g at tolerance %g" % (
        what, (err - tol).max(), tol.flatten()[(err - tol).argmax()])


def queries(T, H, D, dtype, seed):
    return torch.randn(T, H, D, generator=torch.Generator().manual_seed(seed)).to(dtype)


# Requests (length, new tokens): one token, first tokens, lengths around the
# tiles and segments of the kernels, chunks past a column tile.
MIXED = [(1, 1), (31, 1), (33, 2), (64, 64), (65, 1), (127, 3), (128, 1), (129, 7), (255, 1), (257, 5),
         (300, 300), (513, 40), (0, 0), (40, 0), (777, 1), (1030, 9)]


@pytest.mark.parametrize("route", ["split", "whole"])
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("D, V, H, Hkv", [(64, 64, 8, 8), (96, 96, 6, 2), (128, 128, 32, 8), (192, 128, 4, 4),
                                          (192, 192, 3, 1), (256, 256, 16, 2)])
def test_mixed(cuda, D, V, H, Hkv, dtype, route, monkeypatch):
    if route == "whole":
        monkeypatch.setattr(_paged, "_workspace", lambda need, device: None)
    seq, new = zip(*MIXED)
    kv = [draw(n, Hkv, D, V, 100 + n) for n in seq]
    c = Cache(kv, 16, cuda)
    q = queries(sum(new), H, D, dtype, 1)
    got = c(q, new)
    t = 0
    for r, (n, L) in enumerate(MIXED):
        check(got[t:t + L], *rows(q[t:t + L], *kv[r], n), "request %d" % r)
        t += L


@pytest.mark.parametrize("window, first, scale, sink", [
    (1, 0, None, False), (100, 0, None, True), (64, 4, 0.3, False), (257, 300, None, False),
    (5000, 2, -0.1, True), (40, 65, None, True), (0, 0, None, True)])
@pytest.mark.parametrize("dtype, page, order", [(BF16, 16, "pthd"), (F16, 40, "phtd"), (BF16, 3, "phtd")])
def test_windows(cuda, dtype, page, order, window, first, scale, sink):
    cases = [(1, 1), (100, 100), (400, 33), (600, 1), (900, 4), (1300, 130)]
    seq, new = zip(*cases)
    H, Hkv, D = 8, 2, 64
    kv = [draw(n, Hkv, D, D, n) for n in seq]
    c = Cache(kv, page, cuda, order)
    q = queries(sum(new), H, D, dtype, 2)
    sinks = (queries(1, 1, H, dtype, 3)[0, 0] * 3) if sink else None
    got = c(q, new, window=window or None, sink_tokens=first, scale=scale,
            sinks=None if sinks is None else sinks.to(cuda))
    t = 0
    for r, (n, L) in enumerate(cases):
        check(got[t:t + L], *rows(q[t:t + L], *kv[r], n, window, first, scale, sinks), "request %d" % r)
        t += L


def test_many_heads_share_one(cuda):
    cases = [(300, 1), (70, 3)]
    seq, new = zip(*cases)
    kv = [draw(n, 1, 64, 64, n) for n in seq]
    q = queries(4, 71, 64, BF16, 4)
    got = Cache(kv, 16, cuda)(q, new)
    check(got[:1], *rows(q[:1], *kv[0], 300))
    check(got[1:], *rows(q[1:], *kv[1], 70))


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_large_scores(cuda, dtype):
    """Scores far from 0, growing and falling along the keys: the running base has
    to follow them, across segments too."""
    n, D = 1500, 64
    for name, ramp in (("up", torch.linspace(-300, 300, n)), ("down", torch.linspace(300, -300, n)),
                       ("far", torch.full((n,), -5000.0))):
        (kc, ks), v = draw(n, 2, D, D, 6)
        kc = (kc.float() * 0.05).round().to(torch.int8)
        kc[..., 0] = torch.where(ramp >= 0, 100, -100).to(torch.int8)[:, None]
        ks = (ramp.abs() / 100)[:, None].expand(n, 2).contiguous()
        q = torch.zeros(3, 2, D, dtype=dtype)
        q[..., 0] = 8.0
        got = Cache([((kc, ks), v)], 16, cuda)(q, [3])
        check(got, *rows(q, (kc, ks), v, n), name)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("L", [1, 40, 200])
def test_scales_of_any_size(cuda, dtype, L):
    """Zeros, and scales of 2^-60 to 2^60 beside each other in keys (with queries
    as small) and values."""
    n, H, Hkv, D = 700, 8, 2, 128
    (kc, ks), (vc, vs) = draw(n, Hkv, D, D, 8)
    g = torch.Generator().manual_seed(2)
    for s in (ks, vs):
        s[torch.rand(n, Hkv, generator=g) < 0.1] = 0.0
    if dtype == BF16:
        vs *= 2.0 ** torch.randint(-60, 61, (n, Hkv), generator=g).float()
    else:
        vs *= 2.0 ** torch.randint(-20, 9, (n, Hkv), generator=g).float()
    q = queries(L, H, D, dtype, 3)
    got = Cache([((kc, ks), (vc, vs))], 16, cuda)(q, [L])
    check(got, *rows(q, (kc, ks), (vc, vs), n))
    ks *= 2.0 ** 40
    got = Cache([((kc, ks), (vc, vs))], 16, cuda)(q, [L], scale=D ** -0.5 * 2.0 ** -40)
    check(got, *rows(q, (kc, ks), (vc, vs), n, scale=D ** -0.5 * 2.0 ** -40))


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("bad", [NAN, INF, -1.0])
def test_rows_reach_only_tokens_that_see_them(cuda, dtype, bad):
    """A row whose scales are NaN, infinite or (keys) negative makes NaN of the tokens
    that see it and leaves the bits of the others, on both routes."""
    n, L, H, Hkv, D = 900, 200, 8, 2, 128
    (kc, ks), (vc, vs) = draw(n, Hkv, D, D, 5)
    q = queries(L, H, D, dtype, 3)
    base = Cache([((kc, ks), (vc, vs))], 16, cuda)(q, [L])
    row = n - 77
    for side in ("k", "v"):
        if side == "v" and bad == -1.0:
            continue
        k2, v2 = ks.clone(), vs.clone()
        (k2 if side == "k" else v2)[row, 1] = bad
        c = Cache([((kc, k2), (vc, v2))], 16, cuda)
        for new in (L, 40):
            got = c(q[L - new:], [new])
            b = base[L - new:]
            hit = torch.zeros(new, H, dtype=torch.bool, device=cuda)
            hit[max(0, new - 77):, 4:] = True
            assert same(got[~hit], b[~hit])
            assert bool(got[hit].isnan().all())


@pytest.mark.parametrize("per", ["page", "head", "all"])
def test_scales_of_blocks(cuda, per):
    """One scale for a page, a head or all, as views of stride 0."""
    n, H, Hkv, D, page = 300, 8, 4, 64, 32
    (kc, _), (vc, _) = draw(n, Hkv, D, D, 3)
    c = Cache([((kc, torch.ones(n, Hkv)), (vc, torch.ones(n, Hkv)))], page, cuda)
    P = c.k.shape[0]
    g = torch.Generator().manual_seed(1)
    at = {"page": (P, Hkv, 1), "head": (1, Hkv, 1), "all": (1, 1, 1)}[per]
    sk, sv = (torch.exp(torch.randn(at, generator=g) * 0.5).to(cuda) / 40 for _ in range(2))
    sk, sv = sk.expand(P, Hkv, page), sv.expand(P, Hkv, page)
    i = torch.arange(n, device=cuda)
    p = c.table[0].long()[i // page]
    k, v = (kc, sk[p, :, i % page].cpu()), (vc, sv[p, :, i % page].cpu())
    for L in (1, 77):
        q = queries(L, H, D, BF16, L)
        check(c(q, [L], k_scales=sk, v_scales=sv), *rows(q, k, v, n))


# --------------------------------------------------------------------- bits


@pytest.mark.parametrize("window, first", [(0, 0), (150, 5)])
@pytest.mark.parametrize("dtype, D, V, H, Hkv", [(BF16, 128, 128, 32, 8), (F16, 64, 64, 8, 8),
                                                 (F16, 128, 128, 8, 2), (BF16, 256, 256, 4, 2),
                                                 (BF16, 96, 96, 16, 1), (F16, 192, 128, 8, 2),
                                                 (BF16, 192, 192, 4, 4)])
def test_bits_do_not_depend_on_the_call(cuda, dtype, D, V, H, Hkv, window, first, monkeypatch):
    """A request of 700 rows whose last 300 tokens are new: as one chunk, in
    chunks, token by token, between other requests, with and without a
    workspace, over other pages."""
    n, L = 700, 300
    kv = draw(n, Hkv, D, V, D)
    q = queries(L, H, D, dtype, 7).to(cuda)
    kw = dict(window=window or None, sink_tokens=first)
    c = Cache([kv], 16, cuda)
    base = c(q, [L], **kw)
    assert same(Cache([kv], 37, cuda, "pthd", seed=2, fill=0.5)(q, [L], **kw), base)
    # In pieces: the keys behind a piece are in the cache already, unseen.
    for ws in (True, False):
        if not ws:
            monkeypatch.setattr(_paged, "_workspace", lambda need, device: None)
            assert same(c(q, [L], **kw), base)
        at = 0
        for piece in (1, 2, 5, 8, 31, 33, 1, 64, 100, 55):
            c.lens.fill_(n - L + at + piece)
            y = c(q[at:at + piece], [piece], **kw)
            assert same(y, base[at:at + piece]), piece
            y = c(q[at:at + piece], [piece], max_query=piece, max_seq=n - L + at + piece, **kw)
            assert same(y, base[at:at + piece]), piece
            at += piece
        c.lens.fill_(n)
    monkeypatch.undo()
    # Between others, which bring one token, a chunk, nothing.
    others = [(50, 1), (n, L), (900, 200), (n, 1), (5, 0), (n, 7)]
    seq, new = zip(*others)
    m = Cache([kv if s == n else draw(s, Hkv, D, V, s) for s in seq], 16, cuda, seed=3)
    qm = torch.cat([q[L - k:] if s == n else queries(k, H, D, dtype, s).to(cuda) for s, k in others])
    y = m(qm, new, **kw)
    t = 0
    for s, k in others:
        if s == n:
            assert same(y[t:t + k], base[L - k:]), k
        t += k


@pytest.mark.parametrize("D, V", DIMS)
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("window", [None, 190, 1100])
def test_bits_of_every_launch(cuda, dtype, D, V, window):
    """A prompt, halves of it, chunks and single tokens: the same rows, the same
    bits, by every kernel."""
    H, Hkv, n, page = 32, 8, 2200, 64
    g = torch.Generator(device=cuda).manual_seed(D + V)
    q = torch.randn(n, H, D, generator=g, device=cuda).to(dtype)
    k, v = (torch.randn(n, Hkv, d, generator=g, device=cuda) for d in (D, V))
    P = -(-n // page)
    table = torch.randperm(P, generator=g, device=cuda).to(torch.int32)[None]
    kc, vc = (torch.zeros(P, Hkv, page, d, dtype=torch.int8, device=cuda) for d in (D, V))
    ks, vs = torch.zeros(P, Hkv, page, device=cuda), torch.zeros(P, Hkv, page, device=cuda)
    i = torch.arange(n, device=cuda)
    slots = (table[0, i // page] * page + i % page).to(torch.int32)
    bi.paged_cache_update(k, v, kc, vc, slots, k_scales=ks, v_scales=vs)
    run = lambda lo, hi: bi.paged_attention(
        q[lo:hi], kc, vc, table, starts([hi - lo], cuda), torch.tensor([hi], dtype=torch.int32, device=cuda),
        window=window, sink_tokens=3, k_scales=ks, v_scales=vs)
    base = run(0, n)
    for lo, hi in ((0, 1100), (1100, 2200), (700, 1000), (2100, 2200), (2195, 2200), (2000, 2001), (0, 1)):
        assert same(run(lo, hi), base[lo:hi]), (lo, hi)
    back, vback = bi.paged_cache_read(kc, vc, slots, k_scales=ks, v_scales=vs)
    side = lambda c, s, x: ((x / s.transpose(1, 2).flatten(0, 1)[slots.long()][..., None]).round().to(torch.int8).cpu(),
                            s.transpose(1, 2).flatten(0, 1)[slots.long()].cpu())
    kk, vv = side(kc, ks, back), side(vc, vs, vback)
    for lo, hi in ((0, 5), (1500, 1503), (2190, 2200)):
        check(base[lo:hi], *rows(q[lo:hi].cpu(), (kk[0][:hi], kk[1][:hi]), (vv[0][:hi], vv[1][:hi]), hi,
                                 window or 0, 3), "rows %d" % lo)


# -------------------------------------------------------------------- edges


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_pages_that_are_not_there(cuda, dtype):
    """Entries below 0, past the cache and past the table hide their rows."""
    n, page = 600, 16
    kv = [draw(n, 2, 64, 64, r) for r in (1, 2)]
    c = Cache(kv, page, cuda)
    q = queries(41, 4, 64, dtype, 2)
    seen = torch.ones(n, dtype=torch.bool)
    for j, bad in ((0, -1), (1, -2 ** 31), (9, c.k.shape[0]), (20, 2 ** 31 - 1), (37, -1)):
        c.table[:, j] = bad
        seen[j * page:(j + 1) * page] = False
    got = c(q, [40, 1])
    check(got[:40], *rows(q[:40], *kv[0], n, seen=seen))
    check(got[40:], *rows(q[40:], *kv[1], n, seen=seen))
    # A table narrower than the sequence; one of no columns, where nothing is seen.
    seen[10 * page:] = False
    c.table = c.table[:, :10]
    check(c(q, [40, 1], max_seq=n)[:40], *rows(q[:40], *kv[0], n, seen=seen))
    c.table = c.table[:, :0]
    assert bool((c(q, [40, 1], max_seq=n) == 0).all())


def test_tokens_without_a_request_and_bounds(cuda):
    """Padding tokens are 0, a token before every key is 0, a request beyond a
    bound is NaN, and none of them touches another."""
    kv = [draw(s, 2, 64, 64, s) for s in (100, 3, 500)]
    c = Cache(kv, 16, cuda)
    q = queries(60, 4, 64, BF16, 2).to(cuda)
    qs = torch.tensor([5, 15, 20, 50], dtype=torch.int32, device=cuda)
    run = lambda **kw: bi.paged_attention(q, c.k, c.v, c.table, qs, c.lens, k_scales=c.ks, v_scales=c.vs, **kw)
    y = run()
    assert bool((y[:5] == 0).all()) and bool((y[50:] == 0).all())
    assert bool((y[15:17] == 0).all())  # five tokens of a request of three rows
    check(y[5:15], *rows(q[5:15].cpu(), *kv[0], 100))
    check(y[17:20], *rows(q[17:20].cpu(), *kv[1], 3))
    check(y[20:50], *rows(q[20:50].cpu(), *kv[2], 500))
    z = run(max_query=29, max_seq=100)
    assert bool(z[20:50].isnan().all()) and same(z[:20], y[:20]) and same(z[50:], y[50:])
    none = q[:0]
    assert bi.paged_attention(none, c.k, c.v, c.table, qs * 0, c.lens, k_scales=c.ks, v_scales=c.vs).shape == (0, 4, 64)


def test_far_rows(cuda):
    """Pages past 2^31 bytes, and scales past 2^31 elements, from the cache's start."""
    page, Hkv, D, n = 64, 1, 64, 200
    pages = (1 << 31) // (page * D) + 40
    kc = torch.empty(pages, Hkv, page, D, dtype=torch.int8, device=cuda)
    vc = torch.empty(pages, Hkv, page, D, dtype=torch.int8, device=cuda)
    wide = torch.empty(pages, Hkv, page, 65, device=cuda)  # 8.7 GB
    ks, vs = wide[..., 0], wide[..., 64]
    k, v = draw(n, Hkv, D, D, 4)
    far = torch.tensor([[pages - 1, 3, pages - 7, pages - 20]], dtype=torch.int32, device=cuda)
    i = torch.arange(n, device=cuda)
    p = far[0].long()[i // page]
    for cache, scales, (code, s) in ((kc, ks, k), (vc, vs, v)):
        cache[p, :, i % page], scales[p, :, i % page] = code.to(cuda), s.to(cuda)
    for L in (1, 150):
        q = queries(L, 4, D, BF16, L)
        got = bi.paged_attention(q.to(cuda), kc, vc, far, starts([L], cuda),
                                 torch.tensor([n], dtype=torch.int32, device=cuda), k_scales=ks, v_scales=vs)
        check(got, *rows(q, k, v, n))


def test_on_two_streams_and_in_a_graph(cuda):
    """Two calls at once, each with a workspace of its own; a captured one is
    replayed with other lengths."""
    kv = [draw(1500, 2, 128, 128, 1), draw(600, 2, 128, 128, 2)]
    c = Cache(kv, 16, cuda)
    q = queries(9, 8, 128, BF16, 2).to(cuda)
    want = c(q, [1, 8])
    torch.cuda.synchronize()
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    got = []
    for _ in range(10):
        for s in (a, b):
            with torch.cuda.stream(s):
                got.append(c(q, [1, 8]))
    torch.cuda.synchronize()
    assert all(same(g, want) for g in got)
    with torch.cuda.stream(a):
        qs = starts([1, 8], cuda)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=a):
            y = bi.paged_attention(q, c.k, c.v, c.table, qs, c.lens, max_query=8, k_scales=c.ks, v_scales=c.vs)
    for lens in ([1500, 600], [3, 9], [700, 8], [1500, 600]):
        c.lens.copy_(torch.tensor(lens, dtype=torch.int32))
        w = bi.paged_attention(q, c.k, c.v, c.table, qs, c.lens, max_query=8, k_scales=c.ks, v_scales=c.vs)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert same(y, w), lens


def test_compiles(cuda):
    c = Cache([draw(300, 2, 64, 64, 1)], 16, cuda)
    q = queries(5, 4, 64, F16, 2).to(cuda)
    qs = starts([5], cuda)
    fn = lambda q: bi.paged_attention(q, c.k, c.v, c.table, qs, c.lens, window=70, k_scales=c.ks, v_scales=c.vs)
    got = torch.compile(fn, fullgraph=True, backend="aot_eager")(q)
    assert same(got, fn(q))


def laid_bytes(R, Hkv, D, V, longest):
    """Of the rows laid out for the whole route: steps of 64 rows, keys and values
    of 16 bits, two factors a row and two masks, in whole 512 bytes."""
    return R * Hkv * -(-longest // 64) * (-(-(64 * (2 * D + 2 * V) + 512 + 16) // 512) * 512)


# Beside requests of a few tokens and none one of many, with more heads sharing a kv
# head where the kernel of 256 columns is wanted; under a window too.
@pytest.mark.parametrize("D, V, H, chunk, seq, window, first", [
    (64, 64, 8, 600, 2000, 0, 0), (96, 96, 8, 600, 2000, 300, 3), (128, 128, 8, 600, 2000, 0, 0),
    (192, 128, 8, 600, 2000, 300, 3), (192, 192, 8, 600, 2000, 0, 0), (256, 256, 8, 600, 2000, 300, 3),
    (64, 64, 32, 2100, 2300, 0, 0), (96, 96, 32, 2100, 2300, 0, 0), (128, 128, 32, 2100, 2300, 0, 0)])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_rows_laid_out_give_the_same_bits(cuda, D, V, H, chunk, seq, window, first, dtype, monkeypatch):
    """With room for its rows laid out, with room for partial results only, and with
    none: the same bits, pages that are not there and rows of bad scales included."""
    Hkv, lens, new = 2, [900, seq, 0, 77], [1, chunk, 0, 70]
    kv = [draw(n, Hkv, D, V, 60 + i) for i, n in enumerate(lens)]
    kv[1][0][1][5, 1] = INF          # seen by all of the chunk without a window
    kv[1][1][1][seq - 40, 0] = NAN   # by its last tokens
    cache = Cache(kv, 13, cuda, order="phtd" if H == 8 else "pthd", width=-(-seq // 13) + 2)
    cache.table[1, 9] = -1
    cache.table[1, 60] = 1 << 30
    q = queries(sum(new), H, D, dtype, 6)
    most = []

    def limited(limit):
        def workspace(need, device):
            most.append(need)
            n = min(need, limit)
            return torch.full((n,), 0xff, dtype=torch.uint8, device=device) if n else None
        monkeypatch.setattr(_paged, "_workspace", workspace)
        return cache(q, new, window=window or None, sink_tokens=first, max_query=chunk, max_seq=seq)

    full = limited(1 << 40)
    laid = laid_bytes(4, Hkv, D, V, seq)
    assert most[0] >= laid, "not laid out"
    assert same(limited(most[0] - 1), full)
    assert same(limited(most[0] - laid), full) and same(limited(0), full)
    # Its first tokens' neighbours, and tokens that see no bad row, are numbers.
    assert bool(torch.isfinite(full[0]).all()) and bool(torch.isfinite(full[chunk + 1:]).all())
    bad = torch.isnan(full[1:chunk + 1]).any(-1)  # (token, head)
    pos = torch.arange(seq - chunk, seq)
    half = H // 2
    want = torch.zeros(chunk, H, dtype=torch.bool)
    want[:, :half] = (pos >= seq - 40)[:, None]
    want[:, half:] = ((pos < 5 + window) if window else pos >= 5)[:, None]
    if window and first > 5:
        want[:, half:] = True
    assert bool((bad.cpu() == want).all())


def test_rows_laid_out_are_accurate(cuda):
    n, L = 2000, 600
    kv = [draw(n, 2, 128, 128, 3)]
    q = queries(L, 8, 128, BF16, 4)
    got = Cache(kv, 16, cuda)(q, [L])
    want, tol = rows(q, *kv[0], n)
    check(got, want, tol)


def test_many_requests_laid_out(cuda, monkeypatch):
    """More requests than a workgroup has threads, some without tokens, some whole and
    some split, and one past the bounds."""
    R, D, Hkv = 301, 256, 1
    lens = [(37 * r) % 250 + 6 for r in range(R)]
    new = [0 if r % 7 == 3 else 1 if r % 5 == 1 else min(lens[r], 128) for r in range(R)]
    lens[300], new[300] = 260, 1
    kv = [draw(n, Hkv, D, D, r) for r, n in enumerate(lens)]
    cache = Cache(kv, 16, cuda)
    q = queries(sum(new), 8, D, BF16, 5)
    seen = []

    def workspace(need, device):
        seen.append(need)
        return torch.empty(need, dtype=torch.uint8, device=device)

    monkeypatch.setattr(_paged, "_workspace", workspace)
    a = cache(q, new, max_query=128, max_seq=256)
    assert seen[0] >= laid_bytes(R, Hkv, D, D, 256)
    monkeypatch.setattr(_paged, "_workspace", lambda need, device: None)
    assert same(a, cache(q, new, max_query=128, max_seq=256))
    assert bool(torch.isnan(a[-1]).all()) and bool(torch.isfinite(a[:-1]).all())


def test_laid_out_in_a_graph(cuda):
    """The rows are laid out anew in each replay."""
    n, L = 1500, 500
    kv = [draw(n, 2, 192, 192, 8)]
    cache = Cache(kv, 16, cuda)
    q = queries(L, 8, 192, BF16, 9).to(cuda)
    cache(q, [L])
    start = starts([L], cuda)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = bi.paged_attention(q, cache.k, cache.v, cache.table, start, cache.lens, k_scales=cache.ks,
                                 v_scales=cache.vs)
    for i in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert same(out, cache(q, [L]))
        cache.k.neg_()
        cache.vs.mul_(1.5)
        q.copy_(q.roll(1, 0))


def test_a_cache_without_pages(cuda):
    """Nothing is seen: zeros, by one token and by many."""
    empty = torch.empty(0, 2, 16, 64, dtype=torch.int8, device=cuda)
    scales = torch.empty(0, 2, 16, device=cuda)
    table = torch.full((1, 40), -1, dtype=torch.int32, device=cuda)
    lens = torch.tensor([600], dtype=torch.int32, device=cuda)
    for L in (1, 600):
        q = queries(L, 4, 64, BF16, 1).to(cuda)
        for t in (table, table.new_full((1, 40), 3)):
            out = bi.paged_attention(q, empty, empty, t, starts([L], cuda), lens, k_scales=scales, v_scales=scales)
            assert out.shape == (L, 4, 64) and bool((out == 0).all())


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_laid_out_rows_of_any_scale_sinks_and_more_tokens_than_rows(cuda, dtype, monkeypatch):
    """A chunk of more tokens than its request has rows, whose first see nothing; scales
    over many powers of two; logit sinks and a negative scale: as without a workspace."""
    kv = [draw(300, 2, 192, 128, 21, spread=6.0), draw(1400, 2, 192, 128, 22, spread=6.0)]
    new = [520, 520]
    cache = Cache(kv, 16, cuda)
    q = queries(sum(new), 8, 192, dtype, 23)
    sinks = torch.randn(8, generator=torch.Generator().manual_seed(2)).to(dtype).to(cuda)
    seen = []

    def workspace(need, device):
        seen.append(need)
        return torch.full((need,), 0xff, dtype=torch.uint8, device=device)

    for kw in (dict(), dict(sinks=sinks), dict(scale=-0.07), dict(sinks=sinks, scale=-0.07, window=200)):
        kw = dict(kw, max_query=520, max_seq=1400)
        monkeypatch.setattr(_paged, "_workspace", workspace)
        a = cache(q, new, **kw)
        assert seen[-1] >= laid_bytes(2, 2, 192, 128, 1400), kw
        monkeypatch.setattr(_paged, "_workspace", lambda need, device: None)
        assert same(a, cache(q, new, **kw)), kw
        assert bool((a[:220] == 0).all())
        # Without a sink a token's weights sum to 1, and the largest value of what it sees
        # is above bf16's smallest number. (With one they may all be below it: scores here
        # reach far below any sink. f16's smallest number is above the smallest scales.)
        if dtype == BF16 and "sinks" not in kw:
            assert bool((a[220:] != 0).any(-1).all())


@pytest.mark.parametrize("L", [1, 40])
def test_scores_as_far_as_they_go(cuda, L):
    """Of one row alone the result is its value, however large the score, or NaN."""
    D = 64
    kc = torch.zeros(L, 1, D, dtype=torch.int8)
    kc[:, :, 0] = 100
    (vc, vs) = draw(L, 1, D, D, 3)[1]
    vc = vc[:1].expand(L, 1, D).contiguous()
    vs = vs[:1].expand(L, 1).contiguous()
    value = (vc[0, 0].double() * vs[0, 0].double())
    for power, sign in ((8, 1), (20, 1), (20, -1), (27, 1), (27, -1), (31, 1), (31, -1), (60, 1)):
        ks = torch.full((L, 1), 2.0 ** (power - 3) / 100)
        q = torch.zeros(L, 4, D, dtype=BF16)
        q[..., 0] = 8.0 * sign
        got = Cache([((kc, ks), (vc, vs))], 16, cuda)(q, [L], scale=1.0)
        if power > 29:
            assert bool(torch.isnan(got).all()), (power, sign)
        else:  # (p's, the weight's and the result's rounding, and equal rows' sum)
            tol = value.abs() * (2 * UNIT[BF16] + 2.0 ** -20)
            assert bool(((got.double().cpu() - value).abs() <= tol).all()), (power, sign)


@pytest.mark.parametrize("dtype, bound", [(F16, 2.0 ** 28), (BF16, 2.0 ** 30)])
@pytest.mark.parametrize("L", [1, 40])
def test_scores_up_to_the_bound_of_their_type(cuda, dtype, bound, L):
    """Requests of equal rows, whose result is the row's value: for scales of any bits,
    whose scores round up and down, it is that below the bound (of scores times log2 e),
    and NaN past it."""
    D, R = 64, 64
    (vc, vs) = draw(1, 1, D, D, 3)[1]
    value = vc[0, 0].double() * vs[0, 0].double()
    g = torch.Generator().manual_seed(L)
    q = torch.zeros(L * R, 4, D, dtype=dtype)
    q[..., 0] = 8.0
    # p's exponent is off by half a step of the score, which the denominator shares; p
    # itself by 2 units of 32 bits, a weight by its rounding (f16: of 2^-8 at least, by
    # 2^-25 at most where it is subnormal), the result by its own; sums of L.
    tol = value.abs() * (2.05 * UNIT[dtype] + 2.0 ** -17 + 2.0 ** -20) + (2.0 ** -25 if dtype == F16 else 0.0)
    for power in range(20, 31):
        s = 2.0 ** power * (1 + torch.rand(R, generator=g))  # scores times log2 e
        keep = (s < bound * 0.999) | (s > bound * 1.001)
        for sign in (1, -1):
            kv = []
            for r in range(R):
                kc = torch.zeros(L, 1, D, dtype=torch.int8)
                kc[:, :, 0] = 100 * sign
                ks = torch.full((L, 1), float(s[r] / 800 / 1.4426950408889634))
                kv.append(((kc, ks), (vc.expand(L, 1, D).contiguous(), vs.expand(L, 1).contiguous())))
            got = Cache(kv, 16, cuda)(q, [L] * R, scale=1.0).double().cpu().view(R, L, 4, D)
            for r in range(R):
                if not keep[r]:
                    continue
                if s[r] > bound:
                    assert bool(got[r].isnan().all()), (float(s[r]), sign)
                else:
                    assert bool(((got[r] - value).abs() <= tol).all()), (float(s[r]), sign)


@pytest.mark.parametrize("L", [1, 40])
def test_scores_past_the_range_of_32_bits(cuda, L):
    """Below it a row is not seen; above it the token is NaN."""
    D = 64
    _, v = draw(L, 1, D, D, 3)
    ks = torch.full((L, 1), 2.0 ** 127 / 1.4426950408889634)
    q = torch.zeros(L, 4, D, dtype=BF16)
    q[..., 0] = 8.0
    for sign in (1, -1):
        kc = torch.zeros(L, 1, D, dtype=torch.int8)
        kc[:, :, 0] = 100 * sign
        got = Cache([((kc, ks), v)], 16, cuda)(q, [L], scale=1.0)
        assert bool((got.isnan() if sign > 0 else got == 0).all())


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("D, V", [(64, 64), (192, 128)])
def test_bits_of_far_scores(cuda, dtype, D, V, monkeypatch):
    """Scores of 2^22 to 2^28, a few steps of 32 bits apart: split, whole and whole over
    rows laid out, the same bits."""
    n, H, Hkv = 700, 8, 2
    g = torch.Generator().manual_seed(1)
    q = torch.zeros(600, H, D, dtype=dtype)
    q[..., 0] = 8.0
    q = q.to(cuda)
    for power in range(22, 28):
        for sign in (1, -1):
            c = 2.0 ** power * (1 + torch.rand(1, Hkv, generator=g)) / 800
            c = c * (1 + torch.randint(-3, 1, (n, Hkv), generator=g) * 2.0 ** -23)
            c[torch.rand(n, Hkv, generator=g) < 0.01] *= 1 + 2.0 ** -23 * sign
            kc = torch.zeros(n, Hkv, D, dtype=torch.int8)
            kc[..., 0] = 100 * sign
            cache = Cache([((kc, c / 1.4426950408889634), draw(n, Hkv, D, V, power)[1])], 16, cuda)
            base = cache(q, [600], scale=1.0)
            one = cache(q[:1], [1], scale=1.0)
            assert bool(base.isfinite().all())
            assert same(base[-1:], one), (power, sign)
            with monkeypatch.context() as m:
                m.setattr(_paged, "_workspace", lambda need, device: None)
                assert same(cache(q, [600], scale=1.0), base), (power, sign)
                assert same(cache(q[:1], [1], scale=1.0), one), (power, sign)


@pytest.mark.parametrize("D, V, seq, window, first", [(256, 256, 2200, 0, 0), (64, 64, 8192, 0, 0),
                                                      (128, 128, 8192, 2500, 3), (192, 128, 4000, 0, 0)])
@pytest.mark.parametrize("few", [20, 40])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_more_rows_than_there_is_room_for(cuda, D, V, seq, window, first, dtype, few, monkeypatch):
    """64 requests, most with more tokens than are split, one with a chunk: laid out as
    far as there is room (but for 20 tokens, one column tile), the others as without, and
    the bits of a call without any."""
    R, H, Hkv, page = 64, 16, 4, 64
    g = torch.Generator(device=cuda).manual_seed(D + window)
    width = -(-seq // page)
    codes = lambda d: torch.randint(-127, 128, (R * width, Hkv, page, d), generator=g, device=cuda, dtype=torch.int8)
    scales = lambda: torch.exp(torch.randn(R * width, Hkv, page, generator=g, device=cuda)) / 40
    kc, vc, ks, vs = codes(D), codes(V), scales() / 10, scales()
    table = torch.randperm(R * width, generator=g, device=cuda).to(torch.int32).view(R, width)
    table[3, 5] = -1
    new = [1 if r % 5 == 0 else 0 if r % 7 == 3 else 600 if r == 11 else few for r in range(R)]
    lens = [seq - 37 * (r % 9) if r % 4 else 500 + 30 * r for r in range(R)]
    lens[2] = 7  # fewer rows than tokens: some see nothing
    seqs = torch.tensor(lens, dtype=torch.int32, device=cuda)
    q = torch.randn(sum(new), H, D, generator=g, device=cuda).to(dtype)
    most = []

    def limited(limit, **kw):
        def workspace(need, device):
            most.append(need)
            n = min(need, limit)
            return torch.full((n,), 0xff, dtype=torch.uint8, device=device) if n else None
        monkeypatch.setattr(_paged, "_workspace", workspace)
        return bi.paged_attention(q, kc, vc, table, starts(new, cuda), seqs, k_scales=ks, v_scales=vs, max_query=600,
                                  max_seq=seq, window=window or None, sink_tokens=first, **kw)

    full = limited(1 << 40)
    beyond = torch.cat([torch.full((n,), lens[r] > seq) for r, n in enumerate(new)])  # (of 2200 rows one is)
    assert bool((full.isnan().cpu() == beyond[:, None, None]).all())
    laid = laid_bytes(1, 1, D, V, 64)
    nseg = -(-seq // 512)
    if window:
        nseg = min(nseg, (window + 15 // 4 + 1 + 510) // 512 + 1 + 1)  # (ends, and the first rows)
    room = most[0] - R * Hkv * 32 * nseg * (V + 2) * 4
    assert (1 << 27) - laid < room <= (1 << 27) + 512, (most[0], room)
    assert same(limited(0), full) and same(limited(most[0] - 1), full)
    # Rows beyond a bound, and a request alone in its place.
    bound = limited(1 << 40)
    assert same(bound, full)
    t = sum(new[:11])
    one = bi.paged_attention(q[t:t + 600], kc, vc, table[11:12], starts([600], cuda), seqs[11:12], k_scales=ks,
                             v_scales=vs, window=window or None, sink_tokens=first)
    assert same(one, full[t:t + 600])


def test_partial_results_without_memory_for_rows_laid_out(cuda, monkeypatch):
    """Where the workspace cannot be had, what of it single tokens need is asked for."""
    lens, new = [3000, 900, 2500, 40], [1, 1, 900, 1]
    kv = [draw(n, 2, 128, 128, 30 + i) for i, n in enumerate(lens)]
    cache = Cache(kv, 16, cuda)
    q = queries(sum(new), 8, 128, BF16, 6)
    run = lambda: cache(q, new, max_query=900, max_seq=3000)
    full, asked, real = run(), [], _paged._workspace

    def scarce(need, device):
        asked.append(need)
        return real(need, device) if len(asked) > 1 else None

    monkeypatch.setattr(_paged, "_workspace", scarce)
    assert same(run(), full)
    part = 4 * 2 * 32 * -(-3000 // 512) * 130 * 4  # 32 columns of each request
    assert asked == [part + laid_bytes(4, 2, 128, 128, 3000), part]
    asked.clear()

    def none(need, device):
        asked.append(need)

    monkeypatch.setattr(_paged, "_workspace", none)
    assert same(run(), full) and len(asked) == 2


def test_places_of_rows_in_a_graph_and_on_two_streams(cuda):
    """Requests take their places anew in each replay, as their lengths are then."""
    R, H, Hkv, D, page, seq = 64, 8, 4, 128, 64, 4096
    g = torch.Generator(device=cuda).manual_seed(2)
    width = seq // page
    kc, vc = (torch.randint(-127, 128, (R * width, Hkv, page, D), generator=g, device=cuda, dtype=torch.int8)
              for _ in range(2))
    ks, vs = (torch.rand(R * width, Hkv, page, generator=g, device=cuda) / 100 for _ in range(2))
    table = torch.randperm(R * width, generator=g, device=cuda).to(torch.int32).view(R, width)
    q = torch.randn(64 * 20 + 580, H, D, generator=g, device=cuda).to(BF16)
    qs, lens = (torch.zeros(n, dtype=torch.int32, device=cuda) for n in (R + 1, R))

    def run():
        return bi.paged_attention(q, kc, vc, table, qs, lens, max_query=600, max_seq=seq, k_scales=ks, v_scales=vs)

    def fill(new, length):
        qs.copy_(starts(new, cuda))
        lens.copy_(torch.tensor([length(r) for r in range(R)], dtype=torch.int32))

    steps = [([20] * 63 + [600], lambda r: seq), ([40] * 31 + [0] * 32 + [600], lambda r: seq), ([600] + [20] * 63, lambda r: 30 + 60 * r),
             ([1] * 63 + [600], lambda r: seq - r), ([20] * 64, lambda r: seq - 64 * r),
             ([0] * 60 + [465] * 4, lambda r: seq)]
    sizes = (q.shape[0], R, H, Hkv, D, D, 0, 0, 600, seq, 2)
    need = _paged._lib.lib().bi_paged_attention_q8_workspace(*sizes)
    least = _paged._lib.lib().bi_paged_attention_q8_least_workspace(*sizes)
    assert (1 << 27) - laid_bytes(1, 1, D, D, 64) < need - least <= (1 << 27) + 512
    fill(*steps[0])
    run()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run()
    streams = torch.cuda.Stream(), torch.cuda.Stream()
    for step in (*steps, *steps[::-1]):
        fill(*step)
        want = run()
        torch.cuda.synchronize()
        got = []
        for s in streams:
            with torch.cuda.stream(s):
                got.append(run())
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert same(out, want) and all(same(x, want) for x in got)
