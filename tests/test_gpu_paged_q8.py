"""The 8-bit paged cache's write and read on the GPU, exactly: codes, scales and
values are what the definition says in 64 bits."""

import math

import pytest
import torch

import mlx_batch_invariant as bi

from helpers import bits

pytestmark = pytest.mark.gpu
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def codes_of(x):
    """(codes, scales) of rows (..., dim), the scale rounded once to 32 bits; NaN and
    zeros for a row with an infinity or NaN."""
    x = x.double()
    s = (x.abs().amax(-1) / 127).float()
    s = torch.where(x.isfinite().all(-1), s, math.nan)
    by = s.double()[..., None]
    c = torch.where(by > 0, (x / by).round().clamp(-127, 127), torch.zeros_like(x))
    return c.to(torch.int8), s


def same(a, b):
    """The same bits, or NaN both."""
    nan = a.isnan() & b.isnan()
    return a.dtype == b.dtype and bool((bits(a.masked_fill(nan, 0)) == bits(b.masked_fill(nan, 0))).all())


class Pool:
    """Empty int8 caches of two requests' worth of pages with distinct slots for T
    tokens; every byte of caches and scales has a known content before."""

    def __init__(self, T, Hkv, D, V, page, device, order="phtd", seed=0, spare=2):
        pages = -(-T // page) + spare
        g = torch.Generator().manual_seed(seed)
        shape = lambda d: (pages, Hkv, page, d) if order == "phtd" else (pages, page, Hkv, d)
        turn = (lambda t: t) if order == "phtd" else (lambda t: t.transpose(1, 2))
        self.k, self.v = (turn(torch.full(shape(d), 55, dtype=torch.int8, device=device)) for d in (D, V))
        sc = lambda: turn(torch.full(shape(0)[:3], 7.5, device=device))
        self.ks, self.vs = sc(), sc()
        self.slots = torch.randperm(pages * page, generator=g)[:T].to(torch.int32).to(device)
        self.page = page

    def rows(self, t, at):
        return t[(at // self.page).long(), :, (at % self.page).long()]


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("T, Hkv, D, V, page, order, pad", [
    (1, 8, 128, 128, 16, "phtd", 0),
    (3, 8, 64, 64, 8, "pthd", 2),
    (333, 4, 192, 128, 32, "phtd", 0),
    (50, 2, 96, 96, 1, "pthd", 5),
    (17, 3, 50, 7, 5, "phtd", 1),       # rows that are not of 16 bytes
    (40, 1, 256, 256, 256, "pthd", 0),
    (9, 1, 1100, 520, 16, "phtd", 0),   # several units a lane
    (2021, 8, 128, 128, 16, "pthd", 3),
])
def test_update_and_read(cuda, T, Hkv, D, V, page, order, pad, dtype):
    g = torch.Generator().manual_seed(T + D)
    kv = torch.randn(T + pad, Hkv * (D + V), generator=g) * torch.exp(torch.randn(T + pad, 1, generator=g) * 3)
    kv = kv.to(dtype).to(cuda)
    k, v = kv[:, :Hkv * D].view(-1, Hkv, D), kv[:, Hkv * D:].view(-1, Hkv, V)
    p = Pool(T, Hkv, D, V, page, cuda, order)
    slots = torch.cat([p.slots, torch.tensor([-1, 1 << 30, -7, 1 << 20, -1][:pad], dtype=torch.int32, device=cuda)])
    bi.paged_cache_update(k, v, p.k, p.v, slots, k_scales=p.ks, v_scales=p.vs)
    for cache, scale, x in ((p.k, p.ks, k[:T]), (p.v, p.vs, v[:T])):
        c, s = codes_of(x)
        assert bool((p.rows(cache, p.slots) == c).all())
        assert same(p.rows(scale, p.slots), s)
        # Nothing else was written.
        rest = torch.ones(cache.shape[0] * page, dtype=torch.bool, device=cuda)
        rest[p.slots.long()] = False
        at = rest.nonzero()[:, 0]
        assert bool((p.rows(cache, at) == 55).all() and (p.rows(scale, at) == 7.5).all())
        # A value is off by half a step at most (and the product's rounding).
        off = (x.double() - c.double() * s.double()[..., None]).abs()
        assert bool(((off <= s.double()[..., None] * (0.5 + 127 * 2.0 ** -23)) | s.isnan()[..., None]).all())
    for out in (dtype, F32):
        ko, vo = bi.paged_cache_read(p.k, p.v, slots, k_scales=p.ks, v_scales=p.vs, dtype=out)
        for got, cache, scale in ((ko, p.k, p.ks), (vo, p.v, p.vs)):
            assert got.dtype == out and got.is_contiguous() and got.shape[0] == T + pad
            w = (p.rows(cache, p.slots).float() * p.rows(scale, p.slots)[..., None]).to(out)
            assert same(got[:T], w) and not got[T:].any()
    # One token alone: the same codes.
    q = Pool(1, Hkv, D, V, page, cuda, order)
    i = T // 2
    bi.paged_cache_update(k[i:i + 1], v[i:i + 1], q.k, q.v, q.slots, k_scales=q.ks, v_scales=q.vs)
    assert bool((q.rows(q.k, q.slots) == p.rows(p.k, p.slots[i:i + 1])).all())
    assert same(q.rows(q.vs, q.slots), p.rows(p.vs, p.slots[i:i + 1]))


def test_ties_zeros_and_tiny_rows(cuda):
    """Exact halves go to the even code, for any scale; zeros, the smallest
    numbers and the largest."""
    rows = [torch.arange(-127, 129).float()[:256] / 2 for _ in range(3)]
    rows[0][-1] = 127.0          # scale 1: halves are ties
    rows[1] = rows[0] * 2.0 ** -130
    rows[2] = rows[0] * 3.0 * 2.0 ** 20  # scale 3 * 2^20
    rows.append(torch.zeros(256))
    rows.append(torch.full((256,), 2.0 ** -149))           # its scale rounds to 0
    rows.append(torch.arange(256).float() * 2.0 ** -149)   # a scale of few bits
    rows.append(torch.linspace(-1, 1, 256) * 3.4028234e38)
    g = torch.Generator().manual_seed(0)
    # Values next to a tie on either side, for scales of any bits.
    for _ in range(40):
        top = torch.rand((), generator=g) + 0.5
        s = (top.double() / 127).float().double()
        n = torch.randint(-126, 126, (256,), generator=g).double() + 0.5
        x = (n * s).float()
        x = torch.nextafter(x, torch.where(torch.rand(256, generator=g) < 0.5, math.inf, -math.inf).float()) \
            if torch.rand((), generator=g) < 0.7 else x
        x[0] = top
        rows.append(x)
    x = torch.stack(rows)[:, None].to(cuda)
    p = Pool(len(rows), 1, 256, 256, 16, cuda)
    bi.paged_cache_update(x, -x, p.k, p.v, p.slots, k_scales=p.ks, v_scales=p.vs)
    c, s = codes_of(x)
    assert bool((p.rows(p.k, p.slots) == c).all()) and bool((p.rows(p.v, p.slots) == -c).all())
    assert bool((p.rows(p.ks, p.slots) == s).all()) and bool((p.rows(p.vs, p.slots) == s).all())


def test_rows_that_are_not_finite(cuda):
    x = torch.ones(5, 2, 64, device=cuda, dtype=BF16)
    x[1, 0, 3], x[2, 1, 63], x[3, 0, 0] = math.nan, math.inf, -math.inf
    p = Pool(5, 2, 64, 64, 16, cuda)
    bi.paged_cache_update(x, x, p.k, p.v, p.slots, k_scales=p.ks, v_scales=p.vs)
    k, v = bi.paged_cache_read(p.k, p.v, p.slots, k_scales=p.ks, v_scales=p.vs, dtype=BF16)
    odd = ~x.isfinite().all(-1)
    for y in (k, v):
        assert bool((y.isnan().all(-1) == odd).all()) and bool((y[~odd] == 1).all())


@pytest.mark.parametrize("per", ["row", "page", "head", "all"])
def test_given_scales(cuda, per):
    T, Hkv, D, page = 60, 4, 96, 8
    g = torch.Generator().manual_seed(2)
    x = torch.randn(T, Hkv, D, generator=g).to(F16).to(cuda)
    p = Pool(T, Hkv, D, D, page, cuda)
    pages = p.k.shape[0]
    scale = torch.rand(pages, Hkv, page, generator=g).to(cuda) * 0.02 + 0.004
    if per == "page":
        scale = scale[:, :, :1].expand(pages, Hkv, page)
    elif per == "head":
        scale = scale[:1, :, :1].expand(pages, Hkv, page)
    elif per == "all":
        scale = scale[:1, :1, :1].expand(pages, Hkv, page)
    else:
        scale[0] = 0.0
    before = scale.clone()
    x[0, 0, 0], x[1, 1, 1], x[2, 2, 2] = math.nan, math.inf, -math.inf
    bi.paged_cache_update(x, x, p.k, p.v, p.slots, k_scales=scale, v_scales=scale, keep_scales=True)
    assert bool((scale == before).all())
    s = p.rows(scale, p.slots)[..., None].double()
    c = torch.where(s > 0, (x.double().nan_to_num(nan=0.0, posinf=1e6, neginf=-1e6) / s).round().clamp(-127, 127), 0.0)
    assert bool((p.rows(p.k, p.slots) == c.to(torch.int8)).all())
    k, v = bi.paged_cache_read(p.k, p.v, p.slots, k_scales=scale, v_scales=scale)
    assert k.dtype == F32 and bool((k == (c.float() * s.float())).all()) and bool((v == k).all())
    if per != "row":
        with pytest.raises(ValueError, match="expanded"):
            bi.paged_cache_update(x, x, p.k, p.v, p.slots, k_scales=scale, v_scales=scale)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("D, V", [(128, 128), (50, 7)])
def test_read_of_caches_in_the_activations_type(cuda, D, V, dtype):
    """The other caches are copied bit by bit; a slot may stand there twice."""
    g = torch.Generator().manual_seed(D)
    kc = torch.randn(6, 3, 8, D, generator=g).to(dtype).to(cuda)
    vc = torch.randn(6, 8, 3, V, generator=g).to(dtype).to(cuda).transpose(1, 2)
    slots = torch.tensor([47, 0, 0, -1, 48, 13, 1 << 30], dtype=torch.int32, device=cuda)
    k, v = bi.paged_cache_read(kc, vc, slots)
    at = slots.clamp(0, 47).long()
    ok = ((slots >= 0) & (slots < 48))[:, None, None]
    for got, c in ((k, kc), (v, vc)):
        w = torch.where(ok, c[at // 8, :, at % 8], torch.zeros((), dtype=dtype, device=cuda))
        assert got.dtype == dtype and bool((bits(got) == bits(w.contiguous())).all())


def test_far_rows(cuda):
    """Codes past 2^31 bytes and scales past 2^31 elements from the cache's start."""
    page, Hkv, D = 16, 1, 64
    pages = (1 << 27) // page - 1
    kc = torch.empty(pages, Hkv, page, D, dtype=torch.int8, device=cuda)  # 8 GB
    wide = torch.empty(pages, Hkv, page, 17, device=cuda)  # 9 GB: scales at strides of 17
    ks = wide[..., 3]
    last = pages * page - 1
    slots = torch.tensor([last, 0, (1 << 31) // D + 5], dtype=torch.int32, device=cuda)
    x = torch.randn(3, 1, D, generator=torch.Generator().manual_seed(1)).to(BF16).to(cuda)
    other = torch.empty(pages, Hkv, page, 32, dtype=torch.int8, device=cuda)
    ovs = torch.empty(pages, Hkv, page, device=cuda)
    bi.paged_cache_update(x, x[..., :32], kc, other, slots, k_scales=ks, v_scales=ovs)
    c, s = codes_of(x)
    at = slots.long()
    assert bool((kc[at // page, :, at % page] == c).all()) and bool((ks[at // page, :, at % page] == s).all())
    k, _ = bi.paged_cache_read(kc, other, slots, k_scales=ks, v_scales=ovs)
    assert bool((k == c.float() * s[..., None]).all())


def test_on_a_stream_and_in_a_graph(cuda):
    g = torch.Generator().manual_seed(9)
    x = torch.randn(40, 2, 128, generator=g).to(BF16).to(cuda)
    p, q = Pool(40, 2, 128, 128, 16, cuda), Pool(40, 2, 128, 128, 16, cuda)
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        bi.paged_cache_update(x, x, p.k, p.v, p.slots, k_scales=p.ks, v_scales=p.vs)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            bi.paged_cache_update(x, x, p.k, p.v, p.slots, k_scales=p.ks, v_scales=p.vs)
            k, v = bi.paged_cache_read(p.k, p.v, p.slots, k_scales=p.ks, v_scales=p.vs, dtype=BF16)
    for _ in range(3):
        x.mul_(-1.5)
        bi.paged_cache_update(x, x, q.k, q.v, q.slots, k_scales=q.ks, v_scales=q.vs)
        wk, wv = bi.paged_cache_read(q.k, q.v, q.slots, k_scales=q.ks, v_scales=q.vs, dtype=BF16)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert bool((bits(k) == bits(wk)).all() and (bits(v) == bits(wv)).all())
        assert bool((p.k == q.k).all() and (p.vs == q.vs).all())


@pytest.mark.parametrize("keep", [False, True])
def test_compiles(cuda, keep):
    g = torch.Generator().manual_seed(9)
    x = torch.randn(40, 2, 64, generator=g).to(cuda)
    p, q = Pool(40, 2, 64, 64, 16, cuda), Pool(40, 2, 64, 64, 16, cuda)

    def fn(p, x):
        bi.paged_cache_update(x, x, p.k, p.v, p.slots, k_scales=p.ks, v_scales=p.vs, keep_scales=keep)
        return bi.paged_cache_read(p.k, p.v, p.slots, k_scales=p.ks, v_scales=p.vs, dtype=F16)

    a = torch.compile(fn, fullgraph=True, backend="aot_eager")(p, x)
    b = fn(q, x)
    assert bool((bits(a[0]) == bits(b[0])).all() and (bits(a[1]) == bits(b[1])).all())
    assert bool((p.k == q.k).all() and (p.vs == q.vs).all())


def test_nothing_to_do(cuda):
    p = Pool(4, 2, 64, 64, 16, cuda)
    none = torch.empty(0, dtype=torch.int32, device=cuda)
    x = torch.empty(0, 2, 64, device=cuda)
    bi.paged_cache_update(x, x, p.k, p.v, none, k_scales=p.ks, v_scales=p.vs)
    k, v = bi.paged_cache_read(p.k, p.v, none, k_scales=p.ks, v_scales=p.vs)
    assert k.shape == (0, 2, 64) and bool((p.k == 55).all())
    empty = p.k[:0], p.v[:0]
    k, v = bi.paged_cache_read(*empty, p.slots, k_scales=p.ks[:0], v_scales=p.vs[:0])
    assert k.shape == (4, 2, 64) and not k.any() and not v.any()


def test_strides_past_4_gib(cuda):
    """Pages, rows of scales and tokens that lie 5 GiB apart."""
    far = 5 << 30
    pool = torch.zeros(far + (1 << 20), dtype=torch.int8, device=cuda)
    k, v = (pool[at:].as_strided((2, 2, 4, 32), (far, 128, 32, 1)) for at in (0, 4096))
    scales = torch.zeros((far >> 2) + (1 << 16), device=cuda)
    ks, vs = (scales[at:].as_strided((2, 2, 4), (far >> 2, 4, 1)) for at in (0, 4096))
    x = torch.randn(5, 2, 32, generator=torch.Generator().manual_seed(1)).to(BF16).to(cuda)
    tokens = torch.zeros((far >> 1) + (1 << 16), dtype=BF16, device=cuda).as_strided((2, 2, 32), (far >> 1, 32, 1))
    tokens.copy_(x[:2])
    slots = torch.tensor([6, 1], dtype=torch.int32, device=cuda)
    bi.paged_cache_update(tokens, tokens, k, v, slots, k_scales=ks, v_scales=vs)
    codes, s = codes_of(x[:2].cpu())
    for c, cs in ((k, ks), (v, vs)):
        for t, (page, row) in enumerate(((1, 2), (0, 1))):
            assert same(c[page, :, row].cpu().float(), codes[t].float()) and same(cs[page, :, row].cpu(), s[t])
    for got in bi.paged_cache_read(k, v, slots, k_scales=ks, v_scales=vs):
        assert same(got.cpu(), codes.float() * s[..., None])
    with pytest.raises(NotImplementedError, match="4 GiB"):
        one = torch.tensor([0, 1], dtype=torch.int32, device=cuda)
        bi.paged_attention(torch.zeros(1, 2, 64, dtype=BF16, device=cuda),
                           pool.as_strided((2, 2, 4, 64), (far, 256, 64, 1)),
                           pool.as_strided((2, 2, 4, 64), (far, 256, 64, 1)), slots[None], one, one[1:],
                           k_scales=ks, v_scales=vs)
