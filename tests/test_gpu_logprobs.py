"""bi.token_logprobs on the GPU against the definition in 64 bits."""

import math

import pytest
import torch

import mlx_batch_invariant as bi

import helpers

pytestmark = pytest.mark.gpu
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
E = 2.0 ** -24


def bits(t):
    return helpers.bits(t) if t.is_floating_point() else t.reshape(-1).cpu().numpy()


def check(got, x, tokens, top):
    """All rows of `x` finite or -inf, none of -inf alone."""
    V = x.shape[-1]
    y = x.double().reshape(-1, V)
    m = y.amax(-1, keepdim=True)
    d = y - m
    e = d.exp()
    S = e.sum(-1)
    dd = torch.where(e > 0, d, 0.0)
    U, U2 = (e * dd).sum(-1) / S, (e * dd * dd).sum(-1) / S
    ln = S.log()
    # A term's exponent rounds thrice (the difference, its product with log2 e,
    # whose constant is rounded too): 3 E |d|; exp2 is off by 2 E. The sums are
    # chains of a thread's logits (V / 1024 or 32, and as many changes of base,
    # each of them 3 E |d| more at most) and 32 partial sums.
    chain = 64 + 2 * max(32, -(-V // 1024))
    off_s = E * (6 * U.abs() + chain + 4)
    off_ln = off_s + 4 * E * ln.abs() + E
    off_u = E * (6 * U2 + (chain + 8) * U.abs()) + U.abs() * off_s
    lp = d - ln[:, None]
    t = tokens.reshape(-1).long()
    mine = lp.gather(-1, t[:, None])[:, 0]
    g = got.logprobs.double().reshape(-1)
    lead = x.shape[:-1]
    assert got.logprobs.shape == lead == got.entropy.shape
    ok = (g - mine).abs() <= off_ln + 3 * E * (mine.abs() + ln)
    assert bool((ok | (g == mine)).all())  # (-inf both)
    assert bool(((got.entropy.double().reshape(-1) - (ln - U)).abs() <= off_ln + off_u + 3 * E * (ln - U)).all())
    ids = torch.sort(y, dim=-1, descending=True, stable=True).indices[:, :top]
    assert got.top_ids.shape == (*lead, top) == got.top_logprobs.shape
    assert bool((got.top_ids.reshape(len(y), top) == ids).all())
    w = lp.gather(-1, ids)
    h = got.top_logprobs.double().reshape(len(y), top)
    assert bool((((h - w).abs() <= (off_ln + 3 * E * ln)[:, None] + 3 * E * w.abs()) | (h == w)).all())


def rows(shape, dtype, device, seed, std=2.5):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(shape, generator=g) * std).to(dtype).to(device)
    return x, torch.randint(0, shape[-1], shape[:-1], generator=g).to(device)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("shape, top", [
    ((1, 32000), 5), ((3, 32000), 20), ((70, 32000), 64), ((2, 5, 1000), 7), ((9, 1), 1), ((9, 1), 0),
    ((5, 63), 63), ((4, 64), 64), ((6, 259), 33), ((3, 8192), 20), ((3, 8193), 20), ((3, 32768), 20),
    ((3, 32769), 20), ((2, 65001), 64), ((1, 250001), 10), ((600, 999), 1),
])
def test_token_logprobs(cuda, shape, top, dtype):
    x, t = rows(shape, dtype, cuda, shape[-1] + top)
    got = bi.token_logprobs(x, t, top=top)
    check(got, x, t, top)
    # A row alone, its tokens in 32 bits: the same bits.
    flat, ft = x.reshape(-1, shape[-1]), t.reshape(-1)
    r = flat.shape[0] // 2
    one = bi.token_logprobs(flat[r], ft[r].int(), top=top)
    assert one.logprobs.shape == ()
    for a, b in zip(one, got):
        assert bool((bits(a.contiguous()) == bits(b.reshape(flat.shape[0], *a.shape)[r].contiguous())).all())


@pytest.mark.parametrize("V", [777, 32000, 70000])
@pytest.mark.parametrize("case", ["equal", "rising", "falling", "few", "zeros", "steps", "sharp", "far"])
def test_orders_and_ties(cuda, V, case):
    """Logits that are equal, or in order, where the largest lie in one thread,
    or all but a few ruled out: the ids in descending order, ties ascending."""
    x = torch.zeros(4, V)
    i = torch.arange(V)
    if case == "rising":
        x[:] = i / V * 8
    elif case == "falling":
        x[:] = -i / V * 8
    elif case == "few":
        x[:] = -math.inf
        x[:, [V - 1, 5, 6, V // 2]] = torch.tensor([1.0, 2.0, 2.0, -3.0])
        x[3] = -math.inf
        x[3, 9] = 0.5  # one token that is certain
    elif case == "zeros":
        x[:] = torch.where(i % 3 == 0, -0.0, 0.0)
    elif case == "steps":
        x[:] = (i % 7).float()
        x[1] = (i // 8 % 5 == 0).float() * 3  # whole units of the largest
        x[2] = ((i // 8 % 1024) == 17).float()  # all of them one thread's
    elif case == "sharp":
        x[:] = -30000.0
        x[:, V // 3] = 30000.0
    elif case == "far":
        x = torch.randn(4, V, generator=torch.Generator().manual_seed(1)) * 300
    x = x.to(cuda)
    t = torch.tensor([0, 5, V - 1, 9], device=cuda)
    check(bi.token_logprobs(x, t, top=40), x, t, 40)


def test_strides_and_views(cuda):
    x, t = rows((12, 3, 500), F32, cuda, 1)
    for y, tt in ((x[::2], t[::2]), (x[:, 1], t[:, 1]), (x.transpose(0, 1), t.t()),
                  (x[..., 3:402], t.clamp(max=300)), (x[0, 0].expand(4, 500), t[0, 0].expand(4)),
                  (x[..., ::2], t.clamp(max=200))):
        check(bi.token_logprobs(y, tt, top=3), y.contiguous(), tt.contiguous(), 3)
    got = bi.token_logprobs(x[:0], t[:0], top=2)
    assert [tuple(g.shape) for g in got] == [(0, 3), (0, 3), (0, 3, 2), (0, 3, 2)]


def test_alignment_changes_no_bits(cuda):
    """A vocabulary of odd length puts every row at another alignment."""
    x, t = rows((9, 5003), BF16, cuda, 2)
    got = bi.token_logprobs(x, t, top=8)
    for r in range(9):
        one = bi.token_logprobs(x[r:r + 1].clone(), t[r:r + 1], top=8)
        for a, b in zip(one, got):
            assert bool((bits(a) == bits(b[r:r + 1].contiguous())).all())


@pytest.mark.parametrize("V", [100, 32000, 40000])
def test_what_is_not_finite(cuda, V):
    x, t = rows((6, V), F32, cuda, 3)
    x[1, 7] = math.nan
    x[2, 9] = math.inf
    x[3] = -math.inf
    x[4, 8] = -math.nan
    t[5] = V  # not in the vocabulary
    got = bi.token_logprobs(x, t, top=4)
    assert got.logprobs.isnan().tolist() == [False, True, True, True, True, True]
    assert got.entropy.isnan().tolist() == [False, True, True, True, True, False]
    assert got.top_logprobs.isnan().all(1).tolist() == [False, True, True, True, True, False]
    assert got.top_ids[1, 0] == 7 and got.top_ids[2, 0] == 9 and got.top_ids[4, 0] == 8
    assert got.top_ids[3].tolist() == [0, 1, 2, 3]
    t[0] = -1
    assert bi.token_logprobs(x, t).logprobs.isnan()[0]
    # A ruled-out token is impossible; a certain one has no entropy.
    x[0] = -math.inf
    x[0, 4], t[0] = 2.0, 5
    got = bi.token_logprobs(x[:1], t[:1], top=1)
    assert got.logprobs.item() == -math.inf and got.entropy.item() == 0 and got.top_logprobs.item() == 0


def test_on_a_stream_and_in_a_graph(cuda):
    x, t = rows((20, 4000), BF16, cuda, 4)
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        bi.token_logprobs(x, t, top=6)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            got = bi.token_logprobs(x, t, top=6)
    for _ in range(3):
        x.copy_(x.roll(1, 1) * 1.25)
        want = bi.token_logprobs(x, t, top=6)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert bool((bits(a) == bits(b)).all())


def test_compiles(cuda):
    x, t = rows((20, 4000), F16, cuda, 4)
    fn = lambda x, t: tuple(bi.token_logprobs(x, t, top=6))
    got = torch.compile(fn, fullgraph=True, backend="aot_eager")(x, t)
    for a, b in zip(got, fn(x, t)):
        assert bool((bits(a) == bits(b)).all())


@pytest.mark.parametrize("rows, V", [((1 << 24) + 3, 2), ((1 << 22) + 3, 8193)])
def test_more_rows_than_one_launch_takes(cuda, rows, V):
    """Rows of 256 and of 1024 threads, 2^32 and more in all; the same row at a stride of 0."""
    g = torch.Generator().manual_seed(6)
    x = torch.randn(1, V, generator=g).to(BF16).to(cuda)
    t = torch.arange(rows, device=cuda) % V
    top = 1
    got = bi.token_logprobs(x.expand(rows, V), t, top=top)
    one = bi.token_logprobs(x.expand(V, V), t[:V], top=top)
    check(one, x.expand(V, V), t[:V], top)
    assert bool((got.logprobs.view(torch.int32) == one.logprobs[t].view(torch.int32)).all())
    assert bool((got.entropy == one.entropy[0]).all())
    assert bool((got.top_ids == one.top_ids[0]).all()) and bool((got.top_logprobs == one.top_logprobs[0]).all())
    # Rows of their own on both sides of a launch's end.
    if V == 2:
        y = torch.randn(rows, V, generator=torch.Generator(device=cuda).manual_seed(1), device=cuda).to(F16)
        got = bi.token_logprobs(y, t, top=2)
        for a in (0, (1 << 21) - 40, (1 << 22) - 3, rows - 70):
            part = slice(a, a + 70)
            for z, w in zip(got, bi.token_logprobs(y[part], t[part], top=2)):
                assert bool((z[part] == w).all())
        check(got, y, t, 2)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_time_of_rows_with_few_allowed_tokens(cuda, dtype):
    """Three allowed tokens, or equal logits: not tens of times what a row takes whose
    logits differ (3 to 4 times; 40 where every candidate was looked at alone)."""
    x = (torch.randn(3, 131072, generator=torch.Generator().manual_seed(1)) * 2.5).to(dtype).to(cuda)
    few = torch.full_like(x, -math.inf)
    few[:, [1, 70000, 131065]] = x[:, [1, 70000, 131065]]
    t = torch.ones(3, dtype=torch.long, device=cuda)

    def time(x):
        bi.token_logprobs(x, t, top=5)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            for _ in range(10):
                bi.token_logprobs(x, t, top=5)
        best = math.inf
        for _ in range(8):
            a, b = (torch.cuda.Event(enable_timing=True) for _ in range(2))
            a.record()
            graph.replay()
            b.record()
            torch.cuda.synchronize()
            best = min(best, a.elapsed_time(b))
        return best

    base = time(x)
    for y in (few, torch.zeros_like(x)):
        assert time(y) < 15 * base
