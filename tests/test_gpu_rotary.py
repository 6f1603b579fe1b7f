"""bi.rotary on the GPU against the formula in 64 bits."""

import math

import pytest
import torch

import mlx_batch_invariant as bi

from helpers import bits

pytestmark = pytest.mark.gpu
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def want(x, positions, inv_freq, interleaved, offset, scale):
    """(the turned heads in float64, what the kernel may be off)."""
    n, y = inv_freq.shape[0], x.double()
    turn = positions.double()[:, None] * inv_freq
    c, s = (f(turn)[:, None] * scale for f in (torch.cos, torch.sin))
    a = torch.arange(n, device=x.device) * (2 if interleaved else 1) + offset
    b = a + (1 if interleaved else n)
    out, tol = y.clone(), torch.zeros_like(y)
    out[..., a] = y[..., a] * c - y[..., b] * s
    out[..., b] = y[..., a] * s + y[..., b] * c
    # Sine and cosine: the reduced angle is off by 2^-26 turns (9.4e-8 rad) and
    # the functions by 4 units of 2^-24; the scale's product, the two products
    # and their sum round by 2^-24 each; then the result once to the type. (The
    # far angles' own 64 bits: 2^-51 of the angle on both sides.)
    part = abs(scale) * (y[..., a].abs() + y[..., b].abs())
    near = part * (9.5e-8 + 8 * 2.0 ** -24 + (turn.abs() * 2.0 ** -50)[:, None])
    u = torch.finfo(x.dtype).eps / 2
    tiny = torch.finfo(x.dtype).smallest_normal * u
    tol[..., a] = near + u * out[..., a].abs() * 1.01 + tiny
    tol[..., b] = near + u * out[..., b].abs() * 1.01 + tiny
    return out, tol


def check(got, x, *args):
    ref, tol = want(x, *args)
    assert got.shape == x.shape and got.dtype == x.dtype and got.is_contiguous()
    assert bool(((got.double() - ref).abs() <= tol).all())


@pytest.mark.parametrize("T, H, Hkv, D, n, offset, inter, scale, far, dtype", [
    (1, 32, 8, 128, 64, 0, False, 1.0, 8192, BF16),
    (64, 32, 8, 128, 64, 0, True, 1.0, 8192, BF16),
    (3, 5, 1, 64, 32, 0, False, 1.2, 1 << 30, F16),      # far out
    (257, 8, 8, 192, 32, 128, True, 1.0, 100000, BF16),  # the last 64 of 192 dims
    (33, 4, 2, 96, 24, 24, False, 0.5, 4200, F32),       # in the middle
    (7, 3, 3, 50, 25, 0, True, 1.0, 999, F16),           # rows that are not of 16 bytes
    (7, 3, 1, 51, 11, 29, False, 1.0, 999, F32),
    (9, 2, 1, 64, 1, 63 - 1, False, 1.0, 50, BF16),      # one pair
    (9, 2, 1, 64, 0, 0, False, 1.0, 50, BF16),           # none: a copy
    (2021, 16, 8, 64, 16, 0, True, 1.0, 131072, F32),
    (11, 6, 2, 40, 16, 8, False, 1.0, 300, BF16),        # an odd number of units is copied
])
def test_rotary(cuda, T, H, Hkv, D, n, offset, inter, scale, far, dtype):
    g = torch.Generator().manual_seed(T * D)
    qkv = torch.randn(T, H + 2 * Hkv, D, generator=g).to(dtype).to(cuda)
    q, k = qkv[:, :H], qkv[:, H:H + Hkv]
    pos = torch.randint(-far, far, (T,), generator=g, dtype=torch.int32)
    pos[0] = far
    pos = pos.to(cuda)
    f = bi.rotary_frequencies(2 * n, device=cuda) if n else torch.empty(0, dtype=torch.float64, device=cuda)
    qo, ko = bi.rotary(q, k, pos, f, interleaved=inter, offset=offset, scale=scale)
    for got, x in ((qo, q), (ko, k)):
        check(got, x, pos, f, inter, offset, scale)
    # A token alone, from memory of another alignment: the same bits.
    t = T // 2
    odd = torch.empty(H * D + 1, dtype=dtype, device=cuda)[1:].view(1, H, D)
    odd.copy_(q[t:t + 1])
    one, none = bi.rotary(odd, None, pos[t:t + 1], f, interleaved=inter, offset=offset, scale=scale)
    assert none is None and bool((bits(one[0]) == bits(qo[t])).all())


def test_rotary_takes_any_strides(cuda):
    q = torch.randn(128, 6, 10, device=cuda).permute(2, 1, 0)  # last dimension not contiguous
    k = torch.randn(1, 1, 128, device=cuda).expand(10, 2, 128)
    pos = torch.arange(20, dtype=torch.int32, device=cuda)[::2]
    f = bi.rotary_frequencies(128, device=cuda)
    qo, ko = bi.rotary(q, k, pos, f)
    check(qo, q, pos, f, False, 0, 1.0)
    check(ko, k, pos, f, False, 0, 1.0)


def test_turning_back_and_relative_positions(cuda):
    """A turn by -p undoes one by p, and a product of a query and a key depends
    on the distance of their positions."""
    g = torch.Generator().manual_seed(5)
    q, k = (torch.randn(50, 4, 128, generator=g).to(cuda) for _ in range(2))
    pos = torch.randint(0, 1 << 20, (50,), generator=g, dtype=torch.int32).to(cuda)
    f = bi.rotary_frequencies(128, method="parts", factor=4.0, original=2048, device=cuda)
    a, b = bi.rotary(q, k, pos, f)
    # Twice the turn's own error, (9.5e-8 + 8 * 2^-24) of each of two values.
    back, _ = bi.rotary(a, None, -pos, f)
    assert (back - q).abs().max() < 4 * 5.8e-7 * q.abs().max()
    c, d = bi.rotary(q, k, pos + 1000, f)
    s, t = ((x.double() * y.double()).sum(-1) for x, y in ((a, b), (c, d)))
    mag = (q.double().abs() * k.double().abs()).sum(-1).max() * 2
    assert (s - t).abs().max() < 8 * 5.8e-7 * mag


def test_rotary_empty_and_infinite(cuda):
    f = bi.rotary_frequencies(64, device=cuda)
    q = torch.randn(0, 4, 64, device=cuda, dtype=BF16)
    pos = torch.empty(0, dtype=torch.int32, device=cuda)
    a, b = bi.rotary(q, q[:, :1], pos, f)
    assert a.shape == (0, 4, 64) and b.shape == (0, 1, 64)
    # An infinity spoils its own pair only.
    x = torch.ones(2, 2, 64, device=cuda)
    x[0, 1, 5] = math.inf
    got, _ = bi.rotary(x, None, torch.tensor([3, 4], dtype=torch.int32, device=cuda), f)
    odd = ~got.isfinite()
    assert odd[0, 1, [5, 37]].all() and int(odd.sum()) == 2


def test_rotary_on_a_stream_and_in_a_graph(cuda):
    g = torch.Generator().manual_seed(9)
    q, k = (torch.randn(40, h, 128, generator=g).to(BF16).to(cuda) for h in (8, 2))
    pos = torch.arange(40, dtype=torch.int32, device=cuda)
    f = bi.rotary_frequencies(128, device=cuda)
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        bi.rotary(q, k, pos, f)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            a, b = bi.rotary(q, k, pos, f)
    for step in range(3):
        pos.add_(1000)
        q.mul_(-1)
        want_a, want_b = bi.rotary(q, k, pos, f)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert bool((bits(a) == bits(want_a)).all() and (bits(b) == bits(want_b)).all())


@pytest.mark.parametrize("with_k", [True, False])
def test_rotary_compiles(cuda, with_k):
    g = torch.Generator().manual_seed(3)
    q, k = (torch.randn(9, h, 64, generator=g).to(cuda) for h in (4, 2))
    pos = torch.arange(9, dtype=torch.int32, device=cuda)
    f = bi.rotary_frequencies(64, device=cuda)

    def fn(q, k):
        a, b = bi.rotary(q, k, pos, f, interleaved=True)
        return a if b is None else torch.cat([a, b], 1)

    k = k if with_k else None
    got = torch.compile(fn, fullgraph=True, backend="aot_eager")(q, k)
    assert bool((bits(got) == bits(fn(q, k))).all())
