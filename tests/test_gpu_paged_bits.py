"""Bits of the whole route call after call: the same inputs many times, and the
same rows in launches whose tiles begin elsewhere."""

import pytest
import torch

import mlx_batch_invariant as bi

pytestmark = pytest.mark.gpu
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def as_int(x):
    return x.contiguous().view(torch.int32 if x.dtype == F32 else torch.int16)


def difference(a, b):
    """None where the bits of two (B, H, L, D) tensors are the same, else what
    differs: how many values, over which heads, rows and dims."""
    at = (as_int(a) != as_int(b)).nonzero()
    if not at.shape[0]:
        return None
    span = lambda c: "%d..%d (%d)" % (at[:, c].min(), at[:, c].max(), at[:, c].unique().numel())
    return "%d values differ: heads %s, rows %s, dims %s; largest difference %g; first at %s" % (
        at.shape[0], span(1), span(2), span(3), (a.double() - b.double()).abs().max(),
        at[0].tolist())


@pytest.mark.parametrize("D, V", [(64, 64), (96, 96), (128, 128), (192, 128), (192, 192), (256, 256)])
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("window", [190, 1100])
def test_whole_route_repeats_its_bits(cuda, dtype, D, V, window):
    H, Hkv, n = 32, 8, 2200
    g = torch.Generator(device=cuda).manual_seed(D + V)
    rn = lambda *s: torch.randn(*s, generator=g, device=cuda).to(dtype)
    q, k, v = rn(1, H, n, D), rn(1, Hkv, n, D), rn(1, Hkv, n, V)
    run = lambda lo, hi: bi.window_attention(q[:, :, lo:hi], k[:, :, :hi], v[:, :, :hi], window,
                                             sink_tokens=3)
    base = run(0, n)
    for i in range(20 if dtype == F32 else 60):
        for lo, hi in ((0, n), (0, 1100), (1100, n), (703, 1501)):
            y = run(lo, hi)
            if not torch.equal(as_int(y), as_int(base[:, :, lo:hi])):
                # Both sides once more: which of them is the one that changed?
                pytest.fail("call %d of rows %d..%d: %s; again: %s; all rows again: %s" % (
                    i, lo, hi, difference(y, base[:, :, lo:hi]),
                    difference(run(lo, hi), base[:, :, lo:hi]), difference(run(0, n), base)))
