"""The choice of route, as the workspace shows it: a call that is split asks for
memory for its partial results, one that is walked whole for none. The sizes are
those where one route was measured to take 1.4 times the other's time or more
(on 256 compute units, which is what is assumed without a GPU)."""

import pytest

from mlx_batch_invariant import _lib

BF16, F32 = _lib.BF16, _lib.F32


def workspace(D, V, dtype, H, Hkv, R, L, N):
    return _lib.lib().bi_paged_attention_workspace(R * L, R, H, Hkv, D, V, 0, 0, L, N, dtype)


@pytest.mark.parametrize("D, V, dtype, H, Hkv, R, L, N", [
    # microseconds whole, split
    (128, 128, F32, 32, 8, 64, 1, 2048),    # 570, 284
    (128, 128, F32, 32, 8, 64, 1, 300),     # 103, 60
    (256, 256, F32, 32, 8, 64, 1, 2048),    # 1356, 653
    (96, 96, F32, 8, 8, 64, 1, 2048),       # 453, 224
    (256, 256, F32, 8, 8, 1, 1000, 1000),   # 331, 124
    (128, 128, F32, 32, 8, 1, 256, 4096),   # 559, 368
    (192, 192, F32, 32, 8, 1, 256, 4096),   # 1019, 573
    (192, 192, BF16, 32, 8, 1, 128, 8192),  # 437, 139
    (192, 192, BF16, 32, 8, 8, 16, 4096),   # 221, 79
    (192, 192, BF16, 8, 8, 64, 1, 2048),    # 239, 141
    (256, 256, BF16, 32, 8, 1, 256, 8192),  # 513, 344
    (192, 128, BF16, 32, 8, 1, 128, 8192),  # 260, 117
    (64, 64, BF16, 32, 8, 1, 128, 8192),    # 125, 55
    (128, 128, BF16, 32, 8, 1, 1, 8192),    # 185, 19
    (256, 256, F32, 8, 8, 1, 2048, 2048),   # 653, 392
])
def test_split_where_it_is_faster(D, V, dtype, H, Hkv, R, L, N):
    assert workspace(D, V, dtype, H, Hkv, R, L, N) > 0


@pytest.mark.parametrize("D, V, dtype, H, Hkv, R, L, N", [
    (64, 64, BF16, 32, 8, 32, 16, 1024),    # 24, 46
    (128, 128, BF16, 32, 8, 16, 32, 512),   # 22, 47
    (128, 128, BF16, 32, 8, 1, 512, 8192),  # 168, 376
    (64, 64, BF16, 8, 8, 1, 2048, 2048),    # 38, 56
    (192, 192, BF16, 32, 8, 32, 16, 1024),  # 65, 92
    (256, 256, BF16, 32, 8, 16, 32, 512),   # 44, 63
    (128, 128, F32, 32, 8, 32, 16, 1024),   # 152, 209
    (128, 128, F32, 32, 8, 2, 500, 1024),   # 157, 313
])
def test_whole_where_it_is_faster(D, V, dtype, H, Hkv, R, L, N):
    assert workspace(D, V, dtype, H, Hkv, R, L, N) in (0, _few(D, V, dtype, H, Hkv, R, L, N))


def _few(D, V, dtype, H, Hkv, R, L, N):
    """Beside chunks only single tokens and a few are split: at most 32 columns."""
    G = H // Hkv
    seg = (64 if max(D, V) * (4 if dtype == F32 else 2) <= 256 else 32) * (4 if dtype == F32 else 8)
    return R * Hkv * max(G, 32) * -(-N // seg) * (V + 2) * 4


@pytest.mark.parametrize("heads", [65536, 1 << 40, (1 << 62) + 1])
def test_head_counts_that_no_call_takes_need_no_workspace(heads):
    """The same bound as the calls': products of sizes past it passed 64 bits, and
    a division by one of them ended the process."""
    L = _lib.lib()
    assert L.bi_paged_attention_workspace(1 << 24, 1 << 24, heads, heads, 128, 128, 0, 0, 1, 4096, BF16) == 0
    assert L.bi_window_attention_workspace(1 << 24, heads, heads, 1, 4096, 128, 128, 0, 0, BF16) == 0


@pytest.mark.parametrize("R", [1 << 20, 1 << 29])
@pytest.mark.parametrize("Hkv, G", [(1, 1), (8, 4), (128, 1), (255, 257), (1, 65535), (65535, 1)])
@pytest.mark.parametrize("max_query, max_seq", [(1, 1 << 40), (64, 1 << 29), (1 << 29, 1 << 29)])
def test_largest_sizes(R, Hkv, G, max_query, max_seq):
    w = _lib.lib().bi_paged_attention_workspace(min(R * max_query, 1 << 29), R, Hkv * G, Hkv, 256, 256, 0,
                                                0, max_query, max_seq, F32)
    assert 0 <= w <= 1 << 32
