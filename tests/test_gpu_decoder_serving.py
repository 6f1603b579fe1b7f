"""Requests that come and go over one paged cache."""

import pytest
import torch

import mlx_batch_invariant as bi
from mlx_batch_invariant import decoder

from helpers import bits

pytestmark = pytest.mark.gpu


def test_a_row_and_its_pages_are_used_again(cuda):
    """A second prompt in a released row, over pages that the first one held,
    beside a request that goes on: its logits have the bits that it has alone."""
    c = decoder.DecoderConfig(hidden=256, inter=384, heads=4, kv_heads=2, head_dim=64, layers=2,
                              vocab=500)
    m = decoder.build(c, device=cuda, seed=3)
    g = torch.Generator().manual_seed(4)
    a, b, d = (torch.randint(0, c.vocab, (n,), generator=g).to(cuda) for n in (100, 150, 130))
    step = lambda cache, new, *ids: decoder.serve_step(m, cache, torch.cat(ids), new)
    with torch.no_grad(), bi.batch_invariant_mode():
        alone = decoder.PagedCache(c, 1, 200, page_size=16, device=cuda)
        want = [step(alone, [130], d)[0], step(alone, [1], a[:1])[0]]
        # 18 pages: a (7) and b (10), and no more than one left over for d (9).
        cache = decoder.PagedCache(c, 2, 200, page_size=16, num_pages=18, device=cuda)
        step(cache, [100, 150], a, b)
        with pytest.raises(RuntimeError, match="pages"):
            step(cache, [31, 0], d[:31])
        cache.release(1)
        got = [step(cache, [1, 130], a[:1], d)[1], step(cache, [1, 1], a[:1], a[:1])[1]]
    for x, y in zip(want, got):
        assert (bits(x) == bits(y)).all()
    assert cache.lens == [102, 131] and cache.used == 7 + 9
