"""The decoder's serving functions without a GPU: what they refuse before any
launch, and the cache's books."""

import pytest
import torch

from mlx_batch_invariant import decoder

CONFIG = decoder.DecoderConfig(hidden=64, inter=96, heads=2, kv_heads=1, head_dim=64, layers=1, vocab=50)


def cache(**kw):
    return decoder.PagedCache(CONFIG, 2, 100, page_size=16, device="cpu", **kw)


class _Model:
    """Fails if a step gets as far as the model."""

    c = CONFIG

    def embed(self, ids):
        raise AssertionError("not refused")


@pytest.mark.parametrize("ids, new", [
    (torch.zeros(0, dtype=torch.long), [0, 0]),   # a step without tokens has no last token to answer for
    (torch.zeros(3, dtype=torch.long), [1, 1]),
    (torch.zeros(1, 2, dtype=torch.long), [1, 1]),
    (torch.zeros(1, dtype=torch.long), [1, 1]),
])
def test_steps_that_do_not_fit_their_ids_are_refused(ids, new):
    c = cache()
    with pytest.raises(ValueError, match="ids"):
        decoder.serve_step(_Model(), c, ids, new)
    assert c.lens == [0, 0] and c.used == 0  # nothing was taken


def test_a_released_request_gives_its_pages_back():
    c = cache(num_pages=9)
    # As two steps of 40 and 70 tokens leave it: 3 and 5 pages from the front.
    c.tables[0, :3] = c.free[:3]
    c.tables[1, :5] = c.free[3:8]
    c.used, c.lens = 8, [40, 70]
    c.release(0)
    assert c.used == 5 and c.lens == [0, 70]
    assert c.tables[0].tolist() == [-1] * 7 and c.tables[1, :5].tolist() == [3, 4, 5, 6, 7]
    # What is free and what is held are all pages, each once.
    assert sorted(c.free[c.used:].tolist() + c.tables[1, :5].tolist()) == list(range(9))
    c.release(0)  # an empty one: nothing
    c.release(1)
    assert c.used == 0 and sorted(c.free.tolist()) == list(range(9)) and c.lens == [0, 0]
    assert bool((c.tables == -1).all())
    with pytest.raises(IndexError):
        c.release(2)
