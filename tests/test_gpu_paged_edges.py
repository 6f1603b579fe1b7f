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
