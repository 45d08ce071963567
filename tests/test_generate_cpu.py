"""generate's page book-keeping, on the CPU."""

from __future__ import annotations

import pytest
import torch


@pytest.mark.parametrize("page_size", [0, -8, 12])
def test_page_sizes_that_are_refused(page_size):
    from switchyard.generate import PagedCache

    with pytest.raises(ValueError, match="page_size"):
        PagedCache(2, 2, 64, 3, 20, 5, torch.bfloat16, "cpu", page_size)


def test_pages_and_slots():
    from switchyard.generate import PagedCache

    cache = PagedCache(1, 1, 8, 2, 20, 9, torch.bfloat16, "cpu", 8)
    assert cache.kv.shape == (1, 2, 3 + 2 * 2, 1, 8, 8)
    assert cache.prefix_pages.tolist() == [0, 1, 2] and cache.table.tolist() == [[3, 4], [5, 6]]
    cache.lens += 7
    assert cache.own_slots(2).tolist() == [3 * 8 + 7, 4 * 8, 5 * 8 + 7, 6 * 8]
