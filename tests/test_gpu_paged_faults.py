"""What the paged ops report at the next sync, and what they leave as it was."""

from __future__ import annotations

import numpy as np
import pytest

import paged_model as pm
from test_gpu_paged import Batch, Tables, up

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n_free,lens,want", [
    (3, [8, 2], [-1, 0]),      # 3 free, 2 returned, 4 in all
    (4, [0, 1], [0, -1]),      # a full list and one returned
    (-1, [3, 2], [1, 1]),
    (5, [3, 2], [1, 1]),
    (2 ** 31 - 1, [3, 2], [-1, 1])])
def test_block_tables_more_pages_than_there_are(backend, dev, n_free, lens, want):
    """Pages that would not fit the free list, or a count of free pages outside 0..n_pages, are reported at the next
    sync, once; what is computed follows the counts held to 0..n_pages."""
    ps, n_pages, max_rows = 4, 4, 3
    table, free = np.array([[0, 1], [2, -1]], np.int32), np.array([3, 0, 1, 2], np.int32)
    t = Tables(backend, dev, lens, want, table, free, n_free, ps, max_rows)
    ref = pm.block_tables(lens, want, table, free, n_free, ps, n_pages, max_rows, 0)
    t.call()
    with pytest.raises(backend.HipError, match="outside the cache"):
        dev.sync()
    dev.sync()
    t.check(ref, table, free)


def test_block_tables_every_page_free_again_is_no_fault(backend, dev):
    """All pages returned: the list is full, and nothing is reported."""
    table, free = np.array([[0, 1], [2, 3]], np.int32), np.array([4, -1, -1, -1, -1], np.int32)
    t = Tables(backend, dev, [8, 5], [-1, -1], table, free, 1, 4, 2)
    ref = pm.block_tables([8, 5], [-1, -1], table, free, 1, 4, 5, 2, 0)
    assert ref["n_free"] == 5
    t.call()
    dev.sync()
    t.check(ref, table, free)
