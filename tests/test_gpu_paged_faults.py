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


def test_faults_of_replays_and_of_each_context_are_reported_once(backend, dev):
    """Every replay of a graph that holds a bad call is reported by the sync after it, and by that one alone; a graph
    captured without a fault reports one that its inputs bring later; another context's syncs stay clean."""
    one = backend.HipDevice.new(0)
    heads, kv, hd = 2, 1, 64
    try:
        k, v = (up(backend, one, np.zeros((8, kv * hd), np.float16)) for _ in range(2))
        x, q = up(backend, one, np.ones((2, (heads + 2 * kv) * hd), np.float32)), backend.HipBuffer.alloc(one, 2 * heads * hd)
        slots, pos = up(backend, one, np.array([3, 5], np.int32)), up(backend, one, np.zeros(2, np.int32))
        call = lambda: one.qkv_postprocess_paged(x, q, k, v, slots, pos, 2, 2, 4, heads, kv, hd, 10000.0)  # noqa: E731
        call()
        one.sync()
        graph = one.capture(call)
        for bad in (False, True, False, True, True):
            slots.copy_from_host(np.array([3, 8 if bad else 5], np.int32))
            graph.launch()
            dev.sync()
            if bad:
                with pytest.raises(backend.HipError, match="outside the cache"):
                    one.sync()
            one.sync()
        graph.close()
        for b in (k, v, x, q, slots, pos):
            b.close()
    finally:
        one.close()


@pytest.mark.parametrize("requests", [1, 40, 300])  # each of the join's forms
@pytest.mark.parametrize("k_format", [0, 1])
def test_rows_whose_every_page_is_outside_give_zeros(backend, dev, requests, k_format):
    """All positions of request 0 are left out: zeros, as a row that sees nothing gives; the others as they are."""
    b = Batch(backend, dev, 140, [45] * requests, [1] * requests, 0, 16, 8, 2, 64, k_format, k_format)
    want = b.reference()[0]
    b.upload()
    table = b.table.copy()
    table[0] = [-1, b.n_pages, 2 ** 31 - 1, -2 ** 31][:b.stride]
    b.d["table"].copy_from_host(table)
    b.call()
    with pytest.raises(backend.HipError, match="outside the cache"):
        dev.sync()
    dev.sync()
    got = b.d["out"].numpy().reshape(b.max_rows, 8, 64)
    assert (got[0] == 0.0).all() and (got[b.rows:] == 5.0).all()
    if requests > 1:
        assert np.abs(got[1:b.rows] - want[1:b.rows]).max() <= 1e-5 * np.abs(want[1:b.rows]).max()
