"""Attention over a paged cache: every pair of cache formats, heads between the padded sizes, steps far smaller than
their buffers, pages that several requests hold, and row starts and lengths that make no sense."""

from __future__ import annotations

import numpy as np
import pytest

from test_gpu_paged import Batch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("k_format,v_format", [(0, 2), (1, 0), (2, 1)])
@pytest.mark.parametrize("heads,kv_heads,head_dim", [(8, 4, 256), (1, 1, 32), (3, 1, 64), (6, 2, 96), (16, 1, 128), (4, 2, 512), (32, 2, 160)])
def test_attention_mixed_formats(backend, dev, heads, kv_heads, head_dim, k_format, v_format):
    """The pairs in which one cache alone is f16 or coarser."""
    Batch(backend, dev, 101, [0, 3, 40, 131], [1, 1, 1, 1], 75, 16, heads, kv_heads, head_dim, k_format, v_format).run()
    Batch(backend, dev, 102, [0, 30, 7], [3, 1, 19], 33, 7, heads, kv_heads, head_dim, k_format, v_format).run("several rows")
    Batch(backend, dev, 103, [900, 10, 333], [1, 4, 1], 1201, 16, heads, kv_heads, head_dim, k_format, v_format,
          window=700).run("split, window")


@pytest.mark.parametrize("k_format", [0, 1, 2])
@pytest.mark.parametrize("v_format", [0, 1, 2])
@pytest.mark.parametrize("head_dim", [192, 224, 288, 320, 416, 480])
def test_attention_heads_between_padded_sizes(backend, dev, head_dim, k_format, v_format):
    """Heads that fill part of a padded one (256 or 512 dims): products past the head, the join's second half."""
    for window in (0, 90):
        Batch(backend, dev, 104, [0, 500, 12], [1, 2, 40], 130, 24, 4, 2, head_dim, k_format, v_format, window=window).run(f"{window}")
    Batch(backend, dev, 105, [3] * 70, [1] * 70, 300, 16, 2, 1, head_dim, k_format, v_format).run("many")  # blocks of f16


@pytest.mark.parametrize("heads,kv_heads,head_dim,k_format,v_format", [(8, 4, 256, 0, 0), (4, 1, 64, 1, 2), (2, 1, 512, 0, 0)])
def test_attention_captured_for_many_more_rows(backend, dev, heads, kv_heads, head_dim, k_format, v_format):
    """One graph captured for 2048 rows and 40 requests serves steps of a few rows, of none, and of 700: every replay
    gives the eager result within the tolerance, and rows of no request stay."""
    one = backend.HipDevice.new(0)
    try:
        steps = [([300, 5, 0, 61] + [0] * 36, [1, 1, 1, 1] + [0] * 36), ([9] * 40, [1] * 40), ([4] * 40, [0] * 40),
                 ([0, 30, 200] + [7] * 37, [500, 163, 0] + [1] * 37), ([300] + [0] * 39, [0] * 39 + [1])]
        first = Batch(backend, one, 106, *steps[3], 200, 16, heads, kv_heads, head_dim, k_format, v_format, pad=2048 - 700).upload()
        first.stride = 1 << 10
        wide = np.full((40, first.stride), -1, np.int32)
        first.d["table"].close()
        first.d["table"] = backend.HipBuffer.from_host(one, wide)
        graph, state = None, first.d
        for turn, (before, new) in enumerate(steps + steps[:2]):
            b = Batch(backend, one, 107 + turn, before, new, 200, 16, heads, kv_heads, head_dim, k_format, v_format,
                      pad=2048 - sum(new))
            slots = first.n_pages * 16
            assert b.n_pages <= first.n_pages and b.max_rows == 2048
            wide[:] = -1
            wide[:, :b.stride] = b.table
            state["table"].copy_from_host(wide)
            for name in ("q", "lens", "row_start", "prefix"):
                state[name].copy_from_host(np.ascontiguousarray(getattr(b, name)))
            for name in ("k", "v"):
                rows = np.zeros((slots, getattr(b, name).shape[1]), np.uint8)
                rows[:len(getattr(b, name))] = getattr(b, name)
                state[name].copy_from_host(rows)
            first.d = b.d = state
            b.d["out"].copy_from_host(np.full(2048 * heads * head_dim, 5.0, np.float32))
            if graph is None:
                first.call()
                one.sync()
                graph = one.capture(first.call)
            else:
                graph.launch()
                one.sync()
            if b.rows:
                b.check(f"step {turn}")
            else:
                assert (b.d["out"].numpy() == 5.0).all()
        graph.close()
        for x in state.values():
            x.close()
    finally:
        one.close()


def test_attention_pages_that_requests_share(backend, dev):
    """A page may stand in several requests' rows of the table, twice in one, and in the prefix: it is only read."""
    b = Batch(backend, dev, 120, [60, 60, 60], [1, 2, 1], 48, 16, 4, 2, 128)
    b.table[1, :3] = b.table[0, :3]
    b.table[2, 1] = b.table[2, 0]
    b.table[2, 2] = b.prefix[1]
    b.run()


@pytest.mark.parametrize("starts", [[0, 1 << 30, 2, 3], [-5, -1, 1, 3], [3, 2, 1, 0], [0, 1, 2, 6], [0, 1, 2, 2 ** 31 - 1], [-2 ** 31, 0, 1, 2]])
@pytest.mark.parametrize("k_format", [0, 1])
def test_attention_row_starts_that_make_no_sense(backend, dev, starts, k_format):
    """Row starts that do not ascend within 0..max_rows are reported, nothing is written, and the next call is right."""
    b = Batch(backend, dev, 121, [10, 20, 30], [1, 1, 1], 16, 16, 4, 2, 64, k_format, k_format).upload()
    b.d["row_start"].copy_from_host(np.array(starts, np.int32))
    b.call()
    with pytest.raises(backend.HipError, match="outside the cache"):
        dev.sync()
    dev.sync()
    assert (b.d["out"].numpy() == 5.0).all()
    b.d["row_start"].copy_from_host(b.row_start)
    b.call()
    dev.sync()
    b.check()


@pytest.mark.parametrize("k_format", [0, 2])
@pytest.mark.parametrize("lens", [[1 << 30, 21, 31], [11, -9, 31], [11, 21, -2 ** 31], [2 ** 31 - 1, -1, 1 << 20]])
def test_attention_lengths_that_make_no_sense(backend, dev, lens, k_format):
    """Lengths outside 0..table row are reported and taken as its nearest end; places behind a request's own pages have
    no page and are left out.  The other requests' rows are what they are."""
    b = Batch(backend, dev, 122, [10, 20, 30], [1, 1, 1], 16, 16, 4, 2, 64, k_format, k_format)
    true = b.lens.copy()
    b.upload()
    b.d["lens"].copy_from_host(np.array(lens, np.int32))
    b.call()
    with pytest.raises(backend.HipError, match="outside the cache"):
        dev.sync()
    dev.sync()
    got = b.d["out"].numpy().reshape(b.max_rows, 4, 64).astype(np.float64)
    assert (got[3:] == 5.0).all()
    whole = b.reference()[0]
    for r in range(3):
        if 0 <= lens[r] <= b.stride * 16:
            assert lens[r] == true[r]
            want = whole[r]
        elif lens[r] < 0:  # length 0, one row: it stands at the prefix's last position and sees the prefix
            b.lens = true.copy()
            b.lens[r] = 0
            want = b.reference()[0][r]
        else:
            continue  # the NaN behind its own positions is among what it sees
        assert np.abs(got[r] - want).max() <= 1e-5 * np.abs(whole[:3]).max()
